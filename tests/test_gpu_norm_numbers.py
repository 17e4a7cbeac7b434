"""GPU: numbers that a float cannot hold are refused by the norms: as infinity they would give other results than the formulas."""
import pytest
import torch

from lethe_b200 import ops

pytestmark = pytest.mark.gpu


def test_numbers_beyond_fp32():
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    for eps in (1e39, 3.5e38, float("inf")):
        with pytest.raises(ops.GdnError, match="eps"):
            ops.gated_norm(x, x, w, eps=eps)
        with pytest.raises(ops.GdnError, match="eps"):
            ops.residual_norm(x, x, w, eps=eps)
    for scale in (1e39, -3.5e38):
        with pytest.raises(ops.GdnError, match="scale"):
            ops.residual_norm(x, x, w, scale=scale)
    # what a float holds is taken: near its largest, and infinity where the caller says so
    assert bool((ops.residual_norm(x, x, w, eps=3.4e38)[0] != 0).all())
    assert torch.equal(ops.residual_norm(x, None, w, scale=3.4e38)[1].isinf(), (x * 3.4e38).isinf())
    assert bool(ops.residual_norm(x, None, w, scale=float("inf"))[1].isinf().all())
