"""GPU: how many candidates the selection is asked for."""
import pytest
import torch

from lethe_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [-64, -3, -1, 0, 65])
def test_no_such_number(k):
    x, s = torch.randn(2, 3, 50, device="cuda"), torch.zeros(2, 3, device="cuda")
    with pytest.raises(ops.GdnError, match=f"as many candidates .*3 and {k}\\)"):
        ops.beam_select(x, s, k)
    with pytest.raises(ops.GdnError, match="candidates"):
        torch.jit.trace(lambda x, s: ops.beam_select(x, s, k)[:3], (x, s), check_trace=False)


def test_as_many_as_beams():
    x, s = torch.randn(2, 3, 50, device="cuda"), -torch.rand(2, 3, device="cuda")
    for got in (ops.beam_select(x, s), ops.beam_select(x, s, None), torch.jit.trace(lambda x, s: ops.beam_select(x, s)[:3], (x, s), check_trace=False)(x, s)):
        for a, b in zip(got[:3], ops.beam_select(x, s, 3)):
            assert torch.equal(a, b)
