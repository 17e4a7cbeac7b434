"""GPU: gradients of the norms' vectors are sums in 32 bits, rounded once: vectors in 16 bits get the rounding, to the bit, of what the same
values in 32 bits get."""
import pytest
import torch

from lethe_b200 import ops

from .test_gpu_block_norms import randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D", [(3001, 4096), (20011, 64), (777, 100), (300, 8192)])
def test_vectors_in_16_bits(rows, D, dt):
    x, z, dy, dr = (randn(rows, D, seed=i, dt=dt) for i in range(4))
    narrow = [randn(D, seed=i, dt=dt) for i in (4, 5, 6)]

    def sums(vectors):
        w, sc, pw = (v.clone().requires_grad_(True) for v in vectors)
        both = ops.residual_norm(x, z, w, scale=sc, post_weight=pw)
        plain = ops.residual_norm(x, z, w, scale=sc)
        return [both[1].detach(), *torch.autograd.grad(both, (w, sc, pw), (dy, dr)), *torch.autograd.grad(plain, (w, sc), (dy, dr)), *torch.autograd.grad(ops.gated_norm(x, z, w), w, dy)]
    for a, b in zip(sums(narrow), sums([v.float() for v in narrow])):
        assert a.dtype == dt and torch.equal(a, b.to(dt))
