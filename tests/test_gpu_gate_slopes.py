"""GPU: gradients of the gated norm's gate where the gate is far from zero: each within roundings of itself, not of the largest.

60 roundings of 2^-24 as for the norms, and 2 |gate| for the exponential of a rounded argument."""
import pytest
import torch

from lethe_b200 import ops

from .test_gpu_block_norms import K, close, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("D", [64, 100, 1024])
def test_sigmoid_slopes(D, types):
    xt, wt = types
    z = torch.arange(-60, 61, dtype=torch.float32, device="cuda").to(xt)
    R = z.numel()
    x, dy, w = randn(R, D, seed=1, dt=xt), randn(R, D, seed=2, dt=xt), randn(D, seed=3, dt=wt)
    gate = z[:, None].expand(R, D).contiguous().requires_grad_(True)
    y = ops.gated_norm(x, gate, w, activation="sigmoid")
    dz, = torch.autograd.grad(y, gate, dy)
    xd, zd = x.double(), gate.detach().double()
    n = xd / torch.sqrt(xd.square().mean(-1, keepdim=True) + 1e-6)
    want = dy.double() * n * w.double() * torch.sigmoid(zd) * torch.sigmoid(-zd)
    close(dz, want, want.abs(), K + 2 * 60)
    close(y.detach(), n * w.double() * torch.sigmoid(zd), (n * w.double()).abs() * torch.sigmoid(zd), K + 2 * 60)


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
def test_gates_without_bound(act):
    """Far beyond what the exponential holds: the limits, which are finite; an infinite gate of the sigmoid too."""
    far = [1e3, -1e3, 3e38, -3e38] + ([float("inf"), float("-inf")] if act == "sigmoid" else [])
    for dt in (torch.float32, torch.bfloat16):
        gate = torch.tensor(far, device="cuda").to(dt)[:, None].expand(len(far), 64).contiguous().requires_grad_(True)
        x, dy, w = randn(len(far), 64, seed=1, dt=dt), randn(len(far), 64, seed=2, dt=dt), randn(64, seed=3)
        leaf = x.clone().requires_grad_(True)
        dx, dz = torch.autograd.grad(ops.gated_norm(leaf, gate, w, activation=act), (leaf, gate), dy)
        assert bool(dz[1::2].eq(0).all()) and bool(dx[1::2].eq(0).all())
        if act == "sigmoid":
            assert bool(dz.eq(0).all()) and bool(dx.isfinite().all())
        else:
            one = dy.double() * w.double() * x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-6)
            close(dz[0], one[0], one[0].abs())
