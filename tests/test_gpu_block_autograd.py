"""GPU: the operators beside the recurrence under what PyTorch wraps around an autograd function."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

from lethe_b200 import ops

pytestmark = pytest.mark.gpu


def inputs(seed=1):
    gen = torch.Generator().manual_seed(seed)
    d = {n: torch.randn(2, 260, 72, generator=gen).cuda() for n in ("x", "z")}
    d["g"], d["h0"] = -torch.rand(2, 260, 72, generator=gen).cuda(), torch.randn(2, 72, generator=gen).cuda()
    d.update({n: torch.randn(72, generator=gen).cuda() for n in ("w", "pw", "s")})
    return d


OPS = {
    "diag_scan": (lambda x, g, h0: ops.diag_scan(x, g, h0)[0], ("x", "g", "h0")),
    "gated_norm": (ops.gated_norm, ("x", "z", "w")),
    "residual_norm": (lambda x, z, w, s, pw: ops.residual_norm(x, z, w, scale=s, post_weight=pw)[0], ("x", "z", "w", "s", "pw")),
    "residual_norm, plain sum": (lambda x, z, w: ops.residual_norm(x, z, w)[1] * 2 + 0, ("x", "z", "w")),
}
every_op = pytest.mark.parametrize("name", sorted(OPS))


def gradients(f, leaves, out=None):
    o = f(*leaves) if out is None else out
    return torch.autograd.grad(o, leaves, torch.ones_like(o), allow_unused=True)


def same(a, b):
    return all((s is None and t is None) or torch.equal(s, t) for s, t in zip(a, b))


@every_op
def test_forward_mode_is_refused(name):
    f, names = OPS[name]
    d = inputs()
    for dual in names:
        with fwd_ad.dual_level():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(*[fwd_ad.make_dual(d[n], torch.ones_like(d[n])) if n == dual else d[n] for n in names])


@every_op
def test_hooks_that_move_saved_tensors(name):
    f, names = OPS[name]
    d = inputs()
    leaves = [d[n].clone().requires_grad_(True) for n in names]
    want = gradients(f, leaves)

    def unpack(t):                       # eight bytes past whatever the allocator gives
        room = torch.empty(t.nbytes + 8, dtype=torch.uint8, device="cuda")
        return room[8:].view(t.dtype).view(t.shape).copy_(t)
    for move in (lambda t: t.cuda(), unpack):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), move):
            o = f(*leaves)
        got = gradients(f, leaves, o)
        if move is unpack and "norm" in name:      # (rows on another boundary are summed in another order: 60 roundings of terms of order 1)
            assert all(s is None or float((s - t).abs().max()) <= 260 * 2 * 60 * 2 ** -24 * max(1.0, float(t.abs().max())) for s, t in zip(got, want))
        else:
            assert same(got, want)


@every_op
def test_checkpoint(name):
    from torch.utils.checkpoint import checkpoint
    f, names = OPS[name]
    d = inputs()
    leaves = [d[n].clone().requires_grad_(True) for n in names]
    want = gradients(f, leaves)
    assert same(gradients(f, leaves, checkpoint(lambda *t: f(*t), *leaves, use_reentrant=False)), want)


@every_op
def test_a_changed_input_is_noticed(name):
    f, names = OPS[name]
    d = inputs()
    leaves = [d[n].clone().requires_grad_(True) for n in names]
    inner = [t * 1 for t in leaves]
    o = f(*inner)
    with torch.no_grad():
        inner[0].add_(1)
        inner[2].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        gradients(f, leaves, o)


@every_op
@pytest.mark.filterwarnings("ignore")
def test_a_traced_call_computes(name):
    f, names = OPS[name]
    d, e = inputs(), inputs(2)
    traced = torch.jit.trace(lambda *t: f(*t) * 1, tuple(d[n] for n in names), check_trace=False)
    leaves, again = ([e[n].clone().requires_grad_(True) for n in names] for _ in range(2))
    o, want = traced(*leaves), f(*again)
    assert torch.equal(o, want)
    for a, b in zip(gradients(f, leaves, o), gradients(f, again, want)):
        assert a is b is None or torch.equal(torch.zeros_like(b) if a is None else a, torch.zeros_like(a) if b is None else b)


@every_op
def test_no_gradients_no_graph(name):
    f, names = OPS[name]
    d = inputs()
    leaves = [d[n].clone().requires_grad_(True) for n in names]
    with torch.no_grad():
        assert not f(*leaves).requires_grad
    with torch.inference_mode():
        assert not f(*leaves).requires_grad
    assert not f(*[d[n] for n in names]).requires_grad


AWAY = [(n, a) for n in sorted(OPS) for a in OPS[n][1]]


@pytest.mark.parametrize("name,away", AWAY)
def test_an_input_on_the_host_is_refused(name, away):
    f, names = OPS[name]
    d = inputs()
    d[away] = d[away].cpu()
    with pytest.raises(ops.GdnError, match="CUDA device"):
        f(*(d[n] for n in names))


@pytest.mark.parametrize("away", range(3))
def test_a_step_input_on_the_host_is_refused(away):
    t = [torch.zeros(2, 8, device="cuda") for _ in range(3)]
    t[away] = t[away].cpu()
    with pytest.raises(ops.GdnError, match="CUDA device"):
        ops.diag_scan_step(*t)
