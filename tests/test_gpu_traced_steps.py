"""GPU: the one-token calls under torch.jit.trace, as a traced generation loop uses them: they compute, and the state moves on."""
import pytest
import torch

from lethe_b200 import ops

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore")]


def diag(seed, types=(torch.bfloat16, torch.float32), shape=(3, 2, 40)):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=gen).to("cuda", types[0])
    g = -torch.rand(*shape, generator=gen).to("cuda", types[1])
    return x, g, torch.randn(*shape, generator=gen).cuda()


def poison(like):
    """Memory of these sizes that the allocator hands out next holds none of the results."""
    for _ in range(4):
        torch.full_like(like, float("nan"))


@pytest.mark.parametrize("complement", [False, True])
@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
def test_diag_scan_step(types, complement):
    x, g, state = diag(1, types)
    before = state.clone()
    traced = torch.jit.trace(lambda x, g, s: ops.diag_scan_step(x, g, s, complement=complement), (x, g, state))
    assert torch.equal(before, diag(1, types)[2])
    for seed in (2, 3):
        x, g, state = diag(seed, types)
        mine = state.clone()
        want = ops.diag_scan_step(x, g, state, complement=complement)
        for _ in range(2):                     # the second token goes on from the first one's state
            poison(want)
            got = traced(x, g, mine)
            assert got.dtype == want.dtype and torch.equal(got, want) and torch.equal(mine, state)
            want = ops.diag_scan_step(x, g, state, complement=complement)


def test_diag_scan_step_what_is_read_behind_it_is_the_new_state():
    """Two tokens in one trace, and a result that only the state leads to."""
    def two(x, g, s):
        ops.diag_scan_step(x, g, s)
        ops.diag_scan_step(x * 2, g, s)
        return s * 3
    traced = torch.jit.trace(two, diag(1))
    a, b = diag(2), diag(2)
    assert torch.equal(traced(*a), two(*b)) and torch.equal(a[2], b[2])


def test_diag_scan_step_has_no_gradient_and_refuses_as_ever():
    def f(x, g, s):
        return ops.diag_scan_step(x, g, s) * 1
    traced = torch.jit.trace(f, diag(1))
    x, g, state = diag(2)
    assert not traced(x.requires_grad_(True), g, state).requires_grad
    for bad, what in (((x.cpu(), g, state), "CUDA device"), ((x[:1], g, state), "shapes"), ((x, g, state.half()), "fp32")):
        with pytest.raises(Exception, match=what):
            torch.jit.trace(f, bad)
        with pytest.raises(Exception, match=what):
            traced(*bad)


def matrix(seed, gate, delta):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(2, 3, n, generator=gen).to("cuda", torch.bfloat16) for n in (128, 128, 64))
    g = {"none": None, "scalar": -torch.rand(2, 3, generator=gen), "channel": -torch.rand(2, 3, 128, generator=gen)}[gate]
    beta = torch.rand(2, 3, generator=gen) if delta else None
    return [None if t is None else t.cuda() for t in (q, k * 128 ** -0.5, v, g, beta, torch.randn(2, 3, 128, 64, generator=gen))]


@pytest.mark.parametrize("scale", [None, 0.5])
@pytest.mark.parametrize("gate,delta", [("scalar", True), ("channel", True), ("scalar", False), ("none", False)])
def test_gdn_decode_step(gate, delta, scale):
    def call(*given):
        it = iter(given)
        full = [None if t is None else next(it) for t in matrix(1, gate, delta)]
        return ops.gdn_decode_step(*full, scale=scale)
    there = lambda seed: tuple(t for t in matrix(seed, gate, delta) if t is not None)
    traced = torch.jit.trace(call, there(1))
    a, b = there(2), there(2)
    for _ in range(2):
        want = call(*b)
        poison(want)
        assert torch.equal(traced(*a), want) and torch.equal(a[-1], b[-1])
