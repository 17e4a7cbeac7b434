"""GPU: the decode step that goes on from other rows: the bits of the plain step on the rows that it reads, which it leaves as they are."""
import ctypes

import pytest
import torch

from lethe_b200 import native, ops

pytestmark = pytest.mark.gpu
K = 128


def inputs(B, slots, H, V, gate, delta, seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")      # noqa: E731
    q, k = (torch.nn.functional.normalize(rand(B, H, K), dim=-1).to(dtype) for _ in range(2))
    v = rand(B, H, V).to(dtype)
    decay = None if gate == "none" else -torch.nn.functional.softplus(rand(*((B, H) if gate == "scalar" else (B, H, K))))
    beta = torch.sigmoid(rand(B, H)) if delta else None
    return (q, k, v, decay, beta), 0.3 * rand(slots, H, K, V), torch.randint(-1, slots, (B,), generator=g, device="cuda")


def started(state, source):
    return torch.where((source < 0)[:, None, None, None], 0.0, state[source.clamp(min=0)])


@pytest.mark.parametrize("gate,delta", [("none", False), ("scalar", True), ("channel", True), ("scalar", False)])
@pytest.mark.parametrize("B,slots,H,V", [(1, 1, 1, 64), (5, 3, 2, 128), (4, 9, 8, 64), (37, 11, 16, 128), (100, 40, 7, 128), (150, 150, 9, 64)])
def test_bits_of_the_plain_step(B, slots, H, V, gate, delta):
    """Few pairs, and more than the GPU takes at a time (128 channels: the persistent kernel)."""
    for dtype, kind in ((torch.bfloat16, torch.int64), (torch.float32, torch.int32)):
        token, state, source = inputs(B, slots, H, V, gate, delta, B, dtype)
        before, want = state.clone(), started(state, source)
        wo = ops.gdn_decode_step(*token, want)
        out = torch.full((B, H, K, V), float("nan"), device="cuda")
        o = ops.gdn_decode_step(*token, state, source=source.to(kind), out=out)
        assert torch.equal(o, wo) and torch.equal(out, want) and torch.equal(state, before)


def test_against_64_bits():
    """A value of the state: S a, its product with k over 128 terms, the sum; each rounded once in 32 bits, the exponential by 2^-21."""
    for V in (64, 128):
        (q, k, v, g, beta), state, source = inputs(6, 5, 3, V, "scalar", True, 7)
        out = torch.empty(6, 3, K, V, device="cuda")
        o = ops.gdn_decode_step(q, k, v, g, beta, state, source=source, out=out, scale=0.25)
        S = started(state.double(), source) * torch.exp(g.double())[..., None, None]
        kd, qd = k.double()[..., None], q.double()[..., None]
        err = beta.double()[..., None] * (v.double() - (kd * S).sum(2))
        want = S + kd * err[..., None, :]
        size = S.abs() + kd.abs() * (v.double().abs() + (kd * S).abs().sum(2))[..., None, :]
        assert ((out - want).abs() <= size * (2.0**-21 + 132 * 2.0**-24)).all()
        exact, terms = 0.25 * (qd * want).sum(2), 0.25 * (qd.abs() * size).sum(2)
        assert ((o.double() - exact).abs() <= exact.abs() * 2.0**-8 + terms * (2.0**-21 + 264 * 2.0**-24) * 1.01).all()


def test_beams_in_two_buffers():
    """A search that swaps its buffers, against states that are moved in place."""
    B, W, H, V = 3, 4, 2, 128
    mine = [0.1 * torch.randn(B * W, H, K, V, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"), torch.empty(B * W, H, K, V, device="cuda")]
    moved = mine[0].clone()
    for t in range(5):
        token = inputs(B * W, 1, H, V, "channel", True, t)[0]
        parents = torch.randint(0, W, (B, W), generator=torch.Generator(device="cuda").manual_seed(t), device="cuda")
        ops.reorder_states(moved, parents)
        want = ops.gdn_decode_step(*token, moved)
        o = ops.gdn_decode_step(*token, mine[0], source=(parents + W * torch.arange(B, device="cuda")[:, None]).flatten(), out=mine[1])
        mine.reverse()
        assert torch.equal(o, want) and torch.equal(mine[0], moved)


@pytest.mark.parametrize("B,H,V", [(3, 2, 64), (3, 2, 128), (90, 8, 128)])
def test_a_source_outside_gives_nan_and_is_reported(B, H, V):
    word = ctypes.c_int32.from_address(native.ext().status_address(torch.cuda.current_device()))
    token, state, source = inputs(B, 4, H, V, "scalar", True)
    for bad in (-2, 4, 2**40):
        source[1] = bad
        out = torch.zeros(B, H, K, V, device="cuda")
        o = ops.gdn_decode_step(*token, state, source=source, out=out)
        torch.cuda.synchronize()
        assert o[1].isnan().all() and out[1].isnan().all()
        rest = torch.arange(B) != 1
        assert o[rest].isfinite().all() and out[rest].isfinite().all()
        with pytest.raises(ops.GdnError, match="index"):
            ops.gdn_decode_step(*token, state, source=source, out=out)
        assert word.value == 0


def test_refusals():
    token, state, source = inputs(3, 4, 2, 64, "scalar", True)
    out = torch.empty(3, 2, K, 64, device="cuda")
    big = torch.zeros(8, 2, K, 64, device="cuda")
    for kw, s, what in ((dict(source=source), state, "together"), (dict(out=out), state, "together"), (dict(source=source, out=state[:3]), state, "share"),
                        (dict(source=source, out=big[3:6]), big[:4], "share"), (dict(source=source[:2], out=out), state, "shapes"), (dict(source=source.float(), out=out), state, "int32"),
                        (dict(source=source, out=out.half()), state, "fp32"), (dict(source=source, out=out.transpose(0, 1)), state, "expects|contiguous"),
                        (dict(source=source, out=out.clone().requires_grad_(True)), state, "gradient"), (dict(source=source.cpu(), out=out), state, "device"),
                        (dict(source=source, out=out), state[:0], "slot"), (dict(source=source, out=out[:2]), state, "expects")):
        with pytest.raises(ops.GdnError, match=what):
            ops.gdn_decode_step(*token, s, **kw)
    ops.gdn_decode_step(*token, big[:4], source=source, out=big[4:7])
    none = tuple(t[:0] for t in token)
    assert ops.gdn_decode_step(*none, state, source=source[:0], out=out[:0]).shape == (0, 2, 64)


def test_inputs_in_the_memory_of_the_result():
    token, state, source = inputs(3, 4, 2, 128, "channel", True, dtype=torch.float32)
    want = torch.empty(3, 2, K, 128, device="cuda")
    wo = ops.gdn_decode_step(*token, state, source=source, out=want)
    out = torch.zeros(3, 2, K, 128, device="cuda")
    flat, at, views = out.view(-1), 0, []
    for t in (*token, source):
        n = t.numel() * t.element_size() // 4
        part = flat[at:at + n].view(t.dtype).view(t.shape)
        part.copy_(t)
        views.append(part)
        at += n
    o = ops.gdn_decode_step(*views[:5], state, source=views[5], out=out)
    assert torch.equal(o, wo) and torch.equal(out, want)


def test_captured_and_traced():
    token, state, source = inputs(4, 6, 2, 128, "scalar", True)
    out = torch.empty(4, 2, K, 128, device="cuda")
    ops.gdn_decode_step(*token, state, source=source, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = ops.gdn_decode_step(*token, state, source=source, out=out)
    traced = torch.jit.trace(lambda q, k, v, g, b, s, i, out: ops.gdn_decode_step(q, k, v, g, b, s, source=i, out=out), (*token, state, source, out.clone()), check_trace=False)
    for seed in (3, 4):
        other, s, i = inputs(4, 6, 2, 128, "scalar", True, seed)
        for a, b in zip((*token, state, source), (*other, s, i)):
            a.copy_(b)
        want = torch.empty_like(out)
        wo = ops.gdn_decode_step(*other, s, source=i, out=want)
        g.replay()
        assert torch.equal(o, wo) and torch.equal(out, want)
        mine = torch.empty_like(out)
        assert torch.equal(traced(*other, s, i, mine), wo) and torch.equal(mine, want)
