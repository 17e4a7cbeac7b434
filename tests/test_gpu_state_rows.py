"""GPU: states of sequences that are moved - reordered by beams, forked and compacted in a pool.  Nothing is computed, so everything is compared
bit for bit with indexing, what is not to be touched among it."""
import ctypes

import pytest
import torch

from lethe_b200 import native, ops

pytestmark = pytest.mark.gpu


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def values(shape, dtype, seed=0):
    n = 1
    for d in shape:
        n *= d
    raw = torch.randint(0, 256, (max(1, n * torch.empty(0, dtype=dtype).element_size()),), generator=gen(seed), device="cuda", dtype=torch.uint8)
    if dtype == torch.bool:
        return (raw[:n] % 2).bool().view(shape)
    return raw[:n * torch.empty(0, dtype=dtype).element_size()].view(dtype).view(shape)


def bits(t):
    t = t.contiguous()
    return t.view(torch.uint8) if t.dim() and t.dtype != torch.bool else t


def same(a, b):
    return a.shape == b.shape and torch.equal(bits(a), bits(b))


ROWS = [(1,), (3,), (16,), (5, 3), (77, 3), (128, 64), (7, 31, 13), (2, 128, 128), (0,)]
TYPES = [torch.float32, torch.bfloat16, torch.uint8, torch.int64, torch.bool, torch.complex64]


# ---------------------------------------------------------------------------------------------------------------
# Reorder
# ---------------------------------------------------------------------------------------------------------------
def reordered(t, parents):
    B, W = parents.shape
    rows = (torch.arange(B, device="cuda")[:, None] * W + parents).flatten()
    return t.reshape(B * W, *t.shape[1 if t.shape[0] == B * W else 2:])[rows].reshape(t.shape)


@pytest.mark.parametrize("row", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
def test_reorder(dtype, row):
    for B, W in ((1, 1), (3, 4), (2, 7), (1, 16), (5, 1)):
        for kind in (torch.int64, torch.int32):
            parents = torch.randint(0, W, (B, W), generator=gen(W), device="cuda")
            for shape in ((B * W, *row), (B, W, *row)):
                t = values(shape, dtype, 1)
                want = reordered(t, parents)
                assert ops.reorder_states(t, parents.to(kind)) is None
                assert same(t, want)


@pytest.mark.parametrize("W", [2, 5, 8, 31, 32, 33, 64, 65, 100, 255, 256])
def test_reorder_maps(W):
    i = torch.arange(W, device="cuda")
    maps = [i, i.flip(0), i.roll(1), i.roll(-1), i * 0, i * 0 + W - 1, i // 2, torch.randperm(W, generator=gen(1), device="cuda"),
            torch.where(i % 3 == 0, i, i // 3), (i + 1).clamp(max=W - 1)]
    parents = torch.stack(maps)
    for row in ((600,), (3,)):
        t = values((len(maps) * W, *row), torch.float32)
        want = reordered(t, parents)
        ops.reorder_states(t, parents)
        assert same(t, want)


def test_reorder_many_tensors_in_one_call():
    B, W = 3, 5
    parents = torch.randint(0, W, (B, W), generator=gen(), device="cuda")
    for count in (0, 1, 31, 32, 33, 70):
        ts = [values((B * W, 1 + 37 * i), TYPES[i % len(TYPES)], i) if i % 3 else values((B, W, 8 * i + 4), torch.bfloat16, i) for i in range(count)]
        want = [reordered(t, parents) for t in ts]
        ops.reorder_states(tuple(ts), parents)
        assert all(same(a, b) for a, b in zip(ts, want))


LAYOUTS = {      # rows of a larger buffer, and what of it they are
    "slices": lambda b: b[:, 1],
    "every other": lambda b: b[::2, 0],
    "groups last": lambda b: b.view(4, 3, *b.shape[1:]).transpose(0, 1)[:, :, 0],
    "groups apart": lambda b: b.view(3, 4, *b.shape[1:])[:, :2, 2],
}


@pytest.mark.parametrize("n", [16, 9])
@pytest.mark.parametrize("layout", sorted(LAYOUTS))
def test_reorder_strides(layout, n):
    b = values((12, 3, n), torch.float32)
    start = b.clone()
    view = LAYOUTS[layout](b)
    W = {"slices": 4, "every other": 2, "groups last": 4, "groups apart": 2}[layout]
    parents = torch.randint(0, W, (3, W), generator=gen(3), device="cuda")
    want = reordered(view.clone(), parents)
    ops.reorder_states(view, parents)
    assert same(view, want)
    LAYOUTS[layout](start).copy_(want)                                                    # and nothing else
    assert same(b, start)


def test_reorder_slices_of_one_buffer():
    """Layers that lie between one another's rows."""
    b = values((8, 3, 50), torch.bfloat16)
    parents = torch.randint(0, 4, (2, 4), generator=gen(4), device="cuda")
    want = torch.stack([reordered(b[:, i].clone(), parents) for i in range(3)], 1)
    ops.reorder_states(list(b.unbind(1)), parents)
    assert same(b, want)


def test_reorder_refusals():
    t, p = torch.zeros(6, 8, device="cuda"), torch.zeros(2, 3, dtype=torch.long, device="cuda")
    for states, parents, what in (([t, t], p, "share"), ([t, t[3:].view(2, 3, 4)], p, "share|shapes"), (t[:5], p, "shapes"), (t.t().contiguous().t(), p, "contiguous"),
                                  (t, p.float(), "int32"), (t, p[0], "shapes"), (t.clone().requires_grad_(True), p, "gradient"), (t[:1].expand(6, 8), p, "overlap"),
                                  (torch.zeros(48, device="cuda").as_strided((6, 8), (4, 1)), p, "overlap"), ([t, t[:, 4:]], p, "share"), ([t[:, :5], t[:, 4:]], p, "share"),
                                  (t.cpu(), p, "CUDA"), (t, p.cpu(), "CUDA"), (torch.zeros(2 * 257, device="cuda"), torch.zeros(2, 257, dtype=torch.long, device="cuda"), "256"),
                                  (torch.zeros(3, 2, 8, device="cuda"), p, "shapes")):
        with pytest.raises(ops.GdnError, match=what):
            ops.reorder_states(states, parents)
    ops.reorder_states([t[:, :5], t[:, 5:]], p)
    ops.reorder_states([], p)
    ops.reorder_states(torch.zeros(0, 8, device="cuda"), p[:0])
    with torch.inference_mode():
        ops.reorder_states(torch.zeros(6, 8, device="cuda"), p)


def test_a_parent_outside_leaves_its_row_and_is_reported():
    word = ctypes.c_int32.from_address(native.ext().status_address(torch.cuda.current_device()))
    for bad in (-1, 3, 2**40, -(2**40)):
        t = values((6, 5000), torch.float32)
        start = t.clone()
        p = torch.tensor([[1, bad, 0], [2, 2, 2]], device="cuda")
        ops.reorder_states(t, p)
        torch.cuda.synchronize()
        assert same(t, start[[1, 1, 0, 5, 5, 5]])
        assert word.value != 0
        with pytest.raises(ops.GdnError, match="index"):
            ops.reorder_states(t, torch.zeros_like(p))
        assert word.value == 0
    ops.reorder_states(t, torch.zeros_like(p))


def test_parents_in_the_memory_of_a_state():
    b = torch.zeros(4, 6, dtype=torch.long, device="cuda")
    b[:, 0] = torch.tensor([3, 0, 0, 1], device="cuda")
    b[:, 1:] = torch.arange(20, device="cuda").view(4, 5)
    want = b[b[:, 0]]
    ops.reorder_states(b, b[:, 0].view(1, 4))
    assert torch.equal(b, want)


# ---------------------------------------------------------------------------------------------------------------
# Fork and compact
# ---------------------------------------------------------------------------------------------------------------
def forked(states, live, source):
    live, states, target = live.tolist(), [t.clone() for t in states], []
    free, taken = [i for i, x in enumerate(live) if not x], list(live)
    for s in source.tolist():
        if free and (s == -1 or (0 <= s < len(live) and live[s])):
            to = free.pop(0)
            taken[to] = True
            for t in states:
                t[to] = 0 if s == -1 else t[s]
            target.append(to)
        else:
            target.append(-1)
    return states, torch.tensor(target, dtype=torch.long, device="cuda"), torch.tensor(taken, device="cuda")


def compacted(states, live):
    live, states = live.tolist(), [t.clone() for t in states]
    n = sum(live)
    place = [i if x else -1 for i, x in enumerate(live)]
    holes = [i for i in range(n) if not live[i]]
    for s in range(n, len(live)):
        if live[s]:
            place[s] = holes.pop(0)
            for t in states:
                t[place[s]] = t[s]
    return states, torch.tensor(place, dtype=torch.long, device="cuda"), n


def check_fork(states, live, source):
    before, want = live.clone(), forked(states, live, source)
    target, after = ops.fork_states(states, live, source)
    assert torch.equal(live, before) and target.dtype == torch.int64 and after.dtype == torch.bool
    assert torch.equal(target, want[1]) and torch.equal(after, want[2])
    assert all(same(a, b) for a, b in zip(states, want[0]))


def check_compact(states, live):
    before, want = live.clone(), compacted(states, live)
    place, count = ops.compact_states(states, live)
    assert torch.equal(live, before) and place.dtype == count.dtype == torch.int64 and count.dim() == 0
    assert torch.equal(place, want[1]) and int(count) == want[2]
    assert all(same(a, b) for a, b in zip(states, want[0]))


def pools(S, rows=ROWS):
    return [values((S, *row), TYPES[i % len(TYPES)], i) for i, row in enumerate(rows)]


@pytest.mark.parametrize("share", [0.0, 0.1, 0.5, 0.9, 1.0])
@pytest.mark.parametrize("S", [1, 2, 3, 37, 255, 256, 257, 300])
def test_pools(S, share):
    for seed in range(3):
        live = torch.rand(S, generator=gen(seed), device="cuda") < share
        check_compact(pools(S), live)
        for n in (1, 5, S, 2 * S + 3):
            source = torch.randint(-3, S + 2, (n,), generator=gen(seed + n), device="cuda")
            check_fork(pools(S), live, source if seed else source.int())


def test_fork_and_compact_of_whole_rows():
    live = torch.rand(24, generator=gen(1), device="cuda") < 0.5
    rows = [(8, 128, 64), (3, 128, 128), (4097,), (50001,)]
    check_fork(pools(24, rows), live, torch.randint(-1, 24, (12,), generator=gen(2), device="cuda"))
    check_compact(pools(24, rows), live)


def test_fork_one_for_many():
    live = torch.tensor([False, True] + [False] * 62, device="cuda")
    t = values((64, 3000), torch.float32)
    check_fork([t], live, torch.ones(63, dtype=torch.long, device="cuda"))
    assert same(t, t[:1].expand(64, 3000))


@pytest.mark.parametrize("sources", [1, 3, 40])
def test_fork_more_than_l2_holds_at_once(sources):
    """Moves of one source share its loads: more, and fewer, than eight of them, zeros, and rows of no particular size beside them."""
    S, n = 150, 90
    live = torch.zeros(S, dtype=torch.bool, device="cuda")
    live[torch.randperm(S, generator=gen(1), device="cuda")[:45]] = True
    of = torch.cat([live.nonzero().flatten()[:sources], torch.tensor([-1, -2, S + 3], device="cuda"), (~live).nonzero().flatten()[:1]])
    for seed in range(2):
        source = of[torch.randint(0, len(of), (n,), generator=gen(seed), device="cuda")]
        check_fork([values((S, 8, 128, 128), torch.float32), values((S, 7, 9), torch.bfloat16), values((S, 4, 128, 64), torch.float32)], live, source)


@pytest.mark.parametrize("W", [9, 16, 17, 24, 32])
def test_reorder_wide_groups_of_large_rows(W):
    for seed, few in ((0, W), (1, 2)):
        parents = torch.randint(0, few, (3, W), generator=gen(seed), device="cuda")
        ts = [values((3 * W, 100000), torch.uint8), values((3, W, 4, 128, 64), torch.float32), values((3 * W, 999), torch.uint8)]
        want = [reordered(t, parents) for t in ts]
        ops.reorder_states(ts, parents)
        assert all(same(a, b) for a, b in zip(ts, want))


@pytest.mark.parametrize("S", [4096, 65535, 65536])
def test_large_pools(S):
    live = torch.rand(S, generator=gen(S), device="cuda") < 0.5
    half = torch.arange(S, device="cuda") >= S // 2                                      # as many moves as there can be
    for marks in (live, half, ~half):
        check_compact([values((S, 2), torch.int32)], marks)
    source = torch.randint(-1, S, (4096,), generator=gen(1), device="cuda")
    check_fork([values((S, 2), torch.int32), values((S,), torch.uint8)], live, source)
    check_fork([], ~half, source)


def test_pool_strides_and_many_tensors():
    live = torch.rand(20, generator=gen(2), device="cuda") < 0.5
    source = torch.randint(-1, 20, (8,), generator=gen(3), device="cuda")
    b = values((20, 3, 33), torch.bfloat16)
    want = b.clone()
    want[:, 1] = forked([b[:, 1]], live, source)[0][0]
    ops.fork_states([b[:, 1]], live, source)
    assert same(b, want)
    want[:, 0], want[:, 2] = (compacted([b[:, i]], live)[0][0] for i in (0, 2))
    ops.compact_states([b[:, 0], b[:, 2]], live)
    assert same(b, want)
    check_fork([values((20, 1 + i), TYPES[i % 6], i) for i in range(40)], live, source)
    check_compact([values((20, 1 + i), TYPES[i % 6], i) for i in range(40)], live)


def test_pool_refusals():
    t, live, src = torch.zeros(6, 8, device="cuda"), torch.zeros(6, dtype=torch.bool, device="cuda"), torch.zeros(2, dtype=torch.long, device="cuda")
    for states, marks, what in (([t, t], live, "share"), (t[:5], live, "shapes"), (t.t().contiguous().t(), live, "contiguous"), (t, live.int(), "truth"), (t, live[None], "shapes"),
                                (t.clone().requires_grad_(True), live, "gradient"), (t[:1].expand(6, 8), live, "overlap"), (t.cpu(), live, "CUDA"), (t, live.cpu(), "CUDA"),
                                (t[:0], live[:0], "slots"), (torch.zeros(65537, device="cuda"), torch.zeros(65537, dtype=torch.bool, device="cuda"), "slots")):
        for call in (lambda: ops.fork_states(states, marks, src), lambda: ops.compact_states(states, marks)):
            with pytest.raises(ops.GdnError, match=what):
                call()
    for source, what in ((src.float(), "int32"), (src[None], "shapes"), (src.cpu(), "device"), (torch.zeros(4097, dtype=torch.long, device="cuda"), "entries")):
        with pytest.raises(ops.GdnError, match=what):
            ops.fork_states(t, live, source)
    target, after = ops.fork_states(t, live, src[:0])
    assert target.shape == (0,) and torch.equal(after, live) and after.data_ptr() != live.data_ptr()


def test_marks_and_sources_in_the_memory_of_a_state():
    b = torch.zeros(4, 8, dtype=torch.bool, device="cuda")
    b[2:] = True
    marks = b[:, 0]
    want = compacted([b.clone()], marks.clone())
    place, count = ops.compact_states(b, marks)
    assert same(b, want[0][0]) and torch.equal(place, want[1]) and int(count) == 2
    i = torch.tensor([[0, 9], [1, 9], [2, 9], [3, 9]], device="cuda")
    live = torch.tensor([True, False, False, True], device="cuda")
    source = i[:2, 0] * 3                                                                 # 0, 3
    i[:2, 0] = source
    want = forked([i.clone()], live, source)
    target, _ = ops.fork_states(i, live, i[:2, 0])
    assert torch.equal(i, want[0][0]) and torch.equal(target, want[1])


# ---------------------------------------------------------------------------------------------------------------
# Streams, graphs, traces
# ---------------------------------------------------------------------------------------------------------------
def test_captured_and_replayed():
    t, parents = values((12, 3000), torch.float32), torch.zeros(3, 4, dtype=torch.long, device="cuda")
    pool, live, source = values((40, 500), torch.float32, 1), torch.zeros(40, dtype=torch.bool, device="cuda"), torch.zeros(9, dtype=torch.long, device="cuda")
    ops.reorder_states(t, parents), ops.fork_states(pool, live, source), ops.compact_states(pool, live)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.reorder_states(t, parents)
        target, after = ops.fork_states(pool, live, source)
        place, count = ops.compact_states(pool, after)
    for seed in range(4):
        parents.copy_(torch.randint(0, 4, (3, 4), generator=gen(seed), device="cuda"))
        live.copy_(torch.rand(40, generator=gen(seed), device="cuda") < 0.4)
        source.copy_(torch.randint(-1, 40, (9,), generator=gen(seed), device="cuda"))
        want = reordered(t, parents)
        states, to, marks = forked([pool], live, source)
        states, at, n = compacted(states, marks)
        g.replay()
        assert same(t, want) and same(pool, states[0]) and torch.equal(target, to) and torch.equal(after, marks) and torch.equal(place, at) and int(count) == n


def test_other_streams():
    ts, parents = [values((32, 70000), torch.float32, i) for i in range(3)], torch.randint(0, 8, (4, 8), generator=gen(), device="cuda")
    want = [reordered(reordered(t, parents), parents) for t in ts]
    torch.cuda.synchronize()
    for t in ts:
        with torch.cuda.stream(torch.cuda.Stream()):
            ops.reorder_states(t, parents)
            ops.reorder_states(t, parents)
    torch.cuda.synchronize()
    assert all(same(a, b) for a, b in zip(ts, want))


@pytest.mark.filterwarnings("ignore")
def test_traced():
    def move(t, u, p):
        ops.reorder_states([t, u], p)
        ops.reorder_states(t, p)
        return t * 2
    make = lambda s: (torch.randn(6, 40, generator=gen(s), device="cuda"), torch.randn(6, 3, generator=gen(s), device="cuda"), torch.randint(0, 3, (2, 3), generator=gen(s), device="cuda"))      # noqa: E731
    traced = torch.jit.trace(move, make(0), check_trace=False)
    a, b = make(5), make(5)
    assert torch.equal(traced(*a), move(*b)) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])

    def pool(t, live, source):
        target, live = ops.fork_states([t], live, source)
        place, count = ops.compact_states(t, live)
        return target, live, place, count, t + 1
    make = lambda s: (torch.randn(9, 40, generator=gen(s), device="cuda"), torch.rand(9, generator=gen(s), device="cuda") < 0.4, torch.randint(-1, 9, (3,), generator=gen(s), device="cuda"))      # noqa: E731
    traced = torch.jit.trace(pool, make(0), check_trace=False)
    a, b = make(6), make(6)
    for x, y in zip(traced(*a), pool(*b)):
        assert torch.equal(x, y)


def test_versions():
    """Autograd sees that a state was changed."""
    t = torch.randn(4, 8, device="cuda")
    w = torch.randn(4, 8, device="cuda", requires_grad=True)
    y = (w * t).sum()
    ops.reorder_states(t, torch.tensor([[1, 0, 2, 3]], device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
