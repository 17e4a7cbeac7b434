"""GPU: beam search's selection against the definition in 64 bits.

Which candidates are chosen has to be right to the last place: they are whole numbers.  The scores: a term of a beam's sum of exponentials
is 2^-22 off by the hardware's exp2, twice (its tile's maximum, then its segment's), by the two roundings of its argument, |t| 2^-24 each
weighted with 2^t (below 2^-23), and by up to seven roundings of sums in 32 bits, 2^-24 each; the logarithm of the sum is off by as much, at
most 2 2^-22 + 2^-23 + 7 2^-24.  The rest is in 64 bits, and the result is rounded to fp32 once, by half a step."""
import itertools
import math

import pytest
import torch

from lethe_b200 import ops

pytestmark = pytest.mark.gpu
DEAD = float("-inf")
OFF = 2 * 2.0**-22 + 2.0**-23 + 7 * 2.0**-24


def reference(logits, scores, k=None, *, temperature=1.0, allowed=None, finished=None, eos=None, penalty=None):
    B, W, V = logits.shape
    k = W if k is None else k
    x = logits.double() / temperature
    if allowed is not None:
        x = x.masked_fill(~allowed.expand(B, W, V), DEAD)
    s = scores.double()
    pen = torch.ones_like(s) if penalty is None else penalty.double()
    lse = torch.logsumexp(x, 2)
    fin = torch.zeros_like(s, dtype=torch.bool) if finished is None else finished
    counts = s.isfinite() & (pen > 0) & pen.isfinite()
    on = counts & ~fin & lse.isfinite() & ~x.isnan().any(2) & (x < math.inf).all(2)
    value = torch.where(on[..., None], s[..., None] + (x - lse[..., None]), DEAD)
    if eos is not None:
        value[:, :, eos] = torch.where(fin & counts, s, value[:, :, eos])
    rank = (value / pen[..., None]).masked_fill(value == DEAD, DEAD).flatten(1)
    rank, at = rank.sort(stable=True, dim=1, descending=True)
    if W * V < k:
        rank, at = (torch.cat([t, t.new_full((B, k - W * V), fill)], 1) for t, fill in ((rank, DEAD), (at, 0)))
    rank, at = rank[:, :k], at[:, :k]
    none = rank == DEAD
    best = value.flatten(1).gather(1, at).masked_fill(none, DEAD)
    parents, tokens = (at // V).masked_fill(none, 0), (at % V).masked_fill(none, 0 if eos is None else eos)
    ended = None if eos is None else fin.gather(1, parents) | (tokens == eos) | none
    return best, parents, tokens, ended


def check(logits, scores, k=None, **kw):
    got, want = ops.beam_select(logits, scores, k, **kw), reference(logits, scores, k, **kw)
    again = ops.beam_select(logits, scores, k, **kw)
    for a, b in zip(got, again):
        assert (a is None and b is None) or torch.equal(a, b)
    assert got.scores.dtype == torch.float32 and got.parents.dtype == got.tokens.dtype == torch.int64
    assert torch.equal(got.parents, want[1]) and torch.equal(got.tokens, want[2]), (got, want)
    if want[3] is None:
        assert got.finished is None
    else:
        assert got.finished.dtype == torch.bool and torch.equal(got.finished, want[3])
    gone = want[0] == DEAD
    assert torch.equal(got.scores == DEAD, gone)
    err, room = (got.scores.double() - want[0])[~gone].abs(), OFF + want[0][~gone].abs() * 2.0**-24
    assert (err <= room).all(), (err - room).max()
    return got


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def some(B, W, V, dtype=torch.bfloat16, seed=0, spread=2.5):
    g = gen(seed)
    return (torch.randn(B, W, V, generator=g, device="cuda") * spread).to(dtype), -torch.rand(B, W, generator=g, device="cuda") * 3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 31, 64, 1016, 1017, 1023, 1024, 1025, 5003, 32000, 100003])
def test_vocabularies(V, dtype):
    for B, W, k in ((1, 1, 1), (2, 3, 3), (1, 4, 8), (3, 5, 2)):
        check(*some(B, W, V, dtype, V), k)


@pytest.mark.parametrize("W,k", [(1, 64), (64, 64), (64, 1), (33, 40), (16, 32), (2, 63), (7, 33)])
@pytest.mark.parametrize("V", [3, 700, 2048, 40000])
def test_beams_and_candidates(W, k, V):
    check(*some(2, W, V, seed=W + k), k)
    check(*some(2, W, V, torch.float32, seed=W + k), k)


@pytest.mark.parametrize("B,W,V", [(37, 8, 32001), (64, 4, 16384), (200, 2, 3000), (1, 16, 262144)])
def test_many_rows(B, W, V):
    """Enough for segments of several tiles."""
    check(*some(B, W, V), 2 * W)


def test_empty_batch_and_refusals():
    x, s = some(2, 3, 50)
    for r in (ops.beam_select(x[:0], s[:0]), ops.beam_select(x[:0], s[:0], 5, eos=1)):
        assert r.scores.shape[0] == r.parents.shape[0] == r.tokens.shape[0] == 0
    for bad, what in ((lambda: ops.beam_select(x[0], s), "shapes"), (lambda: ops.beam_select(x, s[:1]), "shapes"), (lambda: ops.beam_select(x, s, 0), "candidates"),
                      (lambda: ops.beam_select(x, s, 65), "candidates"), (lambda: ops.beam_select(*some(1, 65, 4)), "beams"), (lambda: ops.beam_select(x[..., :0], s), "vocabulary"),
                      (lambda: ops.beam_select(x.double(), s), "fp32, bf16"), (lambda: ops.beam_select(x, s.long()), "floating"), (lambda: ops.beam_select(x, s, temperature=0.0), "temperature"),
                      (lambda: ops.beam_select(x, s, temperature=float("nan")), "temperature"), (lambda: ops.beam_select(x, s, finished=s > 0), "eos"), (lambda: ops.beam_select(x, s, eos=50), "eos"),
                      (lambda: ops.beam_select(x, s, eos=-1), "eos"), (lambda: ops.beam_select(x, s, allowed=x), "truth"), (lambda: ops.beam_select(x, s, allowed=s[:, :2] > 0), "allowed"),
                      (lambda: ops.beam_select(x, s, finished=s, eos=1), "truth"), (lambda: ops.beam_select(x, s, penalty=s[:1]), "shapes"), (lambda: ops.beam_select(x, s.cpu()), "device")):
        with pytest.raises(ops.GdnError, match=what):
            bad()


LAYOUTS = {
    "one further": lambda x: torch.cat([x, x], 2)[..., 1:1 + x.shape[2]].copy_(x),
    "three further": lambda x: torch.cat([x, x], 2)[..., 3:3 + x.shape[2]].copy_(x),
    "every other": lambda x: torch.stack([x, -x], 3)[..., 0],
    "beams first": lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),
    "a slice of more": lambda x: torch.cat([x, x, x], 1)[:, x.shape[1]:2 * x.shape[1]],
    "negated": lambda x: torch._neg_view(-x),
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", sorted(LAYOUTS))
def test_layouts(layout, dtype):
    x, s = some(3, 4, 3001, dtype)
    y = LAYOUTS[layout](x)
    assert torch.equal(x, y)
    got, want = check(y, s, 8), check(x, s, 8)
    assert torch.equal(got.tokens, want.tokens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1019, 3001, 9001])
def test_every_place_of_a_row_in_memory(V, dtype):
    """Rows that begin and end at every distance from a 16-byte boundary, the largest logits at their ends."""
    for past in range(8):
        buffer = torch.full((2, 3, V + 16), 50.0, dtype=dtype, device="cuda")
        x = buffer[..., past:past + V]
        y, s = some(2, 3, V, dtype, past)
        x.copy_(y)
        x[..., 0], x[..., -1] = 9.0, 8.5
        check(x, s, 6)
        check(x, s, 6, allowed=torch.arange(V, device="cuda") % 3 != 1)


def test_one_row_for_all_beams():
    x, _ = some(2, 1, 5000)
    scores = torch.tensor([[0.0, DEAD, DEAD], [0.0, DEAD, DEAD]], device="cuda")
    check(x.expand(2, 3, 5000), scores, 3)
    check(x.expand(2, 3, 5000), torch.zeros(2, 3, device="cuda"), 7)                      # equal beams: the lowest first
    check(x[:1].expand(5, 3, 5000), -torch.rand(5, 3, generator=gen(), device="cuda"))


def test_rows_far_apart():
    """Beams whose logits lie more than 2^31 elements from one another."""
    V, apart = 3001, 2**31 + 8
    buffer = torch.empty(apart + V, dtype=torch.bfloat16, device="cuda")
    x = buffer.as_strided((1, 2, V), (1, apart, 1))
    y, s = some(1, 2, V)
    x.copy_(y)
    check(x, s, 6)
    check(x.transpose(0, 1), s.t(), 6)


# ---------------------------------------------------------------------------------------------------------------
# Equals, and what is nearly equal
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("W,k", [(1, 1), (1, 64), (3, 10), (8, 8)])
@pytest.mark.parametrize("V", [5, 1000, 9000, 40000])
def test_all_logits_equal(V, W, k):
    x = torch.zeros(2, W, V, dtype=torch.bfloat16, device="cuda")
    check(x, torch.zeros(2, W, device="cuda"), k)
    check(x, -torch.arange(W, device="cuda").float().expand(2, W), k)
    check(torch.where(torch.arange(V, device="cuda") % 2 == 0, 0.0, -0.0).expand(2, W, V).contiguous(), torch.zeros(2, W, device="cuda"), k)      # zeros of both signs


@pytest.mark.parametrize("levels", [2, 5, 40])
@pytest.mark.parametrize("V", [50, 3000, 30000])
def test_few_values(V, levels):
    for k in (4, 64):
        x = torch.randint(0, levels, (3, 4, V), generator=gen(V), device="cuda").to(torch.bfloat16)
        check(x, -torch.rand(3, 4, generator=gen(1), device="cuda"), k)


@pytest.mark.parametrize("k", [4, 40])
@pytest.mark.parametrize("down", [False, True])
def test_sorted_logits(down, k):
    """The largest side by side, in a lane's 16 bytes and in one segment."""
    x = torch.linspace(-9, 9, 20011, device="cuda")
    x = (x.flip(0) if down else x).expand(2, 3, 20011).contiguous()
    check(x, -torch.rand(2, 3, generator=gen(), device="cuda"), k)
    check(x.to(torch.bfloat16), -torch.rand(2, 3, generator=gen(), device="cuda"), k)


@pytest.mark.parametrize("k", [1, 2, 3, 6, 7, 12, 20])
@pytest.mark.parametrize("V", [900, 50021])
def test_beams_one_step_of_fp32_apart(V, k):
    """Rows that hold the same logits in other orders have the same sum of exponentials, so the scores alone order their candidates; sums in 32
    bits differ by more than the scores do."""
    g = gen(V)
    row = torch.randn(V, generator=g, device="cuda") * 2
    x = torch.stack([row, row[torch.randperm(V, generator=g, device="cuda")], row.flip(0), row.roll(5)])[None]
    for ulps in ((0, 1, 2, 3), (3, 0, 2, 1), (1, 3, 0, 2)):
        scores = torch.tensor([[-1.0 - 2.0**-23 * u for u in ulps]], device="cuda")
        order = torch.tensor(ulps, device="cuda").argsort()
        for y in (x, torch.cat([x, x], 2)[..., 3:3 + V].copy_(x)):
            got = ops.beam_select(y, scores, k)
            assert torch.equal(got.parents, order.repeat(5)[None, :k])
            for i, values in enumerate(x[0, got.parents[0], got.tokens[0]].split(4)):
                assert (values == row.sort(descending=True).values[i]).all()


@pytest.mark.parametrize("V", [5, 700, 40000])
def test_beams_that_are_all_but_sure(V):
    """One token of every beam has all but 1e-7 to 1e-13 of the probability, which is nothing beside one in 32 bits, and decides."""
    W = 12
    for seed in range(3):
        rest = -torch.rand(1, W, 1, generator=gen(seed), device="cuda") * 14 - 16 - math.log(V)
        x = rest + torch.rand(1, W, V, generator=gen(seed + 5), device="cuda")
        x.scatter_(2, torch.randint(0, V, (1, W, 1), generator=gen(seed + 9), device="cuda"), 1.0)
        for scores in (torch.zeros(1, W, device="cuda"), torch.full((1, W), -7.0, device="cuda")):
            check(x, scores, W)
            check(x, scores, 5, finished=torch.arange(W, device="cuda")[None] % 5 == 2, eos=0)
            check(x, scores, 20, penalty=torch.full((1, W), 1.7, device="cuda"))


def test_equals_behind_the_cut_hide_another_beams():
    """Many equals of one beam around the last candidate, and one of another beam that lies between them by less than the sums are known."""
    V = 4000
    x = torch.full((1, 2, V), -3.0, device="cuda")
    x[0, 0, :30] = 5.0
    x[0, 1] = x[0, 0].roll(777)                                            # the same logits
    for first in (0, 1):
        scores = torch.tensor([[-2.0, -2.0]], device="cuda")
        scores[0, 1 - first] -= 2.0**-22
        got = ops.beam_select(x, scores, 10)
        assert (got.parents == first).all() and torch.equal(got.tokens[0], torch.arange(10, device="cuda") + 777 * first)


# ---------------------------------------------------------------------------------------------------------------
# Masks, values that are not finite, beams that are not in use
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [40, 3001, 4096, 33000])
def test_masks(V, dtype):
    B, W = 3, 4
    x, s = some(B, W, V, dtype)
    for shape in ((V,), (1, 1, V), (B, 1, V), (W, V), (B, W, V), (B, W, 1), (1,), (B, 1, 1)):
        check(x, s, 6, allowed=torch.rand(shape, generator=gen(V), device="cuda") < 0.5)
    m = torch.rand(B, W, V + 5, generator=gen(1), device="cuda") < 0.1
    check(x, s, 6, allowed=m[..., 3:V + 3])
    check(x, s, 6, allowed=(torch.rand(B, W, 2 * V, generator=gen(2), device="cuda") < 0.3)[..., ::2])
    check(x[..., 1:], s, 6, allowed=m[..., :V - 1])


@pytest.mark.parametrize("temperature", [1.0, 0.9, 1.7])
def test_masks_that_leave_one_token(temperature):
    """Whose log probability is zero, so that the scores decide, and among equal ones the beam."""
    x, _ = some(2, 9, 700, torch.float32)
    m = torch.zeros(2, 9, 700, dtype=torch.bool, device="cuda").scatter_(2, torch.randint(0, 700, (2, 9, 1), generator=gen(8), device="cuda"), True)
    for scores in (torch.zeros(2, 9, device="cuda"), torch.full((2, 9), -3.7, device="cuda"), -torch.arange(9, device="cuda").float().div(3).floor().expand(2, 9)):
        got = check(x, scores, 9, allowed=m, temperature=temperature)
        assert torch.equal(got.scores, scores) and torch.equal(got.parents[0], torch.arange(9, device="cuda"))


def test_masks_that_leave_little_or_nothing():
    x, s = some(2, 3, 5000)
    m = torch.zeros(2, 3, 5000, dtype=torch.bool, device="cuda")
    for eos in (None, 7):
        check(x, s, 5, allowed=m, eos=eos)
        m[0, 1, 4999] = True
        check(x, s, 5, allowed=m, eos=eos)
        m[0, 2, 10:13] = True
        m[1, 0, :40] = True
        got = check(x, s, 12, allowed=m, eos=eos)
        assert (got.scores[0, 4:] == DEAD).all() and (got.tokens[0, 4:] == (eos or 0)).all()
        m.zero_()


def test_values_that_are_not_finite():
    x, s = some(4, 3, 9000, torch.float32)
    m = torch.rand(4, 3, 9000, generator=gen(3), device="cuda") < 0.5
    y = x.clone()
    y[~m] = torch.tensor([float("nan"), math.inf, DEAD, 3e38], device="cuda").repeat(m.numel())[:int((~m).sum())]
    got, want = check(y, s, 6, allowed=m), check(x, s, 6, allowed=m)                      # behind the mask nothing is seen
    assert torch.equal(got.scores, want.scores)
    for bad in (float("nan"), math.inf):
        y = x.clone()
        y[0, 0, 8999] = bad                                                               # a beam without a distribution
        y[1, :, 17] = bad
        y[2, 2] = bad
        got = check(y, s, 6, eos=3)
        assert (got.scores[1] == DEAD).all() and got.finished[1].all()
    y = x.clone()
    y[0, 0], y[1, :, 50:], y[2, 1, ::2] = DEAD, DEAD, DEAD
    check(y, s, 6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_lowest_and_largest_values(dtype):
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x, s = some(2, 3, 3000, dtype)
    y = x.masked_fill(torch.rand(2, 3, 3000, generator=gen(4), device="cuda") < 0.7, low)      # a mask of the type's lowest value
    check(y, s, 9)
    check(torch.full_like(x, low), s, 9)                                                  # every token as likely as another
    check(torch.full_like(x, high), s, 9)
    y = x.clone()
    y[..., 5], y[..., 6] = high, low
    check(y, s, 3)


def test_beams_that_are_not_in_use():
    x, s = some(5, 4, 700)
    s[0, 1:], s[1, 0], s[2], s[3, 3] = DEAD, float("nan"), DEAD, math.inf
    check(x, s, 6)
    pen = torch.rand(5, 4, generator=gen(5), device="cuda") + 0.5
    pen[0, 0], pen[1, 1], pen[3, 0], pen[4, 2] = 0.0, -1.0, float("nan"), math.inf
    check(x, s, 6, penalty=pen)
    x[:, 0] = float("nan")                                                                # a beam that is not in use may hold anything
    s[:, 0] = DEAD
    check(x, s, 6)


def test_finished_beams():
    x, s = some(6, 4, 2500)
    fin = torch.rand(6, 4, generator=gen(6), device="cuda") < 0.4
    fin[0], fin[1] = True, False
    x[fin] = float("nan")                                                                 # not read
    for k in (1, 4, 10):
        got = check(x, s, k, finished=fin, eos=2499)
        assert got.finished[0].all()
        check(x, s, k, finished=fin, eos=0, penalty=torch.rand(6, 4, generator=gen(7), device="cuda") + 0.3)
    s[0, 2] = DEAD
    check(x, s, 5, finished=fin, eos=1)
    check(x, s, 4, eos=1)


@pytest.mark.parametrize("temperature", [1e-6, 0.01, 0.7, 1.5, 50.0, 1e6])
def test_temperatures(temperature):
    for dtype in (torch.bfloat16, torch.float32):
        x, s = some(2, 4, 6000, dtype)
        check(x, s, 8, temperature=temperature)
        check(x, s, 8, temperature=temperature, finished=s < -2, eos=9, penalty=1.0 - s, allowed=x > -1)


def test_other_types_of_scores_and_gradients():
    x, s = some(2, 3, 400)
    got = ops.beam_select(x.clone().requires_grad_(True), s.clone().requires_grad_(True), 4)
    assert not got.scores.requires_grad
    h = s.bfloat16()
    check(x, h, 4)
    assert torch.equal(ops.beam_select(x, h, 4).scores, ops.beam_select(x, h.float(), 4).scores)


# ---------------------------------------------------------------------------------------------------------------
# Streams, graphs, traces
# ---------------------------------------------------------------------------------------------------------------
def test_two_streams_at_once():
    sets = [some(4, 8, 60000, seed=i) for i in range(4)]
    want = [ops.beam_select(*a) for a in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[] for _ in sets]
    for _, (i, st) in itertools.product(range(5), enumerate(streams)):
        with torch.cuda.stream(st):
            got[i].append(ops.beam_select(*sets[i]))
    torch.cuda.synchronize()
    for w, many in zip(want, got):
        for g in many:
            assert torch.equal(g.scores, w.scores) and torch.equal(g.tokens, w.tokens) and torch.equal(g.parents, w.parents)


def test_captured_and_replayed():
    x, s = some(3, 4, 30000)
    fin = torch.zeros(3, 4, dtype=torch.bool, device="cuda")
    ops.beam_select(x, s, 8, finished=fin, eos=3)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for k in (8, 5):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.beam_select(x, s, k, finished=fin, eos=3))
        graphs.append(g)
    for seed in range(4):
        y, t = some(3, 4, 30000, seed=seed + 10)
        x.copy_(y), s.copy_(t), fin.copy_(t < -1.5)
        for g in graphs:
            g.replay()
        for k, o in zip((8, 5), outs):
            for a, b in zip(o, ops.beam_select(x, s, k, finished=fin, eos=3)):
                assert torch.equal(a, b)


def test_traced():
    x, s = some(2, 3, 900)
    m = x > -1
    for f, inputs in ((lambda x, s: ops.beam_select(x, s, 5)[:3], (x, s)), (lambda x, s, m: tuple(ops.beam_select(x, s, 4, allowed=m, finished=s < -2, eos=1, penalty=2 - s)), (x, s, m))):
        traced = torch.jit.trace(f, inputs, check_trace=False)
        y, t = some(2, 3, 900, seed=5)
        other = (y, t, y > -1)[:len(inputs)]
        for a, b in zip(traced(*other), f(*other)):
            assert torch.equal(a, b)
