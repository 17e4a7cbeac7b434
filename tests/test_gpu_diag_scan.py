"""GPU: the element-wise gated recurrence, its backward and its one-token form against the token loop in fp64.

Tolerances count roundings (half a step, 2^-24 relative in fp32, of the absolute recurrence: the same with |x|, |h0|, which
bounds every partial sum).  On its way a value passes at most 8 tokens of a thread and 16 groups of a tile, twice, two roundings
each, 2 x 16 for every tile that its state crosses, and 20 for coefficients (a decay's error counts once per memory length):
k = 120 + 34 tiles.  Results are then rounded once to their type."""
import pytest
import torch

from lethe_b200 import ops

pytestmark = pytest.mark.gpu

TILE = 128
U = 2.0 ** -24
TYPES = {"f32": (torch.float32, torch.float32), "bf16": (torch.bfloat16, torch.float32), "f16": (torch.float16, torch.float32),
         "bf16 g": (torch.bfloat16, torch.bfloat16), "f16 g": (torch.float16, torch.float16)}


def loop(x, g, h0, complement, dh=None, dhT=None):
    """The definition, token by token in fp64, and its derivatives; the same of absolute values for the bounds."""
    x, g = x.double(), g.double()
    a = g.exp()
    u = -torch.expm1(g) * x if complement else x
    h, ha = h0.double(), h0.double().abs()
    hs, has = [h], [ha]
    for t in range(x.shape[1]):
        h, ha = a[:, t] * h + u[:, t], a[:, t] * ha + u[:, t].abs()
        hs.append(h)
        has.append(ha)
    out = {"h": torch.stack(hs[1:], 1) if x.shape[1] else x, "hT": h}
    mag = {"h": torch.stack(has[1:], 1) if x.shape[1] else x, "hT": ha}
    if dh is None:
        return out, mag
    e, ea = dhT.double(), dhT.double().abs()
    dx, dg, mx, mg = (torch.empty_like(x) for _ in range(4))
    for t in reversed(range(x.shape[1])):
        d, da = dh[:, t].double() + e, dh[:, t].double().abs() + ea
        keep = -torch.expm1(g[:, t]) if complement else torch.ones_like(d)
        dx[:, t], mx[:, t] = d * keep, da * keep
        e, ea = a[:, t] * d, a[:, t] * da
        back = hs[t] - x[:, t] if complement else hs[t]
        dg[:, t], mg[:, t] = e * back, ea * (has[t] + (x[:, t].abs() if complement else 0))
    out.update(dx=dx, dg=dg, dh0=e)
    mag.update(dx=mx, dg=mg, dh0=ea)
    return out, mag


def close(got, want, mag, tiles, factor=1):
    """`factor`: 2 for a product of two such values."""
    k = factor * (120 + 34 * tiles)
    step = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    err = (got.double() - want).abs()
    tol = step * want.abs() + k * U * mag * (1 + step) + tiny
    bad = err > tol
    assert got.shape == want.shape and not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()}, worst {float((err / tol).max()):.2f} of the bound"


def make(B, L, inner, types="bf16", gates="mild", seed=1, dev="cuda"):
    xt, gt = TYPES[types]
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(B, L, *inner, generator=gen).to(xt)
    if gates == "mild":
        g = -0.1 * torch.rand(B, L, *inner, generator=gen)
    elif gates == "strong":
        g = -torch.nn.functional.softplus(torch.randn(B, L, *inner, generator=gen) + 3)
    elif gates == "long":
        g = -1e-4 * torch.rand(B, L, *inner, generator=gen)
    else:   # all kinds: none, whole, beyond what fp32 holds, resets, both sides of where the form changes
        kinds = torch.tensor([0.0, -0.0, -1e-30, -1e-6, -0.2499, -0.25, -0.2501, -3.0, -30.0, -120.0, float("-inf")])
        g = kinds[torch.randint(0, len(kinds), (B, L, *inner), generator=gen)]
    h0 = torch.randn(B, *inner, generator=gen)
    dh = torch.randn(B, L, *inner, generator=gen).to(xt)
    dhT = torch.randn(B, *inner, generator=gen)
    return [t.to(dev) for t in (x, g.to(gt), h0, dh, dhT)]


def run(x, g, h0, dh, dhT, complement):
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, g, h0)]
    h, hT = ops.diag_scan(*leaves, complement=complement)
    dx, dg, dh0 = torch.autograd.grad((h, hT), leaves, (dh, dhT))
    return {"h": h.detach(), "hT": hT.detach(), "dx": dx, "dg": dg, "dh0": dh0}


def check(x, g, h0, dh, dhT, complement):
    got = run(x, g, h0, dh, dhT, complement)
    want, mag = loop(x, g, h0, complement, dh, dhT)
    tiles = -(-x.shape[1] // TILE)
    for n in want:
        assert got[n].dtype == {"h": x, "hT": h0, "dx": x, "dg": g, "dh0": h0}[n].dtype
        close(got[n], want[n], mag[n], tiles, 2 if n == "dg" else 1)
    return got


@pytest.mark.parametrize("complement", [False, True])
@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("B,L,inner", [(2, 300, (72,)), (1, 128, (64,)), (3, 129, (33,)), (1, 1, (1,)), (2, 127, (2, 130))])
def test_against_the_token_loop(types, B, L, inner, complement):
    check(*make(B, L, inner, types), complement)


@pytest.mark.parametrize("complement", [False, True])
@pytest.mark.parametrize("gates", ["strong", "long", "kinds"])
def test_decays(gates, complement):
    check(*make(2, 700, (96,), "f32", gates), complement)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("complement", [False, True])
@pytest.mark.parametrize("B,L,inner", [(400, 10, (8,)), (2, 5000, (264,)), (3, 1100, (1040,)), (350, 200, (72,)), (5, 4100, (6, 40))])
def test_more_tiles_than_the_gpu_holds(types, complement, B, L, inner):
    """Copies of whole tiles, and CTAs that do several of them."""
    check(*make(B, L, inner, types, "kinds"), complement)


@pytest.mark.parametrize("L", [2, 7, 8, 9, 255, 256, 257, 2048, 5000])
def test_lengths(L):
    check(*make(1, L, (68,), "bf16", seed=L), False)


def test_a_long_memory_keeps_its_precision():
    """4096 tokens at a constant decay next to one: exp(g) in fp32 is off by 2^-25 to one side, over this memory by 1e-4 of the state."""
    x, g, h0, dh, dhT = make(1, 4096, (64,), "f32")
    g = torch.full_like(g, -1.3e-5)
    x, dh = x.abs(), dh.abs()
    got = check(x, g, h0, dh, dhT, False)
    want, _ = loop(x, g, h0, False, dh, dhT)
    for n in want:
        assert float((got[n].double() - want[n]).norm() / want[n].norm()) < 2e-6


def test_gradients_against_differences():
    x, g, h0, dh, dhT = make(1, 20, (3,), "f32", seed=5)
    got = run(x, g, h0, dh, dhT, True)

    def loss(x, g, h0):
        out, _ = loop(x, g, h0, True)
        return (out["h"] * dh.double()).sum() + (out["hT"] * dhT.double()).sum()
    ins = [t.double() for t in (x, g, h0)]
    for i, n in enumerate(("dx", "dg", "dh0")):
        flat = ins[i].reshape(-1)
        for j in range(0, flat.numel(), 7):
            up, down = flat.clone(), flat.clone()
            up[j] += 1e-5
            down[j] -= 1e-5
            args = [t if k != i else None for k, t in enumerate(ins)]
            d = (loss(*[t if t is not None else up.view_as(ins[i]) for t in args]) - loss(*[t if t is not None else down.view_as(ins[i]) for t in args])) / 2e-5
            assert abs(float(d) - float(got[n].reshape(-1)[j])) <= 1e-5 * max(1.0, abs(float(d)))


def test_strided_inputs_are_read_where_they_lie():
    """Slices of a fused projection, a transposed batch, broadcast batches and channels, an odd start."""
    x, g, h0, dh, dhT = make(2, 200, (72,))
    want = run(x, g, h0, dh, dhT, True)
    proj = torch.zeros(2, 200, 200, dtype=x.dtype, device="cuda")
    for at in (8, 3):
        proj[..., at:at + 72] = x
        wide = torch.zeros(200, 2, 80, device="cuda")
        wide[..., 4:76] = g.transpose(0, 1)
        got = {}
        xv, gv = proj[..., at:at + 72].detach().requires_grad_(True), wide[..., 4:76].transpose(0, 1).detach().requires_grad_(True)
        hv = h0.clone().requires_grad_(True)
        h, hT = ops.diag_scan(xv, gv, hv, complement=True)
        dhv = torch.zeros(200, 2, 72, dtype=dh.dtype, device="cuda").transpose(0, 1).copy_(dh)
        got["dx"], got["dg"], got["dh0"] = torch.autograd.grad((h, hT), (xv, gv, hv), (dhv, dhT))
        got["h"], got["hT"] = h, hT
        for n in want:
            assert torch.equal(got[n], want[n]), (n, at)
    one = g[:1, :, :1].contiguous().requires_grad_(True)
    h, hT = ops.diag_scan(x, one.expand_as(g), h0)
    full = one.detach().expand_as(g).contiguous()
    assert torch.equal(h, ops.diag_scan(x, full, h0)[0])
    dg, = torch.autograd.grad((h, hT), one, (dh, dhT))
    each = run(x, full, h0, dh, dhT, False)["dg"]
    assert torch.allclose(dg, each.sum((0, 2), keepdim=True), rtol=1e-4, atol=1e-3)      # (torch's sum over 144 values)


@pytest.mark.parametrize("types", ["f32", "bf16", "f16 g"])
@pytest.mark.parametrize("B,L,D", [(2, 300, 32), (5, 257, 8), (17, 130, 4), (7, 1000, 24), (3, 64, 28), (40, 500, 12), (900, 40, 16), (2, 2000, 20)])
def test_few_channels_of_many_sequences(types, B, L, D):
    """Batches side by side in a strip, the last strip not full."""
    check(*make(B, L, (D,), types, "kinds"), True)
    x, g, h0, dh, dhT = make(B, L, (D,), types)
    proj = torch.zeros(B, L + 3, 2 * D + 8, dtype=x.dtype, device="cuda")       # another stride for every tensor
    proj[:, 2:L + 2, 8:D + 8] = x
    want, got = run(x, g, h0, dh, dhT, False), {}
    leaves = [proj[:, 2:L + 2, 8:D + 8].detach().requires_grad_(True), g.transpose(0, 1).contiguous().transpose(0, 1).requires_grad_(True), h0.clone().requires_grad_(True)]
    h, hT = ops.diag_scan(*leaves)
    got.update(h=h, hT=hT, **dict(zip(("dx", "dg", "dh0"), torch.autograd.grad((h, hT), leaves, (dh, dhT)))))
    assert all(torch.equal(got[n], want[n]) for n in want)
    # a sequence by itself gives the bits that it has among others
    one = run(x[1:2], g[1:2], h0[1:2], dh[1:2], dhT[1:2], False)
    assert all(torch.equal(one[n], want[n][1:2]) for n in want)


def test_offsets_beyond_32_bits():
    big = torch.empty(3 * (1 << 30) + 64, dtype=torch.bfloat16, device="cuda")
    x, g, h0, dh, dhT = make(1, 3, (64,))
    far = big.as_strided((1, 3, 64), (0, (1 << 30) + 24, 1))
    far.copy_(x)
    want = ops.diag_scan(x, g, h0)
    got = ops.diag_scan(far, g, h0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_no_tokens_no_channels_no_sequences():
    for shape in ((2, 0, 5), (0, 4, 5), (2, 4, 0)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        g = torch.zeros(shape, device="cuda", requires_grad=True)
        h0 = torch.randn(shape[0], shape[2], device="cuda", requires_grad=True)
        h, hT = ops.diag_scan(x, g, h0)
        assert h.shape == x.shape and torch.equal(hT, h0)
        dhT = torch.randn_like(h0)
        dx, dg, dh0 = torch.autograd.grad(hT, (x, g, h0), dhT, allow_unused=True)
        assert torch.equal(dh0, dhT)
        assert ops.diag_scan(x, g)[1].abs().sum() == 0


def test_partial_gradients():
    x, g, h0, dh, dhT = make(2, 150, (40,), "f32")
    full = run(x, g, h0, dh, torch.zeros_like(dhT), False)
    for n, t in (("dx", 0), ("dg", 1), ("dh0", 2)):
        ins = [x, g, h0]
        ins[t] = ins[t].clone().requires_grad_(True)
        h, _ = ops.diag_scan(*ins)
        assert torch.equal(torch.autograd.grad(h, ins[t], dh)[0], full[n])
    only = run(x, g, h0, torch.zeros_like(dh), dhT, False)
    ins = [t.clone().requires_grad_(True) for t in (x, g, h0)]
    for n, a in zip(("dx", "dg", "dh0"), torch.autograd.grad(ops.diag_scan(*ins)[1], ins, dhT)):
        assert torch.equal(a, only[n])
    # no initial state
    a, b = ops.diag_scan(x, g), ops.diag_scan(x, g, torch.zeros_like(h0))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_a_reset_forgets_the_tokens_before():
    x, g, h0, dh, dhT = make(1, 400, (64,), "f32")
    for cut in (1, 128, 200, 399):
        gi = g.clone()
        gi[:, cut] = float("-inf")
        whole = run(x, gi, h0, dh, dhT, False)
        back = run(x[:, cut:], g[:, cut:].clone().index_fill_(1, torch.tensor([0], device="cuda"), float("-inf")), torch.zeros_like(h0), dh[:, cut:], dhT, False)
        front = run(x[:, :cut], g[:, :cut], h0, dh[:, :cut], torch.zeros_like(dhT), False)
        for n in ("h", "dx", "dg"):
            # the pieces have other tiles than the whole, so other roundings
            assert torch.allclose(whole[n][:, cut:], back[n], rtol=1e-5, atol=1e-5) and torch.allclose(whole[n][:, :cut], front[n], rtol=1e-5, atol=1e-5)
        assert bool((whole["dg"][:, cut] == 0).all())


def test_what_is_not_finite_stays_in_its_channel():
    x, g, h0, dh, dhT = make(2, 700, (70,), "f32")
    want = run(x, g, h0, dh, dhT, True)
    for bad in (float("nan"), float("inf")):
        xb, db = x.clone(), dh.clone()
        xb[1, 300, 7] = bad
        db[0, 400, 65] = bad
        got = run(xb, g, h0, db, dhT, True)
        clean = torch.ones(2, 70, dtype=torch.bool, device="cuda")
        clean[1, 7] = clean[0, 65] = False
        for n in ("h", "dx", "dg"):
            assert torch.equal(got[n].transpose(1, 2)[clean], want[n].transpose(1, 2)[clean]), n
        for n in ("hT", "dh0"):
            assert torch.equal(got[n][clean], want[n][clean]), n
        assert torch.equal(got["h"][1, :300, 7], want["h"][1, :300, 7]) and not bool(got["h"][1, 300:, 7].isfinite().any())
        assert torch.equal(got["dx"][0, 401:, 65], want["dx"][0, 401:, 65]) and not bool(got["dx"][0, :401, 65].isfinite().any())


def test_padding_leaves_the_state():
    """x = 0 and g = 0 behind a sequence's end; with the complement any x."""
    x, g, h0, _, _ = make(1, 500, (64,), "bf16")
    for complement in (False, True):
        for end in (1, 130, 384, 499):
            xp, gp = x.clone(), g.clone()
            gp[:, end:] = 0
            if not complement:
                xp[:, end:] = 0
            h, hT = ops.diag_scan(xp, gp, h0, complement=complement)
            # as many tokens, so the same tiles
            assert torch.equal(h[:, :end], ops.diag_scan(x, g, h0, complement=complement)[0][:, :end])
            assert torch.equal(hT.to(h.dtype), h[:, -1]) and float((h[:, end - 1].float() - hT).abs().max()) <= 2 ** -7 * float(hT.abs().max())


def test_long_and_many():
    """Groups of groups of tiles, and more sequences than 65535."""
    x, g, h0, dh, dhT = make(1, 20000, (8,), "f32", "long")
    check(x, g, h0, dh, dhT, False)
    check(*make(70000, 2, (3,), "bf16", "kinds"), True)


def test_two_runs_and_captured_replays_give_the_same_bits():
    x, g, h0, dh, dhT = make(2, 3000, (200,))
    want = run(x, g, h0, dh, dhT, True)
    for _ in range(3):
        again = run(x, g, h0, dh, dhT, True)
        assert all(torch.equal(again[n], want[n]) for n in want)
    graphs = []
    for _ in range(2):                       # two captured steps at once, each with its own workspace
        leaves = [t.clone().requires_grad_(True) for t in (x, g, h0)]
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            torch.autograd.grad(ops.diag_scan(*leaves, complement=True), leaves, (dh, dhT))
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            h, hT = ops.diag_scan(*leaves, complement=True)
            grads = torch.autograd.grad((h, hT), leaves, (dh, dhT))
        graphs.append((graph, s, dict(zip(("h", "hT", "dx", "dg", "dh0"), (h, hT, *grads)))))
    for _ in range(3):
        for graph, s, _ in graphs:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out in graphs:
        assert all(torch.equal(out[n], want[n]) for n in want)


def test_another_stream():
    x, g, h0, dh, dhT = make(2, 1000, (128,))
    want = run(x, g, h0, dh, dhT, False)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(x, g, h0, dh, dhT, False)
    s.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("complement", [False, True])
@pytest.mark.parametrize("B,inner", [(1, (1,)), (3, (130,)), (2, (8, 64)), (70000, (3,)), (5, (1025,))])
def test_step_is_a_token_of_the_scan(types, complement, B, inner):
    x, g, state, _, _ = make(B, 2, inner, types, "kinds")
    want, wT = ops.diag_scan(x[:, :1], g[:, :1], state, complement=complement)
    mine = state.clone()
    h = ops.diag_scan_step(x[:, 0], g[:, 0], mine, complement=complement)
    assert torch.equal(h, want[:, 0]) and torch.equal(mine, wT)


def test_step_reads_a_view_of_the_state_before_it_is_written():
    state = torch.randn(4, 64, device="cuda")
    g = -torch.rand(4, 64, device="cuda")
    want = state.clone()
    a = ops.diag_scan_step(state.clone().flip(0), g, want)
    aliased = state.clone()
    b = ops.diag_scan_step(aliased.as_strided((4, 64), (64, 1)), g, aliased)
    assert torch.equal(b, ops.diag_scan_step(state.clone(), g, state.clone()))
    assert a.shape == b.shape


def test_a_prompt_and_steps_go_on_where_it_ended():
    x, g, h0, _, _ = make(2, 140, (64,), "f32")
    h, hT = ops.diag_scan(x, g, h0)
    _, state = ops.diag_scan(x[:, :130], g[:, :130], h0)
    for t in range(130, 140):
        o = ops.diag_scan_step(x[:, t], g[:, t], state)
        # 2 roundings a token here, and those of another tiling there
        assert torch.allclose(o, h[:, t], rtol=0, atol=float(200 * U * h.abs().max()))
    assert torch.allclose(state, hT, rtol=0, atol=float(200 * U * h.abs().max()))


def test_refusals():
    x, g, h0, _, _ = make(2, 10, (16,))
    for bad, what in (((x[:, :, :8], g, h0), "shapes"), ((x, g, h0[:1]), "shapes"), ((x.double(), g, h0), "fp32, bf16 or fp16"),
                      ((x, g.int(), h0), "floating"), ((x, g, h0.int()), "floating"), ((x[:, 0], g[:, 0], h0), "shapes")):
        with pytest.raises(ops.GdnError, match=what):
            ops.diag_scan(*bad)
    for bad, what in (((x[:, 0], g[:, 0], h0.half()), "fp32"), ((x[:, 0], g[:, 0], h0.t().contiguous().t()), "contiguous"),
                      ((x[:, 0], g[:, :1], h0), "shapes"), ((x[:, 0], g[:, 0], h0.clone().requires_grad_(True)), "gradient")):
        with pytest.raises(ops.GdnError, match=what):
            ops.diag_scan_step(*bad)
    leaf = x.clone().requires_grad_(True)
    h, _ = ops.diag_scan(leaf, g, h0)
    torch.autograd.grad(h, leaf, torch.ones_like(h))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(h, leaf, torch.ones_like(h))
    h, _ = ops.diag_scan(leaf, g, h0)
    d, = torch.autograd.grad(h, leaf, torch.ones_like(h).requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        d.sum().backward()
