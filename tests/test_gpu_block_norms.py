"""GPU: the norms in front of and behind a block against their formulas in fp64.

Tolerances count roundings (half a step, 2^-24 relative in fp32).  A row sum passes at most 16 values of a thread, 5 butterflies
and 16 warps: 40 roundings, 20 on the root; the root, the logistic function (exponential, sum, quotient) and the products add
some 20: 60 in all, of the sum of the absolute values of the terms where terms can cancel.  A sum over rows adds one per row.  Results are rounded once to their type."""
import pytest
import torch

from lethe_b200 import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
K = 60
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def close(got, want, mag, k=K):
    """Within half a step of the result's type and k roundings of `mag`, the sum of the absolute values of the terms."""
    fi = torch.finfo(got.dtype)
    err = (got.double() - want).abs()
    tol = fi.eps / 2 * want.abs() + k * U * mag * (1 + fi.eps / 2) + fi.tiny * fi.eps
    bad = err > tol
    assert got.shape == want.shape and not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()}, worst {float((err / tol).max()):.2f} of the bound"


def rms(x, eps):
    inv = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    return x * inv, inv


def back(d, da, n, inv):
    """Gradient through a norm, and the size of its terms."""
    return inv * (d - n * (d * n).mean(-1, keepdim=True)), inv * (da + n.abs() * (da * n.abs()).mean(-1, keepdim=True))


def rows_sum(t):
    return t.reshape(-1, t.shape[-1]).sum(0)


def randn(*shape, seed=0, dt=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to("cuda", dt)


# ---------------------------------------------------------------------------------------------
def gated_ref(x, z, w, dy, eps, act):
    x, z, w, dy = (t.double() for t in (x, z, w, dy))
    n, inv = rms(x, eps)
    s = torch.sigmoid(z)
    a, slope, bound = (z * s, s * (1 + z * (1 - s)), s * (1 + z.abs() * (1 - s))) if act == "silu" else (s, s * (1 - s), s)
    want, mag = {"y": n * w * a}, {"y": (n * w * a).abs()}
    d = dy * w * a
    want["dx"], mag["dx"] = back(d, d.abs(), n, inv)
    want["dgate"], mag["dgate"] = dy * n * w * slope, (dy * n * w).abs() * bound
    want["dweight"], mag["dweight"] = rows_sum(dy * n * a), rows_sum((dy * n * a).abs())
    return want, mag


def gated_check(x, z, w, dy, eps=1e-6, act="silu"):
    leaves = [t.detach().requires_grad_(True) for t in (x, z, w)]
    y = ops.gated_norm(*leaves, eps=eps, activation=act)
    got = dict(zip(("y", "dx", "dgate", "dweight"), (y.detach(), *torch.autograd.grad(y, leaves, dy))))
    want, mag = gated_ref(x, z, w, dy, eps, act)
    rows = x.numel() // x.shape[-1]
    for n in want:
        assert got[n].dtype == (w if n == "dweight" else x).dtype
        close(got[n], want[n], mag[n], K + (rows if n == "dweight" else 0))
    return got


@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("types", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("shape", [(2, 37, 3, 64), (1, 5, 2, 128), (3, 1), (2, 3, 40), (7, 33), (260, 100)])
def test_gated_norm(types, shape, act):
    xt, wt = (DT[t] for t in types)
    gated_check(randn(*shape, seed=1, dt=xt), 3 * randn(*shape, seed=2).to(xt), randn(shape[-1], seed=3, dt=wt), randn(*shape, seed=4, dt=xt), act=act)


@pytest.mark.parametrize("D", [8, 63, 65, 72, 129, 256, 257, 264, 511, 512, 520, 1000, 1023, 1024, 1032, 2047, 2048, 2056, 4095, 4096, 4104, 8191, 8192])
def test_gated_norm_row_lengths(D):
    gated_check(randn(5, D, seed=D, dt=torch.bfloat16), randn(5, D, seed=D + 1, dt=torch.bfloat16), randn(D, seed=3), randn(5, D, seed=4, dt=torch.bfloat16))


@pytest.mark.parametrize("rows,D", [(1, 64), (4097, 64), (70001, 16), (1501, 2048), (700, 8192)])
def test_gated_norm_many_rows(rows, D):
    got = gated_check(randn(rows, D, seed=1, dt=torch.bfloat16), randn(rows, D, seed=2, dt=torch.bfloat16), randn(D, seed=3), randn(rows, D, seed=4, dt=torch.bfloat16))
    again = gated_check(randn(rows, D, seed=1, dt=torch.bfloat16), randn(rows, D, seed=2, dt=torch.bfloat16), randn(D, seed=3), randn(rows, D, seed=4, dt=torch.bfloat16))
    assert all(torch.equal(got[n], again[n]) for n in got)


def test_gated_norm_zero_rows_and_far_gates():
    x, z, w, dy = (randn(6, 64, seed=i) for i in range(4))
    w = w[0]
    x[0] = 0
    x[1] = 1e-15
    x[2] = 1e15
    z[3], z[4] = 80.0, -80.0
    z[5, ::2], z[5, 1::2] = 300.0, -300.0
    leaves = [t.requires_grad_(True) for t in (x, z, w)]
    y = ops.gated_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    assert all(bool(t.isfinite().all()) for t in (y, *grads))
    want, _ = gated_ref(x.detach(), z.detach(), w.detach(), dy, 1e-6, "silu")
    assert bool((y[0] == 0).all()) and torch.allclose(y.double(), want["y"], rtol=1e-5, atol=1e-30)
    assert torch.allclose(grads[0].double()[:3], want["dx"][:3], rtol=1e-4, atol=1e-4 * float(want["dx"][0].abs().max()))


def test_gated_norm_reads_views_where_they_lie():
    x, z, w, dy = randn(2, 30, 4, 64, seed=1, dt=torch.bfloat16), randn(2, 30, 4, 64, seed=2, dt=torch.bfloat16), randn(64, seed=3), randn(2, 30, 4, 64, seed=4, dt=torch.bfloat16)
    want = gated_check(x, z, w, dy)
    for at in (0, 8, 5):                                  # whole pieces, and a start between them
        proj = torch.full((2, 30, 600), 7.0, dtype=x.dtype, device="cuda")
        zv = proj[..., at:at + 256].unflatten(-1, (4, 64))
        zv.copy_(z)
        xv = torch.empty(30, 2, 4, 64, dtype=x.dtype, device="cuda").transpose(0, 1).copy_(x)       # no two strides: copied
        got = gated_check(xv, zv, w, dy.transpose(1, 2).contiguous().transpose(1, 2))
        if at % 8 == 0:                                   # (element by element the sums have another order)
            assert all(torch.equal(got[n], want[n]) for n in want)
    # a gradient that is a broadcast number
    leaves = [t.clone().requires_grad_(True) for t in (x, z, w)]
    a = torch.autograd.grad(ops.gated_norm(*leaves).sum(), leaves)
    b = torch.autograd.grad(ops.gated_norm(*leaves), leaves, torch.ones_like(x))
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    # one gate for all heads
    one = z[:, :, :1].clone().requires_grad_(True)
    y = ops.gated_norm(x, one.expand_as(x), w)
    d, = torch.autograd.grad(y, one, dy)
    each = gated_check(x, one.detach().expand_as(x).contiguous(), w, dy)["dgate"]
    assert d.shape == one.shape and torch.allclose(d.float(), each.float().sum(2, keepdim=True), rtol=2 ** -6, atol=2 ** -5)


# ---------------------------------------------------------------------------------------------
def residual_ref(x, res, w, scale, pw, dy, dr, eps, r_kept):
    x, w, dy, dr = (t.double() for t in (x, w, dy, dr))
    sc = scale.double() if isinstance(scale, torch.Tensor) else 1.0 if scale is None else scale
    t, n1 = x, None
    if pw is not None:
        n1, inv1 = rms(x, eps)
        t = n1 * pw.double()
    res = torch.zeros_like(x) if res is None else res.double()
    want, mag = {"r": res + sc * t}, {"r": res.abs() + (sc * t).abs()}
    n2, inv2 = rms(r_kept.double(), eps)
    want["y"], mag["y"] = n2 * w, (n2 * w).abs()
    d, da = back(dy * w, (dy * w).abs(), n2, inv2)
    d, da = d + dr, da + dr.abs()
    want["dresidual"], mag["dresidual"] = d, da
    want["dweight"], mag["dweight"] = rows_sum(dy * n2), rows_sum((dy * n2).abs())
    want["dscale"], mag["dscale"] = rows_sum(d * t), rows_sum(da * t.abs())
    if pw is None:
        want["dx"], mag["dx"] = d * sc, da * (sc.abs() if isinstance(sc, torch.Tensor) else abs(sc))
    else:
        u, ua = d * sc, da * (sc.abs() if isinstance(sc, torch.Tensor) else abs(sc))
        want["dx"], mag["dx"] = back(u * pw.double(), ua * pw.double().abs(), n1, inv1)
        want["dpost_weight"], mag["dpost_weight"] = rows_sum(u * n1), rows_sum(ua * n1.abs())
    return want, mag


def residual_check(x, res, w, scale, pw, dy, dr, eps=1e-6):
    named = {"x": x, "residual": res, "weight": w, "scale": scale, "post_weight": pw}
    leaves = {n: t.detach().requires_grad_(True) for n, t in named.items() if isinstance(t, torch.Tensor)}
    a = {**named, **leaves}
    y, r = ops.residual_norm(a["x"], a["residual"], a["weight"], scale=a["scale"], post_weight=a["post_weight"], eps=eps)
    grads = torch.autograd.grad((y, r), list(leaves.values()), (dy, dr))
    got = {"y": y.detach(), "r": r.detach(), **{"d" + n: t for n, t in zip(leaves, grads)}}
    want, mag = residual_ref(x, res, w, scale, pw, dy, dr, eps, r)
    rows = x.numel() // x.shape[-1]
    for n in got:
        like = leaves[n[1:]] if n[0] == "d" else x if n == "y" or res is None else res
        assert got[n].dtype == like.dtype, n
        # two norms, one behind the other, for what passes the branch's
        close(got[n], want[n], mag[n], 2 * K + (rows if n in ("dweight", "dscale", "dpost_weight") else 0))
    return got


def residual_inputs(shape, xt, rt, wt, scale, post, res=True):
    D = shape[-1]
    sc = {"none": None, "number": 0.37, "vector": randn(D, seed=5, dt=wt)}[scale]
    return (randn(*shape, seed=1, dt=xt), 2 * randn(*shape, seed=2, dt=rt) if res else None, randn(D, seed=3, dt=wt), sc, randn(D, seed=4, dt=wt) if post else None,
            randn(*shape, seed=6, dt=xt), randn(*shape, seed=7, dt=rt if res else xt))


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("scale", ["none", "number", "vector"])
@pytest.mark.parametrize("types", [("f32", "f32", "f32"), ("bf16", "f32", "f32"), ("bf16", "bf16", "bf16"), ("bf16", "bf16", "f32"), ("f16", "f32", "f16"), ("f16", "f16", "f32")])
@pytest.mark.parametrize("shape", [(3, 11, 64), (37, 200), (5, 77), (1, 1)])
def test_residual_norm(types, shape, scale, post):
    residual_check(*residual_inputs(shape, *(DT[t] for t in types), scale, post))


@pytest.mark.parametrize("scale,post", [("none", False), ("vector", False), ("vector", True)])
@pytest.mark.parametrize("D", [7, 8, 128, 136, 256, 300, 512, 513, 1024, 1025, 1032, 2048, 2050, 2056, 4096, 4099, 8192])
def test_residual_norm_row_lengths(D, scale, post):
    residual_check(*residual_inputs((5, D), torch.bfloat16, torch.float32, torch.float32, scale, post))


@pytest.mark.parametrize("rows,D", [(1, 128), (9001, 64), (2500, 1024), (1000, 4096), (400, 8192)])
@pytest.mark.parametrize("post", [False, True])
def test_residual_norm_many_rows(rows, D, post):
    ins = residual_inputs((rows, D), torch.bfloat16, torch.bfloat16, torch.bfloat16, "vector", post)
    got, again = residual_check(*ins), residual_check(*ins)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("scale,post", [("none", False), ("number", False), ("vector", True)])
def test_residual_norm_without_a_stream(scale, post):
    residual_check(*residual_inputs((9, 256), torch.bfloat16, None, torch.float32, scale, post, res=False))


def test_residual_norm_partial_gradients():
    x, res, w, sc, pw, dy, dr = residual_inputs((50, 256), torch.bfloat16, torch.float32, torch.float32, "vector", True)
    zero_r, zero_y = torch.zeros_like(dr), torch.zeros_like(dy)
    for only, other in ((0, (dy, zero_r)), (1, (zero_y, dr))):
        full = residual_check(x, res, w, sc, pw, *other)
        leaves = [t.clone().requires_grad_(True) for t in (x, res, w, sc, pw)]
        out = ops.residual_norm(leaves[0], leaves[1], leaves[2], scale=leaves[3], post_weight=leaves[4])[only]
        for n, t in zip(("dx", "dresidual", "dweight", "dscale", "dpost_weight"), torch.autograd.grad(out, leaves, (dy, dr)[only])):
            assert torch.equal(t, full[n]), n
    full = residual_check(x, res, w, sc, pw, dy, dr)
    for i, n in enumerate(("dx", "dresidual", "dweight", "dscale", "dpost_weight")):
        ins = [x, res, w, sc, pw]
        ins[i] = ins[i].clone().requires_grad_(True)
        out = ops.residual_norm(ins[0], ins[1], ins[2], scale=ins[3], post_weight=ins[4])
        assert torch.equal(torch.autograd.grad(out, ins[i], (dy, dr))[0], full[n]), n


def test_residual_norm_the_two_gradients_of_a_plain_sum_are_apart():
    """x and the stream get equal gradients; what a caller does to one must not show in the other."""
    x, res, w, _, _, dy, dr = residual_inputs((5, 64), torch.bfloat16, torch.bfloat16, torch.bfloat16, "none", False)
    a, b = x.clone().requires_grad_(True), res.clone().requires_grad_(True)
    y, r = ops.residual_norm(a, b, w)
    torch.autograd.backward((y, r), (dy, dr))
    before = b.grad.clone()
    assert torch.equal(a.grad, before)
    a.grad.zero_()
    assert torch.equal(b.grad, before)


def test_residual_norm_strides():
    x, res, w, sc, pw, dy, dr = residual_inputs((4, 10, 64), torch.bfloat16, torch.float32, torch.float32, "vector", True)
    want = residual_check(x, res, w, sc, pw, dy, dr)
    for at in (8, 1):
        wide = torch.zeros(4, 10, 200, dtype=x.dtype, device="cuda")
        xv = wide[..., at:at + 64].copy_(x)
        rv = torch.zeros(10, 4, 64, device="cuda").transpose(0, 1).copy_(res)
        got = residual_check(xv, rv, w, sc, pw, dy, dr)
        if at % 8 == 0:
            assert all(torch.equal(got[n], want[n]) for n in want)


def test_one_row_without_further_dimensions():
    x, w = randn(96, seed=1), randn(96, seed=2)
    assert torch.equal(ops.gated_norm(x, x, w), ops.gated_norm(x[None], x[None], w)[0])
    for a, b in zip(ops.residual_norm(x, x, w), ops.residual_norm(x[None], x[None], w)):
        assert torch.equal(a, b[0])


def test_the_same_tensor_twice():
    x, w, dy, dr = randn(7, 64, seed=1, dt=torch.bfloat16), randn(64, seed=2, dt=torch.bfloat16), randn(7, 64, seed=3, dt=torch.bfloat16), randn(7, 64, seed=4, dt=torch.bfloat16)
    a, b, leaf = x.clone().requires_grad_(True), x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    for f, d in ((lambda s, t: ops.residual_norm(s, t, w), (dy, dr)), (lambda s, t: (ops.gated_norm(s, t, w),), (dy,))):
        da, db = torch.autograd.grad(f(a, b), (a, b), d)
        both, = torch.autograd.grad(f(leaf, leaf), leaf, d)
        assert torch.equal(both, da + db)


def test_second_derivatives_are_refused():
    x, w = randn(5, 64).requires_grad_(True), randn(64)
    for f in (lambda: ops.gated_norm(x, x.detach(), w), lambda: ops.residual_norm(x, None, w)[0]):
        d, = torch.autograd.grad(f(), x, torch.ones_like(x).requires_grad_(True), create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            d.sum().backward()


def test_what_is_not_finite_stays_in_its_row():
    x, z, w, dy = (randn(9, 200, seed=i, dt=torch.bfloat16) for i in range(4))
    w = w[0].float()
    want, wantr = ops.gated_norm(x, z, w), ops.residual_norm(x, z, w, scale=w, post_weight=w)
    x[4, 3] = float("nan")
    got, gotr = ops.gated_norm(x, z, w), ops.residual_norm(x, z, w, scale=w, post_weight=w)
    keep = [i for i in range(9) if i != 4]
    assert bool(got[4].isnan().all()) and torch.equal(got[keep], want[keep])
    for a, b in zip(gotr, wantr):
        assert bool(a[4].isnan().all()) and torch.equal(a[keep], b[keep])


def test_empty_rows():
    x = torch.zeros(0, 3, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y = ops.gated_norm(x, x.detach(), w)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == x.shape and dx.shape == x.shape and bool((dw == 0).all())
    y, r = ops.residual_norm(x, x.detach(), w, scale=w)
    dx, dw = torch.autograd.grad(y.sum() + r.sum(), (x, w))
    assert r.shape == x.shape and dx.shape == x.shape and bool((dw == 0).all())


def test_offsets_beyond_32_bits():
    big = torch.empty(3 * (1 << 30) + 64, dtype=torch.bfloat16, device="cuda")
    x, w = randn(3, 64, seed=1, dt=torch.bfloat16), randn(64, seed=2)
    far = big.as_strided((3, 64), ((1 << 30) + 24, 1))
    far.copy_(x)
    assert torch.equal(ops.gated_norm(far, far, w), ops.gated_norm(x, x, w))
    for a, b in zip(ops.residual_norm(far, far, w), ops.residual_norm(x, x, w)):
        assert torch.equal(a, b)


def test_refusals():
    x, w = randn(4, 64, dt=torch.bfloat16), randn(64)
    wide = torch.zeros(2, 8193, device="cuda")
    for f, what in ((lambda: ops.gated_norm(x, x[:2], w), "shapes"), (lambda: ops.gated_norm(x, x.float(), w), "type of x"), (lambda: ops.gated_norm(x, x, w[:8]), "vector"),
                    (lambda: ops.gated_norm(x.double(), x.double(), w), "fp32, bf16 or fp16"), (lambda: ops.gated_norm(x, x, w, activation="relu"), "activation"),
                    (lambda: ops.gated_norm(wide, wide, wide[0]), "8192"), (lambda: ops.gated_norm(x, x, w, eps=-1.0), "eps"), (lambda: ops.gated_norm(x, x, w, eps=float("nan")), "eps"),
                    (lambda: ops.gated_norm(x[:, :0], x[:, :0], w[:0]), "row length"), (lambda: ops.residual_norm(x, x[:1], w), "shapes"),
                    (lambda: ops.residual_norm(x, x.half(), w), "stream"), (lambda: ops.residual_norm(x, x, w, scale=w[:3]), "scale"),
                    (lambda: ops.residual_norm(x, x, w, post_weight=w.int()), "post_weight"), (lambda: ops.residual_norm(wide, wide, wide[0]), "8192")):
        with pytest.raises(ops.GdnError, match=what):
            f()
