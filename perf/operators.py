"""Workloads of the operators around the recurrences, for timing: the element-wise gated recurrence and the norms on both sides of a block.

A case is one call pattern (``call``) at one size:

* ``scan``        ``ops.diag_scan``: h_t = exp(g_t) h_{t-1} + x_t per channel (``complement``: (1 - exp(g_t)) x_t), forward;
* ``scan_train``  the same with its backward;
* ``step``        ``ops.diag_scan_step``: one generated token, the state updated in place;
* ``gated``       ``ops.gated_norm``: RMS norm of a block's output per head, times weight and an activated gate, forward;
* ``gated_train`` the same with its backward;
* ``residual``    ``ops.residual_norm``: r = residual + scale * x (or scale * norm(x) * post_weight), y = norm(r) * weight, forward;
* ``residual_train`` the same with its backward.

Types: ``dtype`` is that of activations, ``wide`` says that the log decay (scan, step) or the residual stream is in 32 bits
whatever ``dtype`` is.  Weights of the norms are in 32 bits with ``wide``, else in ``dtype``.  Sizes are those of the benchmark
configurations and of the tests (8 to 32 heads of 64 or 128 channels, 2048 to 65536 tokens), and the ragged ones between.

``run`` is the framework's calls where ``own`` is true, else the same results from elementary operations in 32 bits.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
# elements of the largest listed cases: no drawn case has more
MOST_SCAN = 65536 * 2048
MOST_NORM = 2 * 8192 * 4096


def _scan(call, B, L, D, *, dtype="bf16", wide=True, gates="mild", complement=False, h0=True, name=None):
    c = {} if name is None else {"name": name}
    c.update(call=call, B=B, L=L, D=D, dtype=dtype, wide=wide, gates=gates, complement=complement, h0=h0)
    return c


def _gated(call, B, L, H, V, *, dtype="bf16", wide=True, activation="silu", name=None):
    c = {} if name is None else {"name": name}
    c.update(call=call, B=B, L=L, H=H, V=V, dtype=dtype, wide=wide, activation=activation)
    return c


def _residual(call, rows, D, *, dtype="bf16", wide=True, scale="channel", post=False, name=None):
    c = {} if name is None else {"name": name}
    c.update(call=call, rows=rows, D=D, dtype=dtype, wide=wide, scale=scale, post=post)
    return c


def listed():
    return [
        # a short prompt of no particular length, evaluated without gradients: a call is launch and latency
        _scan("scan", 1, 37, 512, name="scan_short_prompt"),
        # the headline batch of the benchmark (B=2, L=2048, 8 heads of 128 channels) in training
        _scan("scan_train", 2, 2048, 1024, gates="strong", name="scan_train_B2_L2048_D1024"),
        # batches that end where their documents end, everything in 32 bits, input weighted by what the state forgets
        _scan("scan_train", 3, 3001, 770, dtype="fp32", complement=True, name="scan_train_ragged_fp32"),
        # the longest sequence of the benchmark, decays from a token to thousands of them
        _scan("scan_train", 1, 65536, 2048, gates="long", h0=False, name="scan_train_L65536"),
        # generation for one sequence: launch and host latency
        _scan("step", 1, 1, 1024, name="step_b1"),
        # batched serving
        _scan("step", 512, 1, 4096, complement=True, gates="long", name="step_b512"),
        # the norm behind the recurrence at the generation of one sequence with 8 heads
        _gated("gated", 1, 1, 8, 64, name="gated_decode"),
        # the headline configuration's output, 8 heads of 64 channels, its gate part of a fused projection
        _gated("gated_train", 2, 2048, 8, 64, name="gated_train_B2_L2048_H8_V64"),
        # the third configuration's: 16 heads of 128
        _gated("gated_train", 4, 4096, 16, 128, wide=False, activation="sigmoid", name="gated_train_B4_L4096_H16_V128"),
        # batched serving: a row for each sequence, norms on both sides of the block
        _residual("residual", 64, 2048, post=True, name="residual_decode_b64"),
        # training at the model width of the headline configuration, the stream in 32 bits
        _residual("residual_train", 2 * 2048, 1024, name="residual_train_B2_L2048_D1024"),
        # long batches of a wide model, all in 16 bits, norms on both sides
        _residual("residual_train", 2 * 8192, 4096, wide=False, post=True, name="residual_train_B2_L8192_D4096"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    call = rng.choice(["scan", "scan_train", "scan_train", "scan_train", "step", "gated", "gated_train", "gated_train",
                       "residual", "residual_train", "residual_train"])
    dtype, wide = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.6
    if call in ("scan", "scan_train", "step"):
        gates, complement, h0 = rng.choice(["strong", "mild", "long"]), rng.random() < 0.4, rng.random() < 0.6
        D = _log_int(rng, 1, 4096)
        D = D if rng.random() < 0.2 else -(-D // 8) * 8
        if call == "step":
            return _scan(call, _log_int(rng, 1, 512), 1, D, dtype=dtype, wide=wide, gates=gates, complement=complement)
        L = _log_int(rng, 1, 65536)
        B = _log_int(rng, 1, max(1, min(64, MOST_SCAN // (L * D))))
        if B * L * D > MOST_SCAN:
            D = max(1, MOST_SCAN // (B * L))
        return _scan(call, B, L, D, dtype=dtype, wide=wide, gates=gates, complement=complement, h0=h0)
    if call in ("gated", "gated_train"):
        V = rng.choice([64, 64, 128, 128, 256, _log_int(rng, 1, 1024)])
        H = _log_int(rng, 1, 32)
        L = _log_int(rng, 1, 16384)
        B = _log_int(rng, 1, max(1, min(32, MOST_NORM // (L * H * V))))
        L = max(1, min(L, MOST_NORM // (B * H * V)))
        return _gated(call, B, L, H, V, dtype=dtype, wide=wide, activation=rng.choice(["silu", "silu", "sigmoid"]))
    D = _log_int(rng, 16, 8192)
    D = D if rng.random() < 0.2 else -(-D // 8) * 8
    rows = _log_int(rng, 1, max(1, min(65536, MOST_NORM // D)))
    return _residual(call, rows, D, dtype=dtype, wide=wide, scale=rng.choice(["none", "number", "channel", "channel"]),
                     post=rng.random() < 0.4)


def prepare(case, seed):
    """Seeded inputs.  Activations ~ N(0,1); log decays: ``strong`` -softplus(N(0,1) + 3) and ``mild`` -0.1 U(0,1) as in the
    benchmark, ``long`` per channel a rate between 1e-4 and 1 (log-uniform) times a sigmoid; initial states ~ 0.1 N(0,1);
    residual streams with a few large channels, as trained models have them; weights around one, learned scales around 0.5."""
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[c["dtype"]]
    wdt = torch.float32 if c["wide"] else dt
    call = c["call"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    s = {"case": c}
    if call in ("scan", "scan_train", "step"):
        B, L, D = c["B"], c["L"], c["D"]
        shape = (B, D) if call == "step" else (B, L, D)
        s["x"] = normal(*shape).to(dt)
        if c["gates"] == "strong":
            g = F.softplus(normal(*shape).add_(3.0)).neg_()
        elif c["gates"] == "mild":
            g = rand(*shape).mul_(-0.1)
        else:
            g = normal(*shape).sigmoid_().mul_(-torch.exp(rand(D) * math.log(1e4) - math.log(1e4)))
        s["g"] = g.to(wdt)
        del g
        state = normal(B, D).mul_(0.1)
        if call == "step":
            s["state"] = state
            return s
        s["h0"] = state if c["h0"] else None
        if call == "scan_train":
            s["dh"], s["dhT"] = normal(*shape).to(dt), normal(B, D)
            s["wrt"] = [n for n in ("x", "g", "h0") if s[n] is not None]
    elif call in ("gated", "gated_train"):
        B, L, H, V = c["B"], c["L"], c["H"], c["V"]
        s["x"] = normal(B, L, H, V).mul_(0.5).to(dt)
        # the gate is one part of a projection that also gives the next block's values
        s["gate"] = normal(B, L, 2 * H * V).to(dt)[..., H * V:].unflatten(-1, (H, V))
        s["weight"] = normal(V).mul_(0.1).add_(1.0).to(wdt)
        if call == "gated_train":
            s["dy"] = normal(B, L, H, V).to(dt)
            s["wrt"] = ["x", "gate", "weight"]
    else:
        R, D = c["rows"], c["D"]
        s["x"] = normal(R, D).to(dt)
        s["residual"] = normal(R, D).mul_(1.0 + 9.0 * (rand(D) < 0.02)).to(wdt)
        s["weight"] = normal(D).mul_(0.1).add_(1.0).to(wdt)
        s["post_weight"] = normal(D).mul_(0.1).add_(1.0).to(wdt) if c["post"] else None
        s["scale"] = {"none": None, "number": 0.25, "channel": 0}[c["scale"]]
        if c["scale"] == "channel":
            s["scale"] = normal(D).mul_(0.1).add_(0.5).to(wdt)
        if call == "residual_train":
            s["dy"], s["dr"] = normal(R, D).to(dt), normal(R, D).to(wdt)
            s["wrt"] = [n for n in ("x", "residual", "weight", "post_weight", "scale") if isinstance(s[n], torch.Tensor)]
    for n in s.get("wrt", ()):
        s[n].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------------------
# Plain forms: elementary operations in 32 bits, one rounding at the end
# ------------------------------------------------------------------------------------------------------------------
def _recurrence(c, x):
    """h_t = (1 + c_t) h_{t-1} + x_t along dimension 1, h_{-1} = 0, by doubling: after n steps every h_t holds the last 2^n terms.
    Decays come as c = exp(g) - 1: next to one, 32 bits would round 1 + c by more than what thousands of tokens forgive."""
    L, n = x.shape[1], 1
    c, h = c.clone(), x.clone()
    while n < L:
        h[:, n:] = h[:, n:] + (h[:, :-n] + c[:, n:] * h[:, :-n])
        c[:, n:] = c[:, n:] + c[:, :-n] + c[:, n:] * c[:, :-n]
        n *= 2
    return h


def _plain_scan(s, train):
    comp = s["case"]["complement"]
    x, g = s["x"].detach().float(), s["g"].detach().float()
    c = torch.expm1(g)
    u = -c * x if comp else x.clone()
    if s["h0"] is not None:
        u[:, 0] += torch.exp(g[:, 0]) * s["h0"].detach()
    h = _recurrence(c, u)
    del u
    out = {"h": h.to(s["x"].dtype), "hT": h[:, -1].clone()}
    if not train:
        return out
    d = s["dh"].float().clone()
    d[:, -1] += s["dhT"]
    # backwards in time the gradient of h_t is d_t + exp(g_{t+1}) (gradient of h_{t+1}); the last token has no later one
    later = torch.cat([torch.full_like(c[:, :1], -1.0), c.flip(1)[:, :-1]], 1)
    d = _recurrence(later, d.flip(1)).flip(1)
    del later
    first = torch.zeros_like(h[:, :1]) if s["h0"] is None else s["h0"].detach()[:, None]
    before = torch.cat([first, h[:, :-1]], 1)
    del h
    out["dx"] = (-c * d if comp else d).to(s["x"].dtype)
    out["dg"] = (d * torch.exp(g) * (before - x if comp else before)).to(s["g"].dtype)
    if s["h0"] is not None:
        out["dh0"] = torch.exp(g[:, 0]) * d[:, 0]
    return out


def _plain_step(s):
    g = s["g"].float()
    x = s["x"].float()
    h = torch.exp(g) * s["state"] + (-torch.expm1(g) * x if s["case"]["complement"] else x)
    s["state"].copy_(h)
    return {"h": h.to(s["x"].dtype), "state": s["state"]}


def _rms(x):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _wide_leaves(s, names):
    """The named inputs in 32 bits, as leaves of their own where the case differentiates."""
    return [s[n].detach().float().requires_grad_(n in s.get("wrt", ())) if isinstance(s[n], torch.Tensor) else s[n] for n in names]


def _gradients(s, outs, douts, leaves):
    got = iter(torch.autograd.grad(outs, [t for t in leaves if isinstance(t, torch.Tensor)], douts))
    return {"d" + n: next(got).to(s[n].dtype) for n in s["wrt"]}


def _plain_gated(s, train):
    names = ("x", "gate", "weight")
    x, gate, weight = leaves = _wide_leaves(s, names)
    act = torch.sigmoid(gate)
    if s["case"]["activation"] == "silu":
        act = gate * act
    y = _rms(x) * weight * act
    out = {"y": y.detach().to(s["x"].dtype)}
    if train:
        out.update(_gradients(s, (y,), (s["dy"].float(),), leaves))
    return out


def _plain_residual(s, train):
    names = ("x", "residual", "weight", "post_weight", "scale")
    x, residual, weight, post_weight, scale = leaves = _wide_leaves(s, names)
    t = x if post_weight is None else _rms(x) * post_weight
    r = residual + (t if scale is None else t * scale)
    stored = r.detach().to(s["residual"].dtype)
    seen = r + (stored.float() - r.detach())            # the second norm is that of the stream as it is kept
    y = _rms(seen) * weight
    out = {"y": y.detach().to(s["x"].dtype), "r": stored}
    if train:
        out.update(_gradients(s, (y, r), (s["dy"].float(), s["dr"].float()), leaves))
    return out


# ------------------------------------------------------------------------------------------------------------------
def _own(s):
    from lethe_b200 import ops

    c = s["case"]
    call = c["call"]
    with torch.set_grad_enabled(call.endswith("_train")):
        if call == "step":
            h = ops.diag_scan_step(s["x"], s["g"], s["state"], complement=c["complement"])
            return {"h": h, "state": s["state"]}
        if call in ("scan", "scan_train"):
            names, given = ("h", "hT"), ("dh", "dhT")
            outs = ops.diag_scan(s["x"], s["g"], s["h0"], complement=c["complement"])
        elif call in ("gated", "gated_train"):
            names, given = ("y",), ("dy",)
            outs = (ops.gated_norm(s["x"], s["gate"], s["weight"], eps=EPS, activation=c["activation"]),)
        else:
            names, given = ("y", "r"), ("dy", "dr")
            outs = ops.residual_norm(s["x"], s["residual"], s["weight"], scale=s["scale"], post_weight=s["post_weight"], eps=EPS)
    out = {n: t.detach() for n, t in zip(names, outs)}
    if call.endswith("_train"):
        grads = torch.autograd.grad(outs, [s[n] for n in s["wrt"]], [s[n] for n in given])
        out.update({"d" + n: t for n, t in zip(s["wrt"], grads)})
    return out


def run(s):
    if own:
        return _own(s)
    call = s["case"]["call"]
    if call == "step":
        return _plain_step(s)
    plain = {"scan": _plain_scan, "gated": _plain_gated, "residual": _plain_residual}[call.split("_")[0]]
    with torch.set_grad_enabled(call.endswith("_train")):
        return plain(s, call.endswith("_train"))


def work(case):
    """Bytes: every input read once, every output written once; a backward reads the forward's inputs and the gradients that come in,
    and writes one for each input.  Operations: products and sums of the formulas, an exponential or a root as one."""
    c = dict(case)
    call, train = c["call"], c["call"].endswith("_train")
    e = 4 if c["dtype"] == "fp32" else 2
    w = 4 if c["wide"] else e
    if call == "step":
        n = c["B"] * c["D"]
        return {"bytes": n * (2 * e + w + 8), "flops": 4 * n}
    if call in ("scan", "scan_train"):
        n, states = c["B"] * c["L"] * c["D"], 4 * c["B"] * c["D"]
        ends = states * (2 if c["h0"] else 1)
        if not train:
            return {"bytes": n * (2 * e + w) + ends, "flops": 3 * n}
        return {"bytes": n * (2 * e + w) + ends + n * (3 * e + 2 * w) + states * (3 if c["h0"] else 1), "flops": 11 * n}
    if call in ("gated", "gated_train"):
        n = c["B"] * c["L"] * c["H"] * c["V"]
        if not train:
            return {"bytes": 3 * e * n + w * c["V"], "flops": 9 * n}
        return {"bytes": 8 * e * n + 3 * w * c["V"], "flops": 32 * n}
    n, vectors = c["rows"] * c["D"], 1 + c["post"] + (c["scale"] == "channel")
    forward = n * (2 * e + 2 * w) + vectors * w * c["D"]
    if not train:
        return {"bytes": forward, "flops": (10 if c["post"] else 6) * n}
    # the backward reads the stream and both gradients, and x where a weight or a scale of its branch is learned
    back = n * (e + 2 * w + e + w + (e if c["post"] or c["scale"] == "channel" else 0))
    return {"bytes": forward + back + 2 * vectors * w * c["D"], "flops": (30 if c["post"] else 18) * n}


# ------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits, one token after another, derivatives written out
# ------------------------------------------------------------------------------------------------------------------
def _exact_scan(s, train):
    c = s["case"]
    x, g = s["x"].detach().double(), s["g"].detach().double()
    a, L = torch.exp(g), x.shape[1]
    keep = -torch.expm1(g) if c["complement"] else None
    u = x * keep if c["complement"] else x
    h = torch.zeros_like(x[:, 0]) if s["h0"] is None else s["h0"].detach().double()
    hs = torch.empty(L + 1, *h.shape, dtype=torch.float64, device=h.device)
    hs[0] = h
    for t in range(L):
        torch.addcmul(u[:, t], a[:, t], hs[t], out=hs[t + 1])
    out = {"h": hs[1:].transpose(0, 1), "hT": hs[L]}
    if not train:
        return out
    ds = torch.empty(L, *h.shape, dtype=torch.float64, device=h.device)
    carry = s["dhT"].double()
    dh = s["dh"].double()
    for t in reversed(range(L)):
        torch.add(dh[:, t], carry, out=ds[t])
        carry = a[:, t] * ds[t]
    d, before = ds.transpose(0, 1), hs[:-1].transpose(0, 1)
    out["dx"] = d * keep if c["complement"] else d
    out["dg"] = d * a * (before - x if c["complement"] else before)
    if s["h0"] is not None:
        out["dh0"] = carry
    return out


def _exact_norm(x):
    """x / rms(x), and the map from the gradient of that to the gradient of x."""
    inv = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
    n = x * inv
    return n, lambda d: inv * (d - n * (d * n).mean(-1, keepdim=True))


def _exact_gated(s, train):
    x, z, w = (s[k].detach().double() for k in ("x", "gate", "weight"))
    n, back = _exact_norm(x)
    sg = 1.0 / (1.0 + torch.exp(-z))
    silu = s["case"]["activation"] == "silu"
    act, slope = (z * sg, sg * (1.0 + z * (1.0 - sg))) if silu else (sg, sg * (1.0 - sg))
    out = {"y": n * w * act}
    if train:
        dy = s["dy"].double()
        out["dx"] = back(dy * w * act)
        out["dgate"] = dy * n * w * slope
        out["dweight"] = (dy * n * act).flatten(0, -2).sum(0)
    return out


def _exact_residual(s, train):
    x, res, w = (s[k].detach().double() for k in ("x", "residual", "weight"))
    pw = None if s["post_weight"] is None else s["post_weight"].detach().double()
    sc = s["scale"]
    sc = 1.0 if sc is None else sc.detach().double() if isinstance(sc, torch.Tensor) else sc
    n1, back1 = (x, None) if pw is None else _exact_norm(x)
    t = n1 if pw is None else n1 * pw
    r = res + t * sc
    if s["residual"].dtype != torch.float32:
        r = r.to(s["residual"].dtype).double()          # the stream as it is kept
    n2, back2 = _exact_norm(r)
    out = {"y": n2 * w, "r": r}
    if train:
        dy = s["dy"].double()
        d = s["dr"].double() + back2(dy * w)
        out["dx"] = d * sc if pw is None else back1(d * sc * pw)
        out["dresidual"] = d
        out["dweight"] = (dy * n2).sum(0)
        if pw is not None:
            out["dpost_weight"] = (d * sc * n1).sum(0)
        if isinstance(sc, torch.Tensor):
            out["dscale"] = (d * t).sum(0)
    return out


def exact(case, seed):
    call = case["call"]
    s = prepare(case, seed)
    with torch.no_grad():
        if call == "step":
            g, x = s["g"].double(), s["x"].double()
            h = torch.exp(g) * s["state"].double() + (-torch.expm1(g) * x if case["complement"] else x)
            return {"h": h, "state": h}
        form = {"scan": _exact_scan, "gated": _exact_gated, "residual": _exact_residual}[call.split("_")[0]]
        return form(s, call.endswith("_train"))
