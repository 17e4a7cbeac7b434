"""Workloads of decoding with several hypotheses, for timing: choosing tokens, and moving the recurrent states that belong to them.

A case is one call (``call``) at one size:

* ``select``   ``ops.beam_select``: the best k continuations of B groups of W beams over a vocabulary of V tokens;
* ``reorder``  ``ops.reorder_states``: every beam takes over the states of the beam that it continues, in place;
* ``fork``     ``ops.fork_states``: sequences get free slots of a pool of states and a copy of a live slot's states;
* ``compact``  ``ops.compact_states``: the live slots of a pool move together at its front;
* ``step``     ``ops.gdn_decode_step`` with ``source`` and ``out``: one token, each row going on from another row's state.

States are those of the benchmark configurations and of the tests (8 to 32 heads of 128 x 64 or 128 x 128 values in 32 bits),
``layers`` of them, with the last inputs of a short convolution in 16 bits (``conv`` channels, three tokens each) and, for beams, the
tokens so far (``history``).

``run`` is the framework's calls where ``own`` is true, else the same results from elementary operations.  Candidates of different
beams can be as close as they like, so the selection's plain form is in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
K = 128
# logits, and bytes of states, of the largest listed cases: no drawn case has more
MOST_LOGITS = 64 * 8 * 131072
MOST_STATE = 512 * 2 * 16 * K * 128 * 4
DEAD = float("-inf")


def _select(B, W, V, k, *, dtype="bf16", masked=False, ended=0, penalty=False, temperature=1.0, name=None):
    c = {} if name is None else {"name": name}
    c.update(call="select", B=B, W=W, V=V, k=k, dtype=dtype, masked=masked, ended=ended, penalty=penalty, temperature=temperature)
    return c


def _states(call, layers, H, V, conv, history=0, name=None, **sizes):
    c = {} if name is None else {"name": name}
    c.update(call=call, layers=layers, H=H, V=V, conv=conv, history=history, **sizes)
    return c


def _step(B, slots, sources, H, V, *, gate="scalar", delta=True, fresh=0, name=None):
    c = {} if name is None else {"name": name}
    c.update(call="step", B=B, slots=slots, sources=sources, H=H, V=V, gate=gate, delta=delta, fresh=fresh)
    return c


def listed():
    return [
        # one request with a narrow beam and a small vocabulary: launch and latency
        _select(1, 4, 32000, 4, name="select_b1"),
        # constrained decoding of a few requests: a mask of allowed tokens, some beams ended, twice as many candidates as beams
        _select(3, 5, 32003, 10, dtype="fp32", masked=True, ended=1, penalty=True, temperature=0.7, name="select_constrained"),
        # batched serving
        _select(16, 8, 65536, 8, ended=2, name="select_b16"),
        # the largest batch, a wide vocabulary
        _select(64, 8, 131072, 16, name="select_b64"),
        # one request's beams, four layers of the benchmark's headline heads
        _states("reorder", 4, 8, 64, 512, 256, name="reorder_b1", B=1, W=4, moved=3, sources=2),
        # batched beams at the third configuration's heads
        _states("reorder", 2, 16, 128, 2048, 1024, name="reorder_b64", B=64, W=8, moved=6, sources=3),
        # four samples of one prompt, one new request
        _states("fork", 4, 8, 64, 512, name="fork_one_prompt", slots=19, taken=5, entries=5, sources=1, fresh=1),
        # 32 prompts of eight samples each, 16 new requests
        _states("fork", 2, 16, 128, 2048, name="fork_pool", slots=512, taken=160, entries=272, sources=32, fresh=16),
        # a few requests ended: one row to move per ended one at the front, rows of no particular size
        _states("compact", 3, 5, 64, 77, name="compact_few", slots=37, taken=30, moved=3),
        # a large pool with every other slot given back
        _states("compact", 2, 16, 128, 2048, name="compact_pool", slots=512, taken=256, moved=128),
        # one request's beams in one layer
        _step(4, 4, 2, 8, 64, name="step_b4"),
        # batched beams, half of them continued by others
        _step(512, 512, 256, 16, 128, gate="channel", fresh=8, name="step_b512"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    call = rng.choice(["select", "select", "select", "reorder", "reorder", "fork", "compact", "step", "step"])
    if call == "select":
        W = _log_int(rng, 1, 16)
        V = _log_int(rng, 64, 262144)
        V = V if rng.random() < 0.3 else -(-V // 64) * 64
        B = _log_int(rng, 1, max(1, min(64, MOST_LOGITS // (2 * W * V))))
        return _select(B, W, V, rng.choice([W, W, 2 * W, _log_int(rng, 1, 32)]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                       masked=rng.random() < 0.25, ended=rng.choice([0, 0, W // 3]), penalty=rng.random() < 0.3,
                       temperature=rng.choice([1.0, 1.0, 0.8, 1.3]))
    H, V = _log_int(rng, 1, 32), rng.choice([64, 64, 128])
    row = H * K * V * 4
    if call == "step":
        B = _log_int(rng, 1, max(1, min(1024, MOST_STATE // (2 * row))))
        slots = _log_int(rng, 1, max(1, min(1024, MOST_STATE // (2 * row))))
        fresh = rng.choice([0, 0, _log_int(rng, 1, B)])
        return _step(B, slots, max(1, min(slots, B - fresh, _log_int(rng, 1, slots))), H, V, gate=rng.choice(["none", "scalar", "scalar", "channel"]),
                     delta=rng.random() < 0.7, fresh=fresh if fresh < B else 0)
    layers, conv = _log_int(rng, 1, 8), rng.choice([0, _log_int(rng, 1, 4096), 64 * _log_int(rng, 1, 64)])
    most = max(4, MOST_STATE // (layers * row))
    if call == "reorder":
        W = _log_int(rng, 1, 16)
        B = _log_int(rng, 1, max(1, min(128, most // W)))
        moved = rng.randint(0, W - 1)
        return _states(call, layers, H, V, conv, rng.choice([0, _log_int(rng, 1, 4096)]), B=B, W=W, moved=moved,
                       sources=rng.randint(1, max(1, min(moved, W - 1))))
    slots = _log_int(rng, 4, min(1024, most))
    taken = rng.randint(1, slots - 2)
    if call == "compact":
        return _states(call, layers, H, V, conv, slots=slots, taken=taken, moved=rng.randint(0, min(taken, slots - taken)))
    entries = _log_int(rng, 2, slots - taken)
    fresh = rng.randint(0, entries // 4)
    return _states(call, layers, H, V, conv, slots=slots, taken=taken, entries=entries, sources=rng.randint(1, min(taken, entries - fresh)),
                   fresh=fresh)


# ------------------------------------------------------------------------------------------------------------------
def _pick(rand, rows, n, count):
    """For each of `rows` a random order of n places, its first `count`."""
    return rand(rows, n).argsort(1)[:, :count]


def prepare(case, seed):
    """Seeded inputs.  Logits ~ 2.5 N(0,1) with a few likely tokens in every row; scores fall from beam to beam; states ~ 0.1 N(0,1);
    keys and queries as rows of unit length, log decays -softplus(N(0,1) + 3)."""
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    s = {"case": c}
    if c["call"] == "select":
        B, W, V = c["B"], c["W"], c["V"]
        logits = normal(B, W, V).mul_(2.5)
        at = torch.randint(0, V // 8, (B, W, 8), generator=gen, device="cuda") + torch.arange(8, device="cuda") * (V // 8)
        s["logits"] = logits.scatter_add_(2, at, rand(B, W, 8).mul_(8.0)).to(DTYPES[c["dtype"]])
        s["scores"] = -torch.cumsum(rand(B, W).add_(0.05), 1) - 20.0 * rand(B, 1)
        s["allowed"] = rand(B, W, V) < 0.3 if c["masked"] else None
        s["finished"] = rand(B, W).argsort(1) < c["ended"] if c["ended"] else None
        s["eos"] = 1 if c["ended"] else None
        length = torch.randint(5, 200, (B, W), generator=gen, device="cuda").float()
        s["penalty"] = ((5.0 + length) / 6.0) ** 0.6 if c["penalty"] else None
        return s
    H, V = c["H"], c["V"]
    if c["call"] == "step":
        B, S = c["B"], c["slots"]
        s["state"], s["out"] = normal(S, H, K, V).mul_(0.1), torch.empty(B, H, K, V, device="cuda")
        s["q"], s["k"] = (torch.nn.functional.normalize(normal(B, H, K), dim=-1).to(torch.bfloat16) for _ in range(2))
        s["v"] = normal(B, H, V).to(torch.bfloat16)
        gates = (B, H) if c["gate"] == "scalar" else (B, H, K)
        s["g"] = None if c["gate"] == "none" else -torch.nn.functional.softplus(normal(*gates) + 3.0)
        s["beta"] = torch.sigmoid(normal(B, H)) if c["delta"] else None
        src = _pick(rand, 1, S, c["sources"])[0]
        more = src[torch.randint(0, len(src), (B - c["fresh"] - len(src),), generator=gen, device="cuda")]
        source = torch.cat([src, more, torch.full((c["fresh"],), -1, device="cuda")])
        s["source"] = source[rand(B).argsort()].to(torch.int32)
        return s
    rows = c["B"] * c["W"] if c["call"] == "reorder" else c["slots"]
    s["states"] = [normal(rows, H, K, V).mul_(0.1) for _ in range(c["layers"])]
    if c["conv"]:
        s["states"].append(normal(rows, c["layers"], c["conv"], 3).to(torch.bfloat16))
    if c["history"]:
        s["states"].append(torch.randint(0, 32000, (rows, c["history"]), generator=gen, device="cuda"))
    if c["call"] == "reorder":
        B, W, n, src = c["B"], c["W"], c["moved"], c["sources"]
        # rows in a random order: the first `n` are moved, and what they take over are `src` others, each at least once
        order = _pick(rand, B, W, W)
        parents = torch.arange(W, device="cuda").expand(B, W).clone()
        if n:
            from_kept = min(src, W - n)
            kept = order[:, n:n + from_kept]
            turn = torch.arange(n, device="cuda") % src
            moved_src = order[:, :src - from_kept].roll(-1, 1)
            sources = torch.cat([kept, moved_src], 1)[:, turn]
            own_place = sources == order[:, :n]
            sources = torch.where(own_place, kept[:, :1].expand_as(sources), sources)
            parents.scatter_(1, order[:, :n], sources)
        s["parents"] = parents
        return s
    S, n = c["slots"], c["taken"]
    live = torch.zeros(S, dtype=torch.bool, device="cuda")
    if c["call"] == "compact":
        front, back = _pick(rand, 1, n, n)[0], n + _pick(rand, 1, S - n, S - n)[0]
        live[front[c["moved"]:]] = True
        live[back[:c["moved"]]] = True
        s["live"] = live
        return s
    order = _pick(rand, 1, S, S)[0]
    live[order[:n]] = True
    src = order[:c["sources"]]
    more = src[torch.randint(0, len(src), (c["entries"] - c["fresh"] - len(src),), generator=gen, device="cuda")]
    source = torch.cat([src, more, torch.full((c["fresh"],), -1, device="cuda")])
    s["live"], s["source"] = live, source[rand(c["entries"]).argsort()].to(torch.int32)
    return s


# ------------------------------------------------------------------------------------------------------------------
# Plain forms
# ------------------------------------------------------------------------------------------------------------------
def _plain_select(s):
    c = s["case"]
    B, W, V, k = c["B"], c["W"], c["V"], min(c["k"], c["W"] * c["V"])
    x = s["logits"].double()
    if c["temperature"] != 1.0:
        x = x / c["temperature"]
    if s["allowed"] is not None:
        x = x.masked_fill(~s["allowed"], DEAD)
    top = x.amax(2, keepdim=True).clamp(min=torch.finfo(torch.float64).min)      # (a beam that may say nothing has none)
    lse = (top + torch.log(torch.exp(x - top).sum(2, keepdim=True))).clamp(min=torch.finfo(torch.float64).min)
    scores = s["scores"].double()
    value = scores[:, :, None] + (x - lse)
    del x
    if s["finished"] is not None:
        value.masked_fill_(s["finished"][:, :, None], DEAD)
        value[:, :, s["eos"]] = torch.where(s["finished"], scores, value[:, :, s["eos"]])
    rank = value if s["penalty"] is None else value / s["penalty"].double()[:, :, None]
    rank = rank.reshape(B, W * V)
    # the k largest, of equal ones the first: all above the k-th, and as many of its equals as there is room for
    kth = rank.topk(k, 1).values[:, -1:]
    above, equal = rank > kth, rank == kth
    chosen = above | (equal & (equal.cumsum(1) <= k - above.sum(1, keepdim=True)))
    places = torch.arange(W * V, 0, -1, device=rank.device).expand(B, -1).masked_fill(~chosen, 0)
    index = W * V - places.topk(k, 1).values
    index = index.gather(1, rank.gather(1, index).sort(stable=True, dim=1, descending=True).indices)
    nothing = rank.gather(1, index) == DEAD
    parents, tokens = (index // V).masked_fill(nothing, 0), (index % V).masked_fill(nothing, 0 if s["eos"] is None else s["eos"])
    out = {"scores": value.reshape(B, W * V).gather(1, index).float(), "parents": parents, "tokens": tokens}
    if s["finished"] is not None:
        out["finished"] = s["finished"].gather(1, parents) | (tokens == s["eos"])
    return out


def _plain_reorder(s):
    B, W = s["parents"].shape
    rows = (torch.arange(B, device="cuda")[:, None] * W + s["parents"]).flatten()
    return {"states": [t.copy_(t[rows]) for t in s["states"]]}


def _copy_rows(t, source, target):
    """t[target] = t[source], zeros where the source is -1."""
    rows = t[source.clamp(min=0)]
    rows = rows.masked_fill_((source < 0).view(-1, *[1] * (t.dim() - 1)), 0)
    return t.index_copy_(0, target, rows)


def _plain_fork(s):
    live, source = s["live"], s["source"].long()
    S = live.numel()
    known = (source == -1) | ((source >= 0) & (source < S) & live[source.clamp(0, S - 1)])
    place = known.long().cumsum(0) - 1
    free = (~live).sum()
    ok = known & (place < free)
    slots = live.long().argsort(stable=True)                # free slots first, in their order
    target = torch.where(ok, slots[place.clamp(0, S - 1)], -1)
    # an entry that gets nothing does once more what the first one that gets something does
    first = ok.long().argmax()
    src, dst = torch.where(ok, source, source[first]), torch.where(ok, target, target[first])
    states = [_copy_rows(t, src, dst) for t in s["states"]]
    after = live.index_fill(0, dst, True)
    return {"target": target, "live": after, "states": states}


def _plain_compact(s):
    live = s["live"]
    S, count = live.numel(), live.sum()
    at = torch.arange(S, device="cuda")
    most = S // 2
    leaves, hole = live & (at >= count), ~live & (at < count)
    moves = leaves.sum()
    src = torch.where(leaves, at, at + S).argsort()[:most]
    dst = torch.where(hole, at, at + S).argsort()[:most]
    # as many entries as there can be moves; one behind the last does the first once more, or nothing
    i = torch.arange(most, device="cuda")
    src, dst = torch.where(i < moves, src, torch.where(moves > 0, src[0], 0)), torch.where(i < moves, dst, torch.where(moves > 0, dst[0], 0))
    states = [t.index_copy_(0, dst, t[src]) for t in s["states"]]
    place = torch.where(live, at, -1).scatter(0, src, torch.where(moves > 0, dst, torch.where(live[0], 0, -1)))
    return {"place": place, "count": count, "states": states}


def _plain_step(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    source = s["source"].long()
    state = s["state"][source.clamp(min=0)].masked_fill_((source < 0)[:, None, None, None], 0)
    if s["g"] is not None:
        a = torch.exp(s["g"])
        state = state * (a[..., None, None] if a.dim() == 2 else a[..., None])
    if s["beta"] is not None:
        v = s["beta"][..., None] * (v - (k[..., None] * state).sum(2))
    s["out"].copy_(state + k[..., None] * v[..., None, :])
    o = (q[..., None] * s["out"]).sum(2) * K ** -0.5
    return {"o": o.to(torch.bfloat16), "state": s["out"]}


# ------------------------------------------------------------------------------------------------------------------
def _own(s):
    from lethe_b200 import ops

    c = s["case"]
    if c["call"] == "select":
        best = ops.beam_select(s["logits"], s["scores"], c["k"], temperature=c["temperature"], allowed=s["allowed"], finished=s["finished"],
                               eos=s["eos"], penalty=s["penalty"])
        out = {"scores": best.scores, "parents": best.parents, "tokens": best.tokens}
        if best.finished is not None:
            out["finished"] = best.finished
        return out
    if c["call"] == "reorder":
        ops.reorder_states(s["states"], s["parents"])
        return {"states": s["states"]}
    if c["call"] == "fork":
        target, live = ops.fork_states(s["states"], s["live"], s["source"])
        return {"target": target, "live": live, "states": s["states"]}
    if c["call"] == "compact":
        place, count = ops.compact_states(s["states"], s["live"])
        return {"place": place, "count": count, "states": s["states"]}
    o = ops.gdn_decode_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], source=s["source"], out=s["out"])
    return {"o": o, "state": s["out"]}


def run(s):
    if own:
        return _own(s)
    plain = {"select": _plain_select, "reorder": _plain_reorder, "fork": _plain_fork, "compact": _plain_compact, "step": _plain_step}
    return plain[s["case"]["call"]](s)


def work(case):
    """Bytes: every logit and mask value read once; of states, every row that is read by somebody once, and every row that gets other
    values once (rows that stay are neither).  Operations: an exponential as one."""
    c = dict(case)
    if c["call"] == "select":
        n = c["B"] * c["W"] * c["V"]
        e = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": n * (e + c["masked"]) + c["B"] * (c["W"] * 9 + c["k"] * 21), "flops": 4 * n}
    row = c["H"] * K * c["V"] * 4
    if c["call"] == "step":
        token = c["H"] * (2 * K * 2 + 2 * c["V"] * 2 + 4 * (0 if c["gate"] == "none" else 1 if c["gate"] == "scalar" else K) + 4 * c["delta"])
        return {"bytes": row * (c["sources"] + c["B"]) + c["B"] * (token + 4), "flops": 7 * c["B"] * c["H"] * K * c["V"]}
    row = c["layers"] * (row + 6 * c["conv"]) + 8 * c["history"]
    if c["call"] == "reorder":
        return {"bytes": c["B"] * ((c["moved"] + min(c["sources"], c["moved"])) * row + 8 * c["W"]), "flops": 0}
    if c["call"] == "fork":
        return {"bytes": row * (c["sources"] + c["entries"]) + 2 * c["slots"] + 12 * c["entries"], "flops": 0}
    return {"bytes": row * 2 * c["moved"] + 9 * c["slots"], "flops": 0}


# ------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits: the scores group by group, the step's update as matrix products; rows that are only copied have no rounding
# ------------------------------------------------------------------------------------------------------------------
def _exact_select(s):
    c = s["case"]
    k = min(c["k"], c["W"] * c["V"])
    scores = torch.empty(c["B"], k, dtype=torch.float64, device="cuda")
    for b in range(c["B"]):
        offers = []
        for w in range(c["W"]):
            start = s["scores"][b, w].double()
            divisor = 1.0 if s["penalty"] is None else s["penalty"][b, w].double()
            if s["finished"] is not None and bool(s["finished"][b, w]):
                offers.append(torch.stack([start / divisor, start])[:, None])
                continue
            x = s["logits"][b, w].double() / c["temperature"]
            if s["allowed"] is not None:
                x = x[s["allowed"][b, w]]
            best = x.topk(min(k, x.numel())).values
            value = start + (best - torch.logsumexp(x, 0))
            offers.append(torch.stack([value / divisor, value]))
        rank, value = torch.cat(offers, 1)
        n = min(k, rank.numel())
        scores[b] = DEAD
        scores[b, :n] = value[rank.topk(n).indices]
    return {"scores": scores, "parents": None, "tokens": None, **({} if s["finished"] is None else {"finished": None})}


def _exact_step(s):
    c = s["case"]
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    state = torch.cat([s["state"].double(), torch.zeros_like(s["state"][:1], dtype=torch.float64)])[s["source"].long()]
    if c["gate"] != "none":
        state *= torch.exp(s["g"].double()).reshape(c["B"], c["H"], -1, 1)
    if c["delta"]:
        v = s["beta"].double()[..., None] * (v - torch.matmul(k[:, :, None, :], state)[:, :, 0])
    state += torch.matmul(k[..., None], v[:, :, None, :])
    return {"o": torch.matmul(q[:, :, None, :], state)[:, :, 0] / math.sqrt(K), "state": state}


def exact(case, seed):
    if case["call"] not in ("select", "step"):
        return None
    s = prepare(case, seed)
    return _exact_select(s) if case["call"] == "select" else _exact_step(s)
