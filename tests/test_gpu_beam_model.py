"""GPU: the operators of decoding with several hypotheses together: a model's beam search against one that keeps every hypothesis as a list, and a
pool of slots whose sequences come, are forked, end and are moved."""
import pytest
import torch

from lethe_b200 import ops
from lethe_b200.tiny import TinyDiagLM

pytestmark = pytest.mark.gpu


def model(vocab):
    torch.manual_seed(3)
    m = TinyDiagLM(ops, vocab=vocab, d_model=64, H=2, V=32, layers=2).cuda()
    with torch.no_grad():
        m.head.weight.mul_(4.0)
    return m


@pytest.mark.parametrize("eos", [None, 5])
@pytest.mark.parametrize("beams", [1, 3, 8])
def test_search(beams, eos):
    """Against the same model calls with every hypothesis a list of tokens and a list of states of its own, chosen in 64 bits."""
    V, steps, B = 23, 6, 2
    m = model(V)
    prompt = torch.randint(0, V, (B, 9), generator=torch.Generator().manual_seed(1)).cuda()
    written, scores = m.beam_search(prompt, steps, beams, eos)
    assert written.shape == (B, beams, steps) and scores.shape == (B, beams)
    with torch.no_grad():
        logits, states = m(prompt)
        logits = logits[:, -1:].expand(B, beams, V)
        alive = [[([], 0.0 if w == 0 else float("-inf"), False, [s[b].clone() for s in states]) for w in range(beams)] for b in range(B)]
        for t in range(steps):
            if t:
                batch = [torch.stack([h[3][i] for group in alive for h in group]) for i in range(len(states))]
                logits = m(torch.tensor([h[0][-1] for group in alive for h in group], device="cuda"), batch)[0].view(B, beams, V)
            for b in range(B):
                offers = []
                for w, (tokens, score, done, _) in enumerate(alive[b]):
                    logp = torch.log_softmax(logits[b, w].double(), -1).tolist()
                    offers += [(score, w, eos)] if done else [(score + logp[v], w, v) for v in range(V)]
                offers.sort(key=lambda o: (-o[0], o[1], o[2]))
                after = [[x[b * beams + w].clone() for x in batch] if t else alive[b][w][3] for w in range(beams)]
                alive[b] = [(alive[b][w][0] + [v], float(torch.tensor(c)), alive[b][w][2] or v == eos, after[w]) for c, w, v in offers[:beams]]
    assert written.tolist() == [[h[0] for h in group] for group in alive]
    # a score is rounded to fp32 every step, and a step's sum of exponentials is up to 2^-20 off (no score is over 32)
    want = torch.tensor([[h[1] for h in group] for group in alive], dtype=torch.float64)
    assert (want.abs() < 32).all() and ((scores.double().cpu() - want).abs() <= 2 * steps * (2.0**-20 + 2.0**-20)).all()


def test_scores_are_those_of_the_whole_text():
    """What a hypothesis' score says, against its log probability when it is read from the first token on (1e-3: one token after another and a
    whole prompt differ by roundings of 64-term products in fp32, 2^-17 of logits below 64, in each of seven tokens)."""
    V, steps = 23, 7
    m = model(V)
    prompt = torch.randint(0, V, (2, 5), generator=torch.Generator().manual_seed(2)).cuda()
    written, scores = m.beam_search(prompt, steps, 4)
    text = torch.cat([prompt[:, None].expand(2, 4, 5), written], 2).view(8, -1)
    with torch.no_grad():
        logits = m(text)[0]
    assert logits.abs().max() < 64
    logp = torch.log_softmax(logits.double(), -1)[:, 4:-1].gather(2, text[:, 5:, None]).sum((1, 2)).view(2, 4)
    assert (logp - scores).abs().max() < 1e-3 * 4
    assert (scores[:, :-1] >= scores[:, 1:]).all()


def test_pool():
    """A server's steps: new sequences, forks, tokens, ends, and the live slots moved together; each sequence against one that keeps a state of its own."""
    S, H, V, K = 12, 2, 64, 128
    g = torch.Generator(device="cuda").manual_seed(2)
    pool = [torch.zeros(S, H, K, V, device="cuda"), torch.zeros(S, 5, 3, dtype=torch.bfloat16, device="cuda")]
    other = torch.empty(S, H, K, V, device="cuda")
    live = torch.zeros(S, dtype=torch.bool, device="cuda")
    alone = {}                                                     # slot -> states of its own
    for t in range(25):
        source = torch.randint(-1, S, (3,), generator=g, device="cuda")
        target, after = ops.fork_states(pool, live, source)
        for s, to in zip(source.tolist(), target.tolist()):
            if to >= 0:
                alone[to] = [torch.zeros_like(p[0]) for p in pool] if s < 0 else [x.clone() for x in alone[s]]
        live = after
        q, k = (torch.nn.functional.normalize(torch.randn(S, H, K, generator=g, device="cuda"), dim=-1) for _ in range(2))
        v = torch.randn(S, H, V, generator=g, device="cuda")
        conv = torch.randn(S, 5, 3, generator=g, device="cuda").bfloat16()
        slots = torch.where(live, torch.arange(S, device="cuda"), -1)
        ops.gdn_decode_step(q, k, v, None, None, pool[0], source=slots, out=other)
        pool[0], other = other, pool[0]
        pool[1][live] = conv[live]
        for s, mine in alone.items():
            ops.gdn_decode_step(q[s:s + 1], k[s:s + 1], v[s:s + 1], None, None, mine[0][None])
            mine[1].copy_(conv[s])
        live = live & (torch.rand(S, generator=g, device="cuda") < 0.75)      # given back
        alone = {s: x for s, x in alone.items() if live[s]}
        if t % 3 == 2:
            place, count = ops.compact_states(pool, live)
            alone = {int(place[s]): x for s, x in alone.items()}
            live = torch.arange(S, device="cuda") < count
        assert set(alone) == set(live.nonzero().flatten().tolist())
        for s, x in alone.items():
            assert torch.equal(pool[0][s], x[0]) and torch.equal(pool[1][s], x[1])
