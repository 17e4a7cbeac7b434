"""GPU: candidates of beams with different penalties that have the same rank.  Their order is that of the quotients: -49 / 49 is -1 to the last bit, a product
with what 1 / 49 is rounded to is not."""
from fractions import Fraction

import pytest
import torch

from lethe_b200 import ops

pytestmark = pytest.mark.gpu
# 49, 98, 103, 107, 161, 187, 197: x * (1 / x) is below one in 64 bits
PENALTIES = [1.0, 49.0, 98.0, 3.0, 103.0, 107.0, 7.0, 161.0, 187.0, 0.5, 197.0, 10.0]


def order(scores, penalty):
    rank = [Fraction(s) / Fraction(p) for s, p in zip(scores, penalty)]
    return sorted(range(len(rank)), key=lambda w: (-rank[w], w))


@pytest.mark.parametrize("kind", ["finished", "one token", "both"])
@pytest.mark.parametrize("rank", [-1.0, -3.0, 5.0, -0.25, 0.0])
def test_equal_ranks(kind, rank):
    """Beams that offer one candidate each, their own score: ended ones, and those that may say one token only."""
    W, V = len(PENALTIES), 300
    g = torch.Generator(device="cuda").manual_seed(1)
    for turn in range(W):
        for off in (0, 1):      # 1: every third beam is a little better
            pen = PENALTIES[turn:] + PENALTIES[:turn]
            scores = [rank * p + (off * p / 64 if w % 3 == 2 else 0.0) for w, p in enumerate(pen)]
            s, p = (torch.tensor([v], device="cuda") for v in (scores, pen))
            assert s[0].tolist() == scores
            x = torch.randn(1, W, V, generator=g, device="cuda")
            only = torch.randint(0, V, (1, W, 1), generator=g, device="cuda")
            allowed = torch.zeros(1, W, V, dtype=torch.bool, device="cuda").scatter_(2, only, True)
            ended = torch.tensor([[kind == "finished" or (kind == "both" and w % 2 == 0) for w in range(W)]], device="cuda")
            want = order(scores, pen)
            for k in (1, 2, 5, W):
                got = ops.beam_select(x, s, k, allowed=allowed, finished=ended, eos=7, penalty=p)
                assert got.parents[0].tolist() == want[:k]
                assert got.tokens[0].tolist() == [7 if ended[0, w] else int(only[0, w, 0]) for w in want[:k]]
                assert got.scores[0].tolist() == [scores[w] for w in want[:k]]


def test_several_groups():
    """The same beams in groups with the penalties in other orders."""
    W = len(PENALTIES)
    pen = torch.stack([torch.tensor(PENALTIES).roll(i) for i in range(40)]).cuda()
    got = ops.beam_select(torch.zeros(40, W, 9, device="cuda"), -pen, W, finished=torch.ones(40, W, dtype=torch.bool, device="cuda"), eos=0, penalty=pen)
    assert torch.equal(got.parents, torch.arange(W, device="cuda").expand(40, W)) and torch.equal(got.scores, -pen)
