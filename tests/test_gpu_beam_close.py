"""GPU: how far the sum of a beam's exponentials can be off, and that the order of candidates does not show it.

The first sums of the selection are in 32 bits.  The argument t of 2^t is rounded three times (the difference, log2(e) / T, their product), each by 2^-24 of
|t|.  A sum of n terms with one t = 0 among them and the others not above it is off by those, relative to itself, times the mean of |t| weighted with
2^t.  That mean m is largest where all others have the same t = -(m + 1 / ln 2), and then n - 1 = ln 2 e m 2^m: 8.93 for the 8192 terms that are summed relative to
one of them.  With ln 2 for the derivative of 2^t, the hardware's exp2 (2^-22) and six roundings of sums (2^-24 each) the logarithm of a sum is off by less than
ln 2 * 3 * 2^-24 * 9 + 2^-22 + 6 * 2^-24 = 1.72e-6.  A score is rounded to fp32 once more, by half a step."""
import math

import pytest
import torch

from lethe_b200 import ops

pytestmark = pytest.mark.gpu
BOUND = math.log(2) * 3 * 2.0**-24 * 9 + 2.0**-22 + 6 * 2.0**-24
N = 8192


def flat(tails, head, dtype=torch.float32):
    """Rows of N logits: one `head`, all others as unlikely as another."""
    x = tails.to(dtype)[:, None].expand(-1, N).clone()
    x[:, 0] = head
    return x


def log_probability(x, temperature):
    x = x.double() / temperature
    return x[..., 0] - torch.logsumexp(x, -1)


# 1.429, 1.4085, 0.7145: log2(e) / T in 32 bits is nearly half a step too large, 1.426 and 1.441: too small
@pytest.mark.parametrize("temperature", [1.429, 1.4085, 1.426, 1.441, 0.7145, 0.7, 0.9, 1.0, 1.3])
@pytest.mark.parametrize("head", [10.3, 3.7, 0.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_flat_tails(dtype, head, temperature):
    """The scores of one beam, with the parent's score such that they are near zero and show all of the error; many rows, so that
    a sum has 8192 terms."""
    tails = torch.linspace(head - 8 * temperature, head - 4.5 * temperature, 4200, device="cuda")
    x = flat(tails, head, dtype)
    c = log_probability(x, temperature)
    scores = (-c).float()
    got = ops.beam_select(x[:, None], scores[:, None], 1, temperature=temperature)
    assert (got.tokens == 0).all()
    want = scores.double() + c
    assert ((got.scores[:, 0].double() - want).abs() <= BOUND + want.abs() * 2.0**-24).all()


# tails whose first sums are off most: 1.04e-6 too high a score, 9.3e-7 too low a one
@pytest.mark.parametrize("temperature,tail", [(1.429, 0.626088619), (1.426, 1.48912668), (1.441, -0.572188854), (1.4085, 1.94828939)])
@pytest.mark.parametrize("apart", [1e-8, -1e-8, 5e-8, -5e-8, 1e-7, -1e-7, 5e-7, -5e-7, 1e-6, -1e-6, 2e-6, -2e-6])
def test_beside_a_beam_without_a_sum(apart, temperature, tail):
    """A beam with a flat tail, and one that has ended, whose score is `apart` from the first's best candidate."""
    x = flat(torch.tensor([tail], device="cuda"), 10.3)
    c = log_probability(x, temperature)
    start = (-c).float()
    end = (start.double() + c + apart).float()
    assert ((end.double() - start.double() - c - apart).abs() < 1e-9).all()
    B = 2100      # (of so many rows one warp takes all of each)
    scores = torch.stack([start, end], 1).expand(B, 2)
    finished = torch.tensor([[False, True]], device="cuda").expand(B, 2)
    got = ops.beam_select(x[None].expand(B, 2, N), scores, 2, temperature=temperature, finished=finished, eos=5)
    assert (got.parents[:, 0] == int(apart > 0)).all() and (got.tokens[:, 0] == (5 if apart > 0 else 0)).all()
    pen = torch.tensor([[1.0, 0.5]], device="cuda")      # the same with half the score under half the penalty
    got = ops.beam_select(x[None].expand(B, 2, N), scores * pen, 2, temperature=temperature, finished=finished, eos=5, penalty=pen.expand(B, 2))
    assert (got.parents[:, 0] == int(apart > 0)).all()


@pytest.mark.parametrize("V", [8192, 131072])
@pytest.mark.parametrize("temperature", [0.7, 0.9, 1.429])
def test_beams_with_a_tail_beside_one_another(temperature, V):
    """Two beams whose tails are rounded to different sides, the score of one of them going up step by step past the other's."""
    tails = torch.tensor([10.3 - 8.0 * temperature / 1.44, 10.3 - 8.06 * temperature / 1.44], device="cuda")
    x = flat(tails, 10.3).repeat(1, V // N)      # (a head in every part, so that every sum has its tail)
    x[:, 0] += 1.0
    c = log_probability(x, temperature)
    for moved in (0, 1):
        scores = (-c).float()
        for step in range(-8, 9):
            s = scores.clone()
            s[moved] = scores[moved] * (1 - step * 2.0**-22)
            value = s.double() + c
            assert (value[0] - value[1]).abs() > 1e-9      # (64 bits tell these apart)
            B = 2200 if V == N else 260
            got = ops.beam_select(x.expand(B, 2, V), s.expand(B, 2), 1, temperature=temperature)
            assert (got.parents == int(value[1] > value[0])).all() and (got.tokens == 0).all()
