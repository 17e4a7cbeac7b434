"""GPU: a reorder of tensors whose groups have more than 4 GB of rows, and of more strips of wide groups than there are CTAs."""
import pytest
import torch

from lethe_b200 import ops

pytestmark = pytest.mark.gpu


def filled(rows, row, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-2**31, 2**31, (rows, row), generator=g, device="cuda", dtype=torch.int32)


# rows in units of 4 bytes: those of 16-byte multiples go through the rings, the others through registers; 33 rows and more through the kernel of wide groups
@pytest.mark.parametrize("B,W,row", [(2, 2, (1 << 29) + 1024), (3, 2, (3 << 27) + 77), (1, 3, (1 << 30) + 512), (40, 4, 28_000_000), (9, 256, 260_004), (1, 33, 50_000_007), (2, 100, 6_000_000)])
def test_reorder(B, W, row):
    t, small = filled(B * W, row, 1), filled(B * W, 5, 2)
    parents = torch.randint(0, W, (B, W), generator=torch.Generator(device="cuda").manual_seed(B), device="cuda")
    parents[0] = torch.arange(W, device="cuda").roll(1)
    rows = (torch.arange(B, device="cuda")[:, None] * W + parents).flatten()
    want, few = t[rows], small[rows]
    ops.reorder_states([t, small], parents)
    assert torch.equal(t, want) and torch.equal(small, few)
