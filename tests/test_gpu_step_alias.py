"""GPU: the element-wise recurrence's token with inputs that are views of the state, which it writes: other CTAs' elements, before they are written."""
import pytest
import torch

from lethe_b200 import ops

pytestmark = pytest.mark.gpu

N = 1024      # rows of the state, each a CTA

VIEWS = {
    "transposed": lambda s: s.t(),
    "first row for all": lambda s: s[:1].expand_as(s),
    "last row for all": lambda s: s[-1:].expand_as(s),
    "first channel for all": lambda s: s[:, :1].expand_as(s),
    "itself": lambda s: s,
}


@pytest.mark.parametrize("complement", [False, True])
@pytest.mark.parametrize("which", ["x", "g", "both"])
@pytest.mark.parametrize("view", sorted(VIEWS))
def test_views_of_the_state(view, which, complement):
    gen = torch.Generator().manual_seed(1)
    start = -torch.rand(N, N, generator=gen).cuda()
    x, g = torch.randn(N, N, generator=gen).cuda(), -torch.rand(N, N, generator=gen).cuda()
    of = VIEWS[view]

    def inputs(state):
        return (of(state) if which != "g" else x), (of(state) if which != "x" else g)
    for _ in range(3):
        mine, want = start.clone(), start.clone()
        h = ops.diag_scan_step(*inputs(mine), mine, complement=complement)
        wh = ops.diag_scan_step(*(t.clone(memory_format=torch.contiguous_format) for t in inputs(start)), want, complement=complement)
        assert torch.equal(h, wh) and torch.equal(mine, want)


def test_rows_of_the_state_one_further():
    """An overlapping view of a larger buffer that begins a row later."""
    buffer = -torch.rand(N + 1, N, generator=torch.Generator().manual_seed(2)).cuda()
    x = torch.randn(N, N, generator=torch.Generator().manual_seed(3)).cuda()
    mine, other = buffer.clone(), buffer.clone()
    h = ops.diag_scan_step(x, mine[1:], mine[:-1])
    state = other[:-1].clone()
    wh = ops.diag_scan_step(x, other[1:].clone(), state)
    assert torch.equal(h, wh) and torch.equal(mine[:-1], state) and torch.equal(mine[-1], buffer[-1])
