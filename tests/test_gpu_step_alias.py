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


@pytest.mark.parametrize("which", ["x", "g"])
def test_the_same_memory_under_another_storage(which):
    start = -torch.rand(N, N, generator=torch.Generator().manual_seed(4)).cuda()
    other = torch.randn(N, N, generator=torch.Generator().manual_seed(5)).cuda().abs().neg()
    mine, want = start.clone(), start.clone()
    view = torch.from_dlpack(mine).t()
    assert view.untyped_storage().data_ptr() == mine.data_ptr()
    same = start.t().contiguous()
    h = ops.diag_scan_step(*((view, other) if which == "x" else (other, view)), mine)
    wh = ops.diag_scan_step(*((same, other) if which == "x" else (other, same)), want)
    assert torch.equal(h, wh) and torch.equal(mine, want)


def test_neighbours_in_one_buffer():
    """Input, decay and state as parts of one allocation that do not overlap."""
    buffer = -torch.rand(3, 8, 64, generator=torch.Generator().manual_seed(6)).cuda()
    x, g, state = buffer.clone().unbind(0)
    want = buffer[2].clone()
    h = ops.diag_scan_step(x, g, state)
    assert torch.equal(h, ops.diag_scan_step(buffer[0].clone(), buffer[1].clone(), want)) and torch.equal(state, want)
    assert torch.equal(x, buffer[0]) and torch.equal(g, buffer[1])
