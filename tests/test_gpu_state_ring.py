"""GPU: the rings that move states, and their waits that run out: the kernel ends, every warp as one, and leaves the code of the wait."""
import ctypes

import pytest
import torch

from lethe_b200 import _build, ops

pytestmark = pytest.mark.gpu
SITE = 812


def run(steps, starved=-1, hole=0, limit=2_000_000):
    call = ctypes.CDLL(_build.build_probe()).lethe_probe_ring
    call.argtypes = [ctypes.c_void_p] * 3 + [ctypes.c_int] * 3 + [ctypes.c_longlong] + [ctypes.c_void_p] * 2
    data = torch.randint(1, 256, (4, 8, 512), dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(steps))
    out, status = torch.zeros_like(data), torch.zeros(1, dtype=torch.int32, device="cuda")
    begun = torch.full((4, 32), -1, dtype=torch.int32, device="cuda")
    assert call(data.data_ptr(), out.data_ptr(), status.data_ptr(), steps, starved, hole, limit, begun.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert bool((begun == begun[:, :1]).all())
    return data, out, status, begun[:, 0].tolist()


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 6, 7, 8, 100])
def test_strips_arrive(steps):
    data, out, status, begun = run(steps)
    n = min(steps, 8)
    assert int(status) == 0 and begun == [steps] * 4
    assert torch.equal(out[:, :n], data[:, :n]) and not out[:, n:].any()


@pytest.mark.parametrize("hole", [0, 1, 2, 3, 5, 11])
@pytest.mark.parametrize("starved", [0, 3, 4])
def test_a_strip_that_never_comes(starved, hole):
    steps = 200_000
    data, out, status, begun = run(steps, starved, hole)
    assert int(status) == SITE
    for w, n in enumerate(begun):
        if starved in (w, 4):
            assert hole < n <= hole + 4                   # (three steps are on their way in ahead of the one that is stored, and one more)
            n = min(hole, 8)
            assert torch.equal(out[w, :n], data[w, :n])
            assert hole >= 8 or not out[w, hole:].any()   # nothing is stored out of what did not come
        else:
            assert 8 < n < steps                          # (the limit is over long before so many steps are: they left early)
            assert torch.equal(out[w], data[w])
    with pytest.raises(ops.GdnError, match=str(SITE)):
        ops.check_status(status)


def test_the_next_call_is_not_touched():
    run(50, 1, 4)
    data, out, status, _ = run(50)
    assert int(status) == 0 and torch.equal(out, data)
    t = torch.randn(6, 5000, device="cuda")
    want = t[torch.tensor([1, 1, 0, 4, 3, 3], device="cuda")]
    ops.reorder_states(t, torch.tensor([[1, 1, 0], [1, 0, 0]], device="cuda"))
    assert torch.equal(t, want)
