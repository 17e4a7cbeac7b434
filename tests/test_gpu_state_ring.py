"""GPU: the rings that move states, and their waits that run out: the kernel ends, every warp as one, and leaves the code of the wait."""
import ctypes

import pytest
import torch

from lethe_b200 import _build, native, ops

from .test_beam_cabi_cpu import States

pytestmark = pytest.mark.gpu
SITE = 812


def run(steps, starved=-1, hole=0, limit=2_000_000, index=0):
    call = ctypes.CDLL(_build.build_probe()).lethe_probe_ring
    call.argtypes = [ctypes.c_void_p] * 3 + [ctypes.c_int] * 3 + [ctypes.c_longlong, ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    data = torch.randint(1, 256, (4, 8, 512), dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(steps))
    out, status = torch.zeros_like(data), torch.zeros(1, dtype=torch.int32, device="cuda")
    begun = torch.full((4, 32), -1, dtype=torch.int32, device="cuda")
    assert call(data.data_ptr(), out.data_ptr(), status.data_ptr(), steps, starved, hole, limit, begun.data_ptr(), index, torch.cuda.current_stream().cuda_stream) == 0
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


INDEX = 11


@pytest.mark.parametrize("index", [1, 2])
def test_an_index_outside_does_not_hide_a_wait(index):
    """Reported before a wait gives up, or after; without one it stands."""
    assert int(run(50, index=index)[2]) == INDEX
    for starved in (0, 2, 4):
        assert int(run(50, starved, 7, index=index)[2]) == SITE


@pytest.mark.parametrize("W", [4, 40])
def test_what_stands_in_the_status_word_stays(W):
    """Parents and sources outside, where a wait has left its code that the host has not read yet: through the C calls, on a word of their own."""
    lib = native.lib()
    lib.lethe_gdn_reorder_states.argtypes = [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p, ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p]
    stream = torch.cuda.current_stream().cuda_stream
    for row in (64, 5):
        t = torch.randn(W, row, device="cuda")
        before = t.clone()
        parents = torch.arange(W, device="cuda")
        parents[1], parents[2] = W, -1
        s = (States * 1)(States(t.data_ptr(), 4 * row, 4 * row, 4 * row * W))
        for was in (0, 213, INDEX):
            status = torch.tensor([was], dtype=torch.int32, device="cuda")
            assert lib.lethe_gdn_reorder_states(s, 1, 1, W, parents.data_ptr(), 1, status.data_ptr(), stream) == 0
            assert int(status) == (was or INDEX) and torch.equal(t, before)


@pytest.mark.parametrize("B,V", [(3, 64), (400, 128)])
def test_a_step_leaves_the_status_word_too(B, V):
    call = native.lib().lethe_gdn_decode_step_from
    call.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
    q, v, state, out = (torch.randn(B, 2, *n, device="cuda") for n in ((128,), (V,), (128, V), (128, V)))
    o = torch.empty(B, 2, V, dtype=torch.bfloat16, device="cuda")
    source = torch.arange(B, device="cuda")
    source[1] = B
    a = ops._DecodeArgs(B=B, H=2, K=128, V=V, gate=0, delta=0, scale=1.0, q=q.data_ptr(), k=q.data_ptr(), v=v.data_ptr(), state=state.data_ptr(), o=o.data_ptr(), in_f32=1)
    for was in (0, 213):
        status = torch.tensor([was], dtype=torch.int32, device="cuda")
        assert call(ctypes.addressof(a), B, source.data_ptr(), 1, out.data_ptr(), status.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        assert int(status) == (was or INDEX)
