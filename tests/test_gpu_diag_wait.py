"""GPU: a wait of the element-wise recurrence that runs out ends the kernel, leaves its code, and lets everybody pass."""
import ctypes

import pytest
import torch

from lethe_b200 import _build, ops

pytestmark = pytest.mark.gpu


def test_a_word_that_nobody_writes():
    call = ctypes.CDLL(_build.build_probe()).lethe_probe_look_wait
    call.argtypes = [ctypes.c_void_p] * 3 + [ctypes.c_longlong] + [ctypes.c_void_p] * 3
    words = torch.full((64,), -1, dtype=torch.int64, device="cuda")
    head = torch.full((2,), -1, dtype=torch.int32, device="cuda")
    status, trace = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((2,), -1, dtype=torch.int32, device="cuda")
    got = torch.full((64,), 7, dtype=torch.int64, device="cuda")
    limit = 2_000_000
    rc = call(words.data_ptr(), head.data_ptr(), status.data_ptr(), limit, trace.data_ptr(), got.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert int(status) == 900 and head.tolist() == [-1, 0] and bool((got == 0).all())
    first, second = trace.tolist()
    assert limit // 1024 <= first <= 20 * limit // 1024
    assert second <= 200                                      # some 32 looks at the word, one at the word that lets everybody pass
    with pytest.raises(ops.GdnError, match="900"):
        ops.check_status(status)
    # the context is intact
    x, g = torch.randn(1, 5000, 64, device="cuda"), -torch.rand(1, 5000, 64, device="cuda")
    assert bool(ops.diag_scan(x, g)[0].isfinite().all())
