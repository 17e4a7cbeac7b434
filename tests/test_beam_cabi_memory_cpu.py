"""CPU: the C calls of decoding with several hypotheses refuse results in the memory of what other CTAs still read, before they touch a GPU."""
import ctypes

import pytest
import torch

from lethe_b200 import _build, native

from .test_beam_cabi_cpu import ONE, refused

# The addresses are none: with a GPU, a call that is not refused would run on them.
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="only where no kernel can be launched")
I32, I64, P = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    _build.build()
    L = native.lib()
    L.lethe_gdn_fork_states.argtypes = [P, I32, I64, P, P, I32, I64, P, P, P, P]
    L.lethe_gdn_compact_states.argtypes = [P, I32, I64, P, P, P, P, P]
    return L


def passed(lib, rc):
    """As far as the look for the GPU of an address that is none."""
    assert rc == 9, (rc, lib.lethe_gdn_strerror(rc))


def test_fork_states(lib):
    S, n = 64, 16
    call = lambda live=0x20000, src=0x30000, s64=1, t=0x40000, after=0x50000: lib.lethe_gdn_fork_states(ONE, 1, S, live, src, s64, n, t, after, 0x60000, None)      # noqa: E731
    for bad in (dict(after=0x20000), dict(after=0x20000 + S - 1), dict(after=0x20000 - S + 1), dict(after=0x30000), dict(after=0x30000 + 8 * n - 1), dict(after=0x30000 + 4 * n - 1, s64=0),
                dict(after=0x40000), dict(after=0x40000 + 8 * n - 1), dict(t=0x20000), dict(t=0x20000 + S - 8), dict(t=0x20000 - 8 * n + 8), dict(t=0x30000), dict(t=0x30000, s64=0)):
        refused(lib, call(**bad), b"memory of what is read")
    for good in (dict(), dict(after=0x20000 + S), dict(after=0x20000 - S), dict(after=0x30000 + 8 * n), dict(after=0x30000 + 4 * n, s64=0), dict(after=0x40000 + 8 * n), dict(t=0x20000 + S),
                 dict(live=0x30000 + 8 * n)):
        passed(lib, call(**good))


def test_compact_states(lib):
    S = 64
    call = lambda live=0x20000, place=0x30000, count=0x40000: lib.lethe_gdn_compact_states(ONE, 1, S, live, place, count, 0x50000, None)      # noqa: E731
    for bad in (dict(place=0x20000), dict(place=0x20000 + S - 8), dict(place=0x20000 - 8 * S + 8), dict(count=0x20000), dict(count=0x20000 + S - 8), dict(count=0x30000),
                dict(count=0x30000 + 8 * S - 8)):
        refused(lib, call(**bad), b"memory of what is read")
    for good in (dict(), dict(place=0x20000 + S), dict(place=0x20000 - 8 * S), dict(count=0x20000 + S), dict(count=0x20000 - 8), dict(count=0x30000 + 8 * S)):
        passed(lib, call(**good))
