"""CPU: the C calls of decoding with several hypotheses refuse results in the memory of what other CTAs still read, before they touch a GPU, and take
states of any size that a GPU holds."""
import ctypes

import pytest
import torch

from lethe_b200 import _build, native, ops

from .test_beam_cabi_cpu import ONE, States, beam, refused

# The addresses are none: with a GPU, a call that is not refused would run on them.
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="only where no kernel can be launched")
I32, I64, P = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    _build.build()
    L = native.lib()
    L.lethe_gdn_reorder_states.argtypes = [P, I32, I64, I32, P, I32, P, P]
    L.lethe_gdn_fork_states.argtypes = [P, I32, I64, P, P, I32, I64, P, P, P, P]
    L.lethe_gdn_compact_states.argtypes = [P, I32, I64, P, P, P, P, P]
    L.lethe_gdn_decode_step_from.argtypes = [P, I64, P, I32, P, P, P]
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


def test_beam_select(lib):
    B, W = 2, 3
    size = dict(scores=4, penalty=4, finished=1, out_scores=4, parents=8, tokens=8, out_finished=1)
    at = dict(scores=0x20000, penalty=0x21000, finished=0x22000, out_scores=0x30000, parents=0x40000, tokens=0x50000, out_finished=0x60000, work=0x70000)
    work_bytes = lambda k: lib.lethe_gdn_beam_work_bytes(B, W, 100, k, 0)      # noqa: E731
    call = lambda k, **kw: lib.lethe_gdn_beam_select(ctypes.byref(beam(**{**at, **dict(B=B, W=W, k=k, eos=7, work_bytes=work_bytes(k)), **kw})), None)      # noqa: E731
    rows = lambda n, k: size[n] * B * (W if n in ("scores", "penalty", "finished") else k)      # noqa: E731
    outs, ins = ("out_scores", "parents", "tokens", "out_finished"), ("scores", "penalty", "finished")
    for k in (3, 5):
        passed(lib, call(k))
        need = work_bytes(k)
        for o in outs:
            for other in (*ins, *outs):
                if o == other:
                    continue
                # (results of eight bytes lie on boundaries of eight)
                for place in (at[other], at[other] + (rows(other, k) - 1) // 8 * 8, at[other] - (rows(o, k) - 1) // 8 * 8):
                    own = place == at[other] and k == W and (o, other) in (("out_scores", "scores"), ("out_scores", "penalty"), ("out_finished", "finished"))
                    if own:
                        passed(lib, call(k, **{o: place}))
                    else:
                        refused(lib, call(k, **{o: place}), b"memory of what is read")
                passed(lib, call(k, **{o: at[other] + (rows(other, k) + 7) // 8 * 8}))
        for n in (*ins, *outs):
            refused(lib, call(k, **{n: at["work"] + need // 8 * 8 - 8}), b"memory of what is read")
            passed(lib, call(k, **{n: at["work"] + need}))


def test_decode_step_from(lib):
    B, H, V = 2, 2, 64
    base = dict(B=B, H=H, K=128, V=V, gate=2, delta=1, scale=1.0, q=0x1000000, k=0x1100000, v=0x1200000, g=0x1300000, beta=0x1400000, state=0x2000000, o=0x1500000)
    out, row = 0x9000000, H * 128 * V * 4

    def call(source=0x1600000, s64=1, **kw):
        a = ops._DecodeArgs(**{**base, **kw})
        return lib.lethe_gdn_decode_step_from(ctypes.byref(a), 4, source, s64, out, 0x1700000, None)
    passed(lib, call())
    size = dict(q=2 * B * H * 128, k=2 * B * H * 128, v=2 * B * H * V, g=4 * B * H * 128, beta=4 * B * H, o=2 * B * H * V)
    for n, e in size.items():
        for place in (out, out + B * row - 4, out - e + 4):
            refused(lib, call(**{n: place}), b"memory of what is read")
        for place in (out + B * row, out - e):
            passed(lib, call(**{n: place}))
    refused(lib, call(in_f32=1, q=out - size["q"]), b"memory of what is read")
    refused(lib, call(source=out + 8), b"memory of what is read")
    refused(lib, call(source=out - 8), b"memory of what is read")
    passed(lib, call(source=out - 8, s64=0))


def test_large_states(lib):
    """12 MB rows of 512 groups, one row of 100 GB, more groups than a grid has CTAs."""
    for W in (2, 4, 32, 33, 256):
        for B, row in ((512, 12 << 20), (128, 32 << 20), (1, 100 << 30), (2, 1 << 37), (1 << 30, 1 << 10), (3, (5 << 30) + 4)):
            s = (States * 2)(States(0x10000, row, row, row * W), States(0x10000 + row * W * B, 64, 64, 64 * W))
            passed(lib, lib.lethe_gdn_reorder_states(s, 2, B, W, 0x20000, 1, 0x30000, None))
        for B, row in ((1, (1 << 38) + 1), (1 << 30, 1 << 36)):
            refused(lib, lib.lethe_gdn_reorder_states((States * 1)(States(0x10000, row, row, row * W)), 1, B, W, 0x20000, 1, 0x30000, None), b"sizes")
