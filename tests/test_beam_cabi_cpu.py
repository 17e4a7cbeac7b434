"""CPU: the C calls of decoding with several hypotheses reject bad arguments before they touch a GPU, and the PyTorch surface tensors that are not on one."""
import ctypes

import pytest
import torch

from lethe_b200 import _build, native, ops

I32, I64, P, D, F, Z, U32 = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_double, ctypes.c_float, ctypes.c_size_t, ctypes.c_uint32


class Beam(ctypes.Structure):
    _fields_ = [("B", I64), ("V", I64), ("W", I32), ("k", I32), ("x_type", I32), ("temperature", D), ("logits", P), ("logits_batch", I64), ("logits_beam", I64),
                ("allowed", P), ("allowed_batch", I64), ("allowed_beam", I64), ("scores", P), ("finished", P), ("penalty", P), ("eos", I64), ("out_scores", P),
                ("parents", P), ("tokens", P), ("out_finished", P), ("work", P), ("work_bytes", Z)]


class States(ctypes.Structure):
    _fields_ = [("data", P), ("row_bytes", I64), ("stride", I64), ("group_stride", I64)]


@pytest.fixture(scope="module")
def lib():
    _build.build()
    L = native.lib()
    L.lethe_gdn_beam_work_bytes.restype, L.lethe_gdn_beam_work_bytes.argtypes = Z, [I64, I32, I64, I32, I32]
    L.lethe_gdn_reorder_states.argtypes = [P, I32, I64, I32, P, I32, P, P]
    L.lethe_gdn_fork_states.argtypes = [P, I32, I64, P, P, I32, I64, P, P, P, P]
    L.lethe_gdn_compact_states.argtypes = [P, I32, I64, P, P, P, P, P]
    L.lethe_gdn_decode_step_from.argtypes = [P, I64, P, I32, P, P, P]
    return L


def refused(lib, rc, word):
    assert rc != 0 and word in lib.lethe_gdn_strerror(rc), (rc, lib.lethe_gdn_strerror(rc))


def beam(**kw):
    base = dict(B=2, V=100, W=3, k=3, temperature=1.0, logits=0x10000, logits_batch=300, logits_beam=100, scores=0x20000, eos=-1, out_scores=0x30000, parents=0x40000,
                tokens=0x50000, work=0x60000, work_bytes=1 << 30)
    base.update(kw)
    return Beam(**base)


def test_beam_select(lib):
    call = lambda **kw: lib.lethe_gdn_beam_select(ctypes.byref(beam(**kw)), None)      # noqa: E731
    for n in ("logits", "scores", "out_scores", "parents", "tokens", "work"):
        refused(lib, call(**{n: None}), b"null")
    for bad in (dict(B=0), dict(B=1 << 40), dict(V=0), dict(V=(1 << 30) + 1), dict(W=0), dict(W=65), dict(k=0), dict(k=65), dict(x_type=3), dict(x_type=-1), dict(eos=100),
                dict(eos=-2), dict(finished=0x1000), dict(out_finished=0x1000), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
                dict(temperature=float("inf")), dict(B=1 << 20, W=64, V=1 << 30)):
        refused(lib, call(**bad), b"sizes")
    for bad in (dict(logits=0x10002), dict(x_type=1, logits=0x10001), dict(scores=0x20002), dict(penalty=0x1001), dict(parents=0x40004), dict(work=0x60008), dict(out_scores=0x30001)):
        refused(lib, call(**bad), b"align")
    refused(lib, call(work_bytes=lib.lethe_gdn_beam_work_bytes(2, 3, 100, 3, 0) - 1), b"workspace")
    assert lib.lethe_gdn_beam_select(None, None) != 0


def test_beam_work_bytes(lib):
    assert lib.lethe_gdn_beam_work_bytes(2, 3, 100, 3, 0) == 6 * (16 + 8 * 20)           # a list a row, of 16 more than asked for, made even
    assert lib.lethe_gdn_beam_work_bytes(2, 3, 1021, 3, 0) == 6 * (16 + 8 * 20)          # 1024 logits a list, the row up to 3 behind a 16-byte boundary
    assert lib.lethe_gdn_beam_work_bytes(2, 3, 1022, 3, 0) == 12 * (16 + 8 * 20)
    assert lib.lethe_gdn_beam_work_bytes(2, 3, 1017, 3, 1) == 6 * (16 + 8 * 20)          # 16 bits: up to 7
    assert lib.lethe_gdn_beam_work_bytes(2, 3, 1018, 3, 1) == 12 * (16 + 8 * 20)
    assert lib.lethe_gdn_beam_work_bytes(1, 1, 2000, 33, 1) == 16 + 8 * 50                # more candidates than lanes: two tiles at least
    for bad in ((0, 1, 1, 1, 0), (1, 0, 1, 1, 0), (1, 65, 1, 1, 0), (1, 1, 0, 1, 0), (1, 1, 1, 0, 0), (1, 1, 1, 65, 0), (1, 1, 1, 1, 3)):
        assert lib.lethe_gdn_beam_work_bytes(*bad) == 0


ONE = (States * 1)(States(0x10000, 64, 64, 256))


def test_reorder_states(lib):
    call = lambda s=ONE, n=1, B=2, W=4, p=0x20000, p64=1, status=0x30000: lib.lethe_gdn_reorder_states(s, n, B, W, p, p64, status, None)      # noqa: E731
    for bad in (dict(s=None), dict(p=None), dict(status=None), dict(n=0), dict(n=-1), dict(s=(States * 1)(States(None, 64, 64, 256)))):
        refused(lib, call(**bad), b"null")
    for bad in (dict(B=0), dict(W=0), dict(W=257), dict(B=1 << 40), dict(s=(States * 1)(States(0x10000, 0, 64, 256))), dict(s=(States * 1)(States(0x10000, -8, 64, 256))),
                dict(s=(States * 1)(States(0x10000, 1 << 41, 64, 256)))):
        refused(lib, call(**bad), b"sizes")
    refused(lib, call(p=0x20004), b"align")
    refused(lib, call(p=0x20002, p64=0), b"align")


def test_fork_states(lib):
    call = lambda s=ONE, n=1, S=8, live=0x20000, src=0x30000, s64=1, e=3, t=0x40000, after=0x50000, status=0x60000: lib.lethe_gdn_fork_states(s, n, S, live, src, s64, e, t, after, status, None)      # noqa: E731
    for bad in (dict(s=None), dict(live=None), dict(src=None), dict(t=None), dict(after=None), dict(status=None), dict(n=-1)):
        refused(lib, call(**bad), b"null")
    for bad in (dict(S=0), dict(S=65537), dict(e=0), dict(e=4097), dict(s=(States * 1)(States(0x10000, 0, 64, 0)))):
        refused(lib, call(**bad), b"sizes")
    for bad in (dict(src=0x30004), dict(src=0x30001, s64=0), dict(t=0x40004)):
        refused(lib, call(**bad), b"align")


def test_compact_states(lib):
    call = lambda s=ONE, n=1, S=8, live=0x20000, place=0x30000, count=0x40000, status=0x50000: lib.lethe_gdn_compact_states(s, n, S, live, place, count, status, None)      # noqa: E731
    for bad in (dict(s=None), dict(live=None), dict(place=None), dict(count=None), dict(status=None), dict(n=-1)):
        refused(lib, call(**bad), b"null")
    for bad in (dict(S=0), dict(S=65537)):
        refused(lib, call(**bad), b"sizes")
    for bad in (dict(place=0x30004), dict(count=0x40001)):
        refused(lib, call(**bad), b"align")


def test_decode_step_from(lib):
    def call(slots=4, source=0x70000, s64=1, out=0x9000000, status=0x90000, **kw):
        base = dict(B=2, H=2, K=128, V=64, gate=0, delta=0, scale=1.0, q=0x10000, k=0x20000, v=0x30000, state=0x40000, o=0x50000)
        base.update(kw)
        a = ops._DecodeArgs(**base)
        return lib.lethe_gdn_decode_step_from(ctypes.byref(a), slots, source, s64, out, status, None)
    for bad in (dict(source=None), dict(out=None), dict(status=None), dict(state=None), dict(q=None), dict(gate=1), dict(delta=1)):
        refused(lib, call(**bad), b"null")
    for bad in (dict(slots=0), dict(slots=1 << 60), dict(K=64), dict(V=32), dict(B=0), dict(B=1 << 30)):
        refused(lib, call(**bad), b"sizes")
    for bad in (dict(source=0x70004), dict(source=0x70002, s64=0), dict(out=0x9000002), dict(state=0x40002)):
        refused(lib, call(**bad), b"align")
    row = 2 * 128 * 64 * 4
    for out in (0x40000, 0x40000 + 4 * row - 4, 0x40000 - 2 * row + 4):      # in the state's memory, at both ends
        refused(lib, call(out=out), b"combination")


def test_the_surface_refuses_tensors_on_the_host():
    x, i = torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.long)
    live = torch.zeros(2, dtype=torch.bool)
    s = torch.zeros(2, 1, 128, 64)
    q, v = torch.zeros(2, 1, 128), torch.zeros(2, 1, 64)
    for f in (lambda: ops.beam_select(x, x[..., 0]), lambda: ops.reorder_states(x.view(6, 8), i), lambda: ops.fork_states(x, live, i[0]), lambda: ops.compact_states([x], live),
              lambda: ops.gdn_decode_step(q, q, v, None, None, s, source=i[:, 0], out=s.clone())):
        with pytest.raises(ops.GdnError, match="CUDA device"):
            f()
