"""CPU: the C calls beside the recurrence reject bad arguments before they touch a GPU, and the PyTorch surface tensors that are not on one."""
import ctypes

import pytest
import torch

from lethe_b200 import _build, native, ops

I32, I64, P, F, Z = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float, ctypes.c_size_t


class Diag(ctypes.Structure):
    _fields_ = [("B", I64), ("L", I64), ("D", I64), ("x_type", I32), ("g_type", I32), ("complement", I32), ("x", P), ("x_batch", I64), ("x_token", I64),
                ("g", P), ("g_batch", I64), ("g_token", I64), ("h0", P), ("h", P), ("hT", P), ("states", P), ("d_h", P), ("d_h_batch", I64), ("d_h_token", I64),
                ("dhT", P), ("dx", P), ("dg", P), ("dh0", P), ("work", P), ("work_bytes", Z), ("status", P)]


class Gated(ctypes.Structure):
    _fields_ = [("rows", I64), ("inner", I64), ("D", I32), ("x_type", I32), ("w_type", I32), ("silu", I32), ("eps", F), ("x", P), ("x_outer", I64), ("x_inner", I64),
                ("gate", P), ("gate_outer", I64), ("gate_inner", I64), ("weight", P), ("y", P), ("dy", P), ("dx", P), ("dgate", P), ("dweight", P), ("work", P), ("work_bytes", Z)]


class Residual(ctypes.Structure):
    _fields_ = [("rows", I64), ("D", I32), ("x_type", I32), ("r_type", I32), ("w_type", I32), ("eps", F), ("scale_value", F), ("x", P), ("x_stride", I64),
                ("residual", P), ("residual_stride", I64), ("weight", P), ("post_weight", P), ("scale", P), ("r", P), ("y", P), ("dy", P), ("dr", P), ("dx", P),
                ("dresidual", P), ("dweight", P), ("dpost_weight", P), ("dscale", P), ("work", P), ("work_bytes", Z)]


@pytest.fixture(scope="module")
def lib():
    _build.build()
    L = native.lib()
    L.lethe_gdn_diag_states_bytes.restype, L.lethe_gdn_diag_states_bytes.argtypes = Z, [I64, I64, I64, I32]
    L.lethe_gdn_diag_work_bytes.restype, L.lethe_gdn_diag_work_bytes.argtypes = Z, [I64, I64, I64, I32, I32]
    L.lethe_gdn_norm_work_bytes.restype, L.lethe_gdn_norm_work_bytes.argtypes = Z, [I64, I32, I32]
    return L


def refused(lib, call, a, word, *more):
    rc = getattr(lib, call)(ctypes.byref(a), *more, None)
    assert rc != 0 and word in lib.lethe_gdn_strerror(rc), (call, rc)


def diag(**kw):
    base = dict(B=1, L=4, D=8, x=0x10000, g=0x20000, h=0x30000, states=0x40000, status=0x50000, x_batch=32, x_token=8, g_batch=32, g_token=8, work=0x60000, work_bytes=1 << 30)
    base.update(kw)
    return Diag(**base)


@pytest.mark.parametrize("call", ["lethe_gdn_diag_forward", "lethe_gdn_diag_backward"])
def test_diag(lib, call):
    for n in ("x", "g", "status"):
        refused(lib, call, diag(**{n: None}), b"null")
    refused(lib, call, diag(h=None, states=None), b"null")
    for bad in (dict(B=0), dict(L=0), dict(D=0), dict(L=-3), dict(x_type=3), dict(x_type=1, g_type=2), dict(x_type=0, g_type=1), dict(B=1 << 40), dict(L=1 << 60), dict(D=1 << 50)):
        refused(lib, call, diag(**bad), b"sizes")
    assert getattr(lib, call)(None, None) != 0


def test_diag_step(lib):
    state = P(0x70000)
    refused(lib, "lethe_gdn_diag_step", diag(x=None), b"null", state)
    refused(lib, "lethe_gdn_diag_step", diag(), b"null", None)
    refused(lib, "lethe_gdn_diag_step", diag(D=0), b"sizes", state)
    refused(lib, "lethe_gdn_diag_step", diag(B=1 << 40), b"sizes", state)
    refused(lib, "lethe_gdn_diag_step", diag(g_type=1), b"sizes", state)


def test_sizes(lib):
    assert lib.lethe_gdn_diag_states_bytes(2, 300, 10, 1) == 2 * 5 * 10 * 4          # one for every 64 tokens
    assert lib.lethe_gdn_diag_states_bytes(2, 300, 10, 0) == 2 * 7 * 10 * 4          # fp32: 48
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (-1, 1, 1)):
        assert lib.lethe_gdn_diag_states_bytes(*bad, 1) == 0 and lib.lethe_gdn_diag_work_bytes(*bad, 1, 0) == 0
    for back, tile in ((0, 128), (1, 64)):                                            # one tile: nothing to hand on
        assert lib.lethe_gdn_diag_work_bytes(1, tile, 64, 1, back) == 0
        assert lib.lethe_gdn_diag_work_bytes(1, tile + 1, 64, 1, back) == 128 + (2 + 1 + 1) * 64 * 8
    assert lib.lethe_gdn_norm_work_bytes(3, 100, 2) == 3 * 100 * 2 * 4
    assert lib.lethe_gdn_norm_work_bytes(1 << 40, 8192, 3) < 1 << 27     # bounded by the CTAs, not by the rows
    for bad in ((0, 8, 1), (4, 0, 1), (4, 8193, 1), (4, 8, 0), (4, 8, 4)):
        assert lib.lethe_gdn_norm_work_bytes(*bad) == 0


def gated(**kw):
    base = dict(rows=4, inner=1, D=64, eps=1e-6, x=0x10000, x_outer=64, gate=0x20000, gate_outer=64, weight=0x30000, y=0x40000, dy=0x50000, dx=0x60000, dgate=0x70000)
    base.update(kw)
    return Gated(**base)


@pytest.mark.parametrize("call", ["lethe_gdn_gated_norm", "lethe_gdn_gated_norm_vjp"])
def test_gated(lib, call):
    for n in ("x", "gate", "weight"):
        refused(lib, call, gated(**{n: None}), b"null")
    refused(lib, call, gated(y=None, dy=None), b"null")
    for bad in (dict(rows=0), dict(inner=0), dict(D=0), dict(D=8193), dict(x_type=5), dict(x_type=1, w_type=2), dict(eps=-1.0), dict(eps=float("nan"))):
        refused(lib, call, gated(**bad), b"sizes")


def test_gated_work(lib):
    call = "lethe_gdn_gated_norm_vjp"
    refused(lib, call, gated(dweight=0x80000), b"null")
    refused(lib, call, gated(dweight=0x80000, work=0x90000, work_bytes=4), b"workspace")
    refused(lib, call, gated(dweight=0x80000, work=0x90004, work_bytes=1 << 20), b"align")


def residual(**kw):
    base = dict(rows=4, D=64, eps=1e-6, scale_value=1.0, x=0x10000, x_stride=64, residual=0x20000, residual_stride=64, weight=0x30000, r=0x40000, y=0x50000, dy=0x60000, dr=0x70000)
    base.update(kw)
    return Residual(**base)


@pytest.mark.parametrize("call", ["lethe_gdn_residual_norm", "lethe_gdn_residual_norm_vjp"])
def test_residual(lib, call):
    for n in ("r", "weight"):
        refused(lib, call, residual(**{n: None}), b"null")
    for bad in (dict(rows=0), dict(D=0), dict(D=8193), dict(r_type=1), dict(x_type=1, r_type=2), dict(x_type=2, w_type=1), dict(eps=-1.0)):
        refused(lib, call, residual(**bad), b"sizes")


def test_residual_vjp(lib):
    call = "lethe_gdn_residual_norm_vjp"
    refused(lib, call, residual(x=None, post_weight=0x1000), b"null")
    refused(lib, call, residual(x=None, dscale=0x1000), b"null")
    refused(lib, call, residual(dpost_weight=0x1000, work=0x2000, work_bytes=1 << 20), b"combination")
    refused(lib, call, residual(dweight=0x1000, dscale=0x2000, work=0x90000, work_bytes=4 * 64 * 4), b"workspace")


def test_the_surface_refuses_tensors_on_the_host():
    x, w = torch.zeros(2, 3, 8), torch.zeros(8)
    for f in (lambda: ops.diag_scan(x, x), lambda: ops.diag_scan_step(x[:, 0], x[:, 0], x[:, 0].contiguous()), lambda: ops.gated_norm(x, x, w), lambda: ops.residual_norm(x, x, w)):
        with pytest.raises(ops.GdnError, match="CUDA device"):
            f()
