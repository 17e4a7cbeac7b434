"""CPU: further arguments that the C calls beside the recurrence refuse before they touch a GPU."""
import ctypes

import pytest

from .test_block_cabi_cpu import diag, gated, lib, refused, residual  # noqa: F401  (lib: the fixture)

NORMS = [("lethe_gdn_gated_norm", gated), ("lethe_gdn_gated_norm_vjp", gated), ("lethe_gdn_residual_norm", residual), ("lethe_gdn_residual_norm_vjp", residual)]


@pytest.mark.parametrize("call,make", NORMS)
def test_an_infinite_eps(lib, call, make):      # noqa: F811
    refused(lib, call, make(eps=float("inf")), b"sizes")


def off(make, name, by, **more):
    """The arguments with one pointer `by` bytes past a boundary."""
    a = make(**more)
    setattr(a, name, (getattr(a, name) or 0x900000) + by)
    return a


@pytest.mark.parametrize("call", ["lethe_gdn_diag_forward", "lethe_gdn_diag_backward"])
def test_diag_pointers_between_elements(lib, call):      # noqa: F811
    for types in (dict(x_type=0, g_type=0), dict(x_type=1, g_type=0), dict(x_type=2, g_type=2)):
        for n in ("x", "h", "d_h", "dx"):
            refused(lib, call, off(diag, n, 2 if types["x_type"] == 0 else 1, **types), b"align")
        for n in ("g", "dg"):
            refused(lib, call, off(diag, n, 2 if types["g_type"] == 0 else 1, **types), b"align")
        for n in ("h0", "hT", "states", "dhT", "dh0", "status"):
            refused(lib, call, off(diag, n, 2, **types), b"align")


def test_diag_step_pointers_between_elements(lib):      # noqa: F811
    state = ctypes.c_void_p(0x70000)
    for n in ("x", "h", "g"):
        refused(lib, "lethe_gdn_diag_step", off(diag, n, 2), b"align", state)
    refused(lib, "lethe_gdn_diag_step", diag(), b"align", ctypes.c_void_p(0x70002))


@pytest.mark.parametrize("call", ["lethe_gdn_gated_norm", "lethe_gdn_gated_norm_vjp"])
def test_gated_pointers_between_elements(lib, call):      # noqa: F811
    for types in (dict(x_type=0, w_type=0), dict(x_type=1, w_type=0), dict(x_type=2, w_type=2)):
        for n in ("x", "gate", "y", "dy", "dx", "dgate"):
            refused(lib, call, off(gated, n, 2 if types["x_type"] == 0 else 1, **types), b"align")
        for n in ("weight", "dweight"):
            refused(lib, call, off(gated, n, 2 if types["w_type"] == 0 else 1, **types), b"align")


@pytest.mark.parametrize("call", ["lethe_gdn_residual_norm", "lethe_gdn_residual_norm_vjp"])
def test_residual_pointers_between_elements(lib, call):      # noqa: F811
    for types in (dict(x_type=0, r_type=0, w_type=0), dict(x_type=1, r_type=0, w_type=0), dict(x_type=2, r_type=2, w_type=2)):
        for n in ("x", "y", "dy", "dx"):
            refused(lib, call, off(residual, n, 2 if types["x_type"] == 0 else 1, **types), b"align")
        for n in ("residual", "r", "dr", "dresidual"):
            refused(lib, call, off(residual, n, 2 if types["r_type"] == 0 else 1, **types), b"align")
        for n in ("weight", "post_weight", "scale", "dweight", "dpost_weight", "dscale"):
            refused(lib, call, off(residual, n, 2 if types["w_type"] == 0 else 1, **types), b"align")


END = (1 << 63) - 1


@pytest.mark.parametrize("call", ["lethe_gdn_diag_forward", "lethe_gdn_diag_backward"])
def test_diag_sizes_at_the_end_of_64_bits(lib, call):      # noqa: F811
    for bad in (dict(L=END), dict(L=END - 60), dict(D=END), dict(D=END - 60), dict(B=END), dict(B=END, L=END, D=END)):
        refused(lib, call, diag(**bad), b"sizes")


def test_diag_step_sizes_at_the_end_of_64_bits(lib):      # noqa: F811
    for bad in (dict(D=END), dict(D=END - 200), dict(B=END), dict(B=END, D=END)):
        refused(lib, "lethe_gdn_diag_step", diag(**bad), b"sizes", ctypes.c_void_p(0x70000))


def test_diag_work_of_sizes_that_are_refused(lib):      # noqa: F811
    for bad in ((END, 1000, 64), (1, END, 64), (1, 1000, END), (1 << 40, 1 << 40, 1)):
        assert lib.lethe_gdn_diag_work_bytes(*bad, 1, 0) == 0
