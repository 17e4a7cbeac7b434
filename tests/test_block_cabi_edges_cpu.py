"""CPU: further arguments that the C calls beside the recurrence refuse before they touch a GPU."""
import pytest

from .test_block_cabi_cpu import diag, gated, lib, refused, residual  # noqa: F401  (lib: the fixture)

NORMS = [("lethe_gdn_gated_norm", gated), ("lethe_gdn_gated_norm_vjp", gated), ("lethe_gdn_residual_norm", residual), ("lethe_gdn_residual_norm_vjp", residual)]


@pytest.mark.parametrize("call,make", NORMS)
def test_an_infinite_eps(lib, call, make):      # noqa: F811
    refused(lib, call, make(eps=float("inf")), b"sizes")
