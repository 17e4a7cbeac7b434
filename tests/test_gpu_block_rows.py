"""GPU: which rows the norms around a block sum over: places of a CTA that no row fills, rows of the last turn."""
import pytest
import torch

from .test_gpu_block_norms import gated_check, randn, residual_check, residual_inputs

pytestmark = pytest.mark.gpu

# rows that do not fill the CTAs' places (16 rows of up to 128 values, 8 of 256, 2 of 1024 at once, 1 of more)
SPARE = [(1, 64), (3, 64), (17, 128), (260, 100), (9, 200), (5, 1000), (3, 8192)]


@pytest.mark.parametrize("eps", [0.0, 1e-60])      # (which is 0 in fp32)
@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("rows,D", SPARE)
def test_gated_norm_without_eps(rows, D, types, eps):
    xt, wt = types
    for act in ("silu", "sigmoid"):
        gated_check(randn(rows, D, seed=1, dt=xt), randn(rows, D, seed=2, dt=xt), randn(D, seed=3, dt=wt), randn(rows, D, seed=4, dt=xt), eps=eps, act=act)


@pytest.mark.parametrize("eps", [0.0, 1e-60])
@pytest.mark.parametrize("scale,post", [("none", False), ("number", True), ("vector", False), ("vector", True)])
@pytest.mark.parametrize("rows,D", SPARE)
def test_residual_norm_without_eps(rows, D, scale, post, eps):
    for types in ((torch.float32, torch.float32, torch.float32), (torch.bfloat16, torch.float32, torch.float32), (torch.float16, torch.float16, torch.float16)):
        residual_check(*residual_inputs((rows, D), *types, scale, post), eps=eps)
