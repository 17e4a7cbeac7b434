"""GPU: which rows the norms around a block sum over: places of a CTA that no row fills, rows of the last turn."""
import pytest
import torch

from lethe_b200 import ops

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


# several turns of the CTAs, the last one not full, and every number of rows of a CTA
MANY = [(70001, 16), (20011, 64), (9001, 250), (2501, 1024), (2501, 700), (1501, 2048), (601, 8192)]


@pytest.mark.parametrize("rows,D", MANY)
def test_every_row_counts_once_in_the_sums_over_rows(rows, D):
    """A gradient that is zero but for one row: the sums are that row's terms, to the bit (what is added to them is zeros)."""
    x, z = randn(rows, D, seed=1, dt=torch.bfloat16), randn(rows, D, seed=2, dt=torch.bfloat16)
    vectors = [randn(D, seed=i) for i in (3, 4, 5)]

    def sums(x, z, dy):
        w, sc, pw = (v.clone().requires_grad_(True) for v in vectors)
        y, r = ops.residual_norm(x, z, w, scale=sc, post_weight=pw)
        plain, _ = ops.residual_norm(x, z, w, scale=sc)
        return [*torch.autograd.grad(ops.gated_norm(x, z, w), w, dy), *torch.autograd.grad((y, r), (w, sc, pw), (dy, dy)), *torch.autograd.grad(plain, (w, sc), dy)]
    dy = torch.zeros_like(x)
    for i in (0, 1, 31, rows // 3, rows // 2, rows - 17, rows - 2, rows - 1):
        dy[i] = 1
        for got, want in zip(sums(x, z, dy), sums(x[i:i + 1].clone(), z[i:i + 1].clone(), dy[i:i + 1].clone())):
            assert bool((want != 0).any()) and torch.equal(got, want), i
        dy[i] = 0


def test_as_many_inner_rows_as_32_bits_count():
    """Close to 2^31 rows of each of two: places are summed beyond what a signed number holds, and the step from one to the other comes behind that."""
    inner = (1 << 31) - 1000
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("40 GB of memory")
    gate = torch.empty(2, 1 << 31, 1, dtype=torch.bfloat16, device="cuda")
    for part in gate.view(-1).split(1 << 28):
        part.uniform_(-3, 3)
    z = gate[:, 1000:]
    x = torch.ones(2, inner, 1, dtype=torch.bfloat16, device="cuda")
    with torch.no_grad():
        y = ops.gated_norm(x, z, torch.ones(1, device="cuda"), activation="sigmoid")
    for o in (0, 1):
        for part in (slice(0, 30000), slice(1 << 30, (1 << 30) + 30000), slice(inner - 30000, inner)):
            want = torch.sigmoid(z[o, part].double()) / (1 + 1e-6) ** 0.5
            assert bool(((y[o, part].double() - want).abs() <= 2 ** -8 * 1.01 * want).all()), (o, part)
    del gate, z, x, y
    torch.cuda.empty_cache()
