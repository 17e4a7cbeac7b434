"""GPU: the operators beside the recurrence together, as a model uses them: training, a prompt, single tokens, a captured step."""
import types

import pytest
import torch
import torch.nn.functional as F

from lethe_b200 import ops
from lethe_b200.tiny import TinyDiagLM, delayed_copy_batch

pytestmark = pytest.mark.gpu

# fp32 model against the same in fp64: products of up to 128 terms and some 20 operations one behind the other, each a few roundings of 2^-24
BOUND = 128 * 20 * 2.0 ** -24


def plain():
    """The operators as formulas, in the type of their inputs."""
    def scan(x, g, h0=None, *, complement=False):
        h, out = torch.zeros_like(x[:, 0]) if h0 is None else h0, []
        for t in range(x.shape[1]):
            a = torch.exp(g[:, t].to(x.dtype))
            h = a * h + ((1 - a) * x[:, t] if complement else x[:, t])
            out.append(h)
        return torch.stack(out, 1), h

    def rms(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)

    def residual_norm(x, residual, weight, *, scale=None, post_weight=None):
        r = (x if post_weight is None else rms(x) * post_weight) * (1 if scale is None else scale)
        r = r if residual is None else residual + r
        return rms(r) * weight, r
    return types.SimpleNamespace(diag_scan=scan, residual_norm=residual_norm, gated_norm=lambda x, z, w: rms(x) * w * F.silu(z))


def models(seed=0):
    torch.manual_seed(seed)
    mine = TinyDiagLM(ops).cuda()
    ref = TinyDiagLM(plain()).cuda().double()
    ref.load_state_dict({k: v.double() for k, v in mine.state_dict().items()})
    return mine, ref


def batch(B=3, L=150):
    x, y = delayed_copy_batch(B, L, 40, seed=1)
    return x.cuda(), y.cuda()


def test_training_gradients():
    mine, ref = models()
    x, y = batch()
    got, want = [], []
    for model, out in ((mine, got), (ref, want)):
        logits, _ = model(x)
        loss = F.cross_entropy(logits.flatten(0, 1), y.flatten())
        out += [logits, *torch.autograd.grad(loss, list(model.parameters()))]
    for a, b in zip(got, want):
        assert float((a.detach().double() - b.detach()).norm()) <= BOUND * float(b.detach().norm()) + 1e-9


def test_a_prompt_and_tokens_after_it():
    mine, ref = models(1)
    x, _ = batch()
    with torch.no_grad():
        want, _ = ref(x)
        logits, states = mine(x[:, :131])
        for t in range(131, 150):
            step, states = mine(x[:, t], states)
            assert float((step.double() - want[:, t]).norm()) <= BOUND * float(want[:, t].norm())
        assert float((logits.double() - want[:, :131]).norm()) <= BOUND * float(want[:, :131].norm())


def test_a_captured_training_step_gives_the_gradients_of_the_eager_one():
    mine, _ = models(2)
    x, y = batch()
    params = list(mine.parameters())

    def step():
        logits, _ = mine(x)
        return torch.autograd.grad(F.cross_entropy(logits.flatten(0, 1), y.flatten()), params)
    want = [t.clone() for t in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert float((a - b).norm()) <= BOUND * float(b.norm()) + 1e-9      # (the library's matrix products may choose otherwise under capture)


def test_beside_the_chunked_op():
    """The norms around gdn_chunk, in bf16 with the stream in fp32: what it returns goes through as it lies, gradients reach all inputs."""
    gen = torch.Generator().manual_seed(3)
    def rand(*s, dt=torch.bfloat16):
        return torch.randn(*s, generator=gen).to("cuda", dt).requires_grad_(True)
    B, L, H, K, V = 2, 128, 2, 128, 64
    x, stream, w, wo = rand(B, L, 256), rand(B, L, 256, dt=torch.float32), rand(256), rand(V)
    maps = rand(256, H * (2 * K + 2 * V))
    y, r = ops.residual_norm(x, stream, w, scale=0.5)
    q, k, v, z = (y @ maps * 0.05).split([H * K, H * K, H * V, H * V], -1)
    o, _ = ops.gdn_chunk(q.unflatten(-1, (H, K)), k.unflatten(-1, (H, K)), v.unflatten(-1, (H, V)), -torch.rand(B, L, H, device="cuda"), torch.rand(B, L, H, device="cuda"),
                         use_qk_l2norm=True)
    u = ops.gated_norm(o, z.unflatten(-1, (H, V)), wo)
    grads = torch.autograd.grad(u.float().square().sum() + r.sum(), (x, stream, w, wo, maps))
    assert u.dtype == torch.bfloat16 and r.dtype == torch.float32
    assert all(bool(t.isfinite().all()) and float(t.float().norm()) > 0 for t in grads)
