"""GPU: the C call of the selection with as many candidates as beams, whose results take the place of what it reads."""
import ctypes

import pytest
import torch

from lethe_b200 import native, ops

from .test_beam_cabi_cpu import Beam

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("where", ["scores", "penalty"])
@pytest.mark.parametrize("B,W,V", [(1, 4, 900), (70, 8, 5000), (300, 3, 33)])
def test_new_scores_in_the_place_of_old_ones(B, W, V, where):
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(B, W, V, generator=g, device="cuda").bfloat16()
    s = -torch.rand(B, W, generator=g, device="cuda") * 3
    pen = torch.rand(B, W, generator=g, device="cuda") + 0.5
    fin = torch.rand(B, W, generator=g, device="cuda") < 0.3
    want = ops.beam_select(x, s, finished=fin, eos=3, penalty=pen)
    parents, tokens = (torch.empty(B, W, dtype=torch.long, device="cuda") for _ in range(2))
    lib = native.lib()
    lib.lethe_gdn_beam_work_bytes.restype = ctypes.c_size_t
    lib.lethe_gdn_beam_work_bytes.argtypes = [ctypes.c_int64, ctypes.c_int32, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32]
    need = lib.lethe_gdn_beam_work_bytes(B, W, V, W, 1)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    best = dict(scores=s, penalty=pen)[where]
    a = Beam(B=B, V=V, W=W, k=W, x_type=1, temperature=1.0, logits=x.data_ptr(), logits_batch=W * V, logits_beam=V, scores=s.data_ptr(), finished=fin.data_ptr(),
             penalty=pen.data_ptr(), eos=3, out_scores=best.data_ptr(), parents=parents.data_ptr(), tokens=tokens.data_ptr(), out_finished=fin.data_ptr(),
             work=work.data_ptr(), work_bytes=need)
    call = lib.lethe_gdn_beam_select
    call.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    assert call(ctypes.addressof(a), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(best, want.scores) and torch.equal(fin, want.finished) and torch.equal(parents, want.parents) and torch.equal(tokens, want.tokens)
