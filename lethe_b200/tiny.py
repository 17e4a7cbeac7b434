"""A small language-model block around the op, for the training-loop evidence the reference keeps
(``results/gdn2_tiny_train_*.json`` of the reference project: B=4, L=256, H=2, d_k=128, d_v=64, 300 Adam
steps at lr 0.01 on a delayed-copy task, loss 3.67 -> below 1e-3, no NaN; arms for the scalar-gate
delta rule, KDA, GLA and SSD).

The block follows the layout of a gated-delta-rule layer: token embedding, a two-tap causal mixing of
neighbouring tokens (the short convolution such layers put in front of q, k, v), linear maps to q, k, v,
the log decay and the erase / write gate, the six-input op, and an output head.  The op is passed in,
so the same module trains through the CUDA library (``lethe_b200.ops.gdn2_op``) or through any callable
with the reference's signature ``op(q, k, v, g, b, w) -> o``.

``TinyDiagLM`` is the same for the element-wise gated recurrence: blocks of norm, recurrence, gated norm and residual sum, with a
prompt and single tokens for generation.
"""

from __future__ import annotations

import torch
import torch.nn as nn
from torch import Tensor

ARMS = ("gdn", "kda", "gla", "ssd")


def delayed_copy_batch(B: int, L: int, vocab: int, delay: int = 1, seed: int = 0) -> tuple[Tensor, Tensor]:
    """Tokens ``x [B, L]`` drawn uniformly and targets ``y[t] = x[t - delay]`` (``y[t] = 0`` for t < delay)."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randint(1, vocab, (B, L), generator=gen)
    y = torch.zeros_like(x)
    y[:, delay:] = x[:, :-delay]
    return x, y


class TinyGdnLM(nn.Module):
    """``arm``: "gdn" scalar gate + beta (b = w = beta broadcast), "kda" channel-wise gate + beta,
    "gla" channel-wise gate without the delta term (b = 0, w = 1), "ssd" scalar gate without it."""

    def __init__(self, op, arm: str = "gdn", vocab: int = 40, d_model: int = 64, H: int = 2, K: int = 128, V: int = 64):
        super().__init__()
        if arm not in ARMS:
            raise ValueError(f"arm must be one of {ARMS}")
        self.op, self.arm, self.vocab, self.H, self.K, self.V = op, arm, vocab, H, K, V
        self.emb = nn.Embedding(vocab, d_model)
        self.mix = nn.Linear(2 * d_model, d_model)
        self.q = nn.Linear(d_model, H * K, bias=False)
        self.k = nn.Linear(d_model, H * K, bias=False)
        self.v = nn.Linear(d_model, H * V, bias=False)
        self.g = nn.Linear(d_model, H * (K if arm in ("kda", "gla") else 1))
        self.beta = nn.Linear(d_model, H)
        self.head = nn.Linear(H * V, vocab)

    def forward(self, x: Tensor) -> Tensor:
        B, L = x.shape
        H, K, V = self.H, self.K, self.V
        e = self.emb(x)
        prev = torch.cat([torch.zeros_like(e[:, :1]), e[:, :-1]], dim=1)
        h = torch.tanh(self.mix(torch.cat([e, prev], dim=-1)))
        q = self.q(h).view(B, L, H, K)
        k = self.k(h).view(B, L, H, K)
        v = self.v(h).view(B, L, H, V)
        g = -torch.nn.functional.softplus(self.g(h)).view(B, L, H, -1).expand(B, L, H, K).contiguous()
        if self.arm in ("gdn", "kda"):
            beta = torch.sigmoid(self.beta(h)).view(B, L, H, 1)
            b, w = beta.expand(B, L, H, K).contiguous(), beta.expand(B, L, H, V).contiguous()
        else:
            b, w = torch.zeros(B, L, H, K, device=x.device), torch.ones(B, L, H, V, device=x.device)
        o = self.op(q, k, v, g, b, w)
        return self.head(o.reshape(B, L, H * V).to(h.dtype))


class DiagBlock(nn.Module):
    """``x``: output of the block before, ``stream``: the residual stream in fp32.  y, stream = residual_norm(x, stream); value, log
    decay and gate from y; the element-wise recurrence; gated norm per head; output map."""

    def __init__(self, ops, d_model: int, H: int, V: int, depth: int):
        super().__init__()
        self.ops, self.H, self.V = ops, H, V
        self.norm, self.out_norm = nn.Parameter(torch.ones(d_model)), nn.Parameter(torch.ones(V))
        self.scale = nn.Parameter(torch.full((d_model,), 1.0 if depth == 0 else 0.5))
        self.proj = nn.Linear(d_model, 3 * H * V, bias=False)      # value, decay, gate: read where they lie in its output
        self.out = nn.Linear(H * V, d_model, bias=False)

    def forward(self, x: Tensor, stream: Tensor | None, state: Tensor | None = None) -> tuple[Tensor, Tensor, Tensor]:
        """``[B, L, d_model]``, or ``[B, d_model]`` for one token with ``state [B, H, V]``, which is updated in place."""
        y, stream = self.ops.residual_norm(x, stream, self.norm, scale=self.scale)
        value, decay, gate = self.proj(y).unflatten(-1, (3, self.H, self.V)).unbind(-3)
        g = -torch.nn.functional.softplus(decay.float() - 2.0)
        if x.dim() == 2:
            h = self.ops.diag_scan_step(value, g, state, complement=True)
        else:
            h, state = self.ops.diag_scan(value, g, state, complement=True)
        o = self.ops.gated_norm(h, gate, self.out_norm)
        return self.out(o.flatten(-2)), stream, state


class TinyDiagLM(nn.Module):
    """``ops``: ``lethe_b200.ops`` or anything with its ``diag_scan``, ``diag_scan_step``, ``gated_norm`` and ``residual_norm`` (``beam_search``: ``beam_select`` and
    ``reorder_states`` too)."""

    def __init__(self, ops, vocab: int = 40, d_model: int = 64, H: int = 2, V: int = 64, layers: int = 2):
        super().__init__()
        self.ops = ops
        self.emb = nn.Embedding(vocab, d_model)
        self.blocks = nn.ModuleList(DiagBlock(ops, d_model, H, V, i) for i in range(layers))
        self.norm = nn.Parameter(torch.ones(d_model))
        self.head = nn.Linear(d_model, vocab)

    def forward(self, tokens: Tensor, states: list[Tensor | None] | None = None) -> tuple[Tensor, list[Tensor]]:
        """Logits and the blocks' states.  ``tokens [B, L]``, or ``[B]`` with the states of the tokens before (updated in place)."""
        states = [None] * len(self.blocks) if states is None else states
        x, stream, after = self.emb(tokens), None, []
        for block, state in zip(self.blocks, states):
            x, stream, state = block(x, stream, state)
            after.append(state)
        y, _ = self.ops.residual_norm(x, stream, self.norm)
        return self.head(y), after

    @torch.no_grad()
    def beam_search(self, prompt: Tensor, steps: int, beams: int, eos: int | None = None) -> tuple[Tensor, Tensor]:
        """The ``beams`` best continuations found for every ``prompt [B, L]``: tokens ``[B, beams, steps]`` and log probabilities
        ``[B, beams]``, best first.  Every beam has its own states, which follow the beams that are gone on from."""
        B = prompt.shape[0]
        logits, states = self(prompt)
        scores = torch.full((B, beams), float("-inf"), device=prompt.device)
        scores[:, 0] = 0.0                                          # (all beams are the same one)
        states = [s.repeat_interleave(beams, 0) for s in states]
        logits = logits[:, -1:].expand(B, beams, -1)
        written = torch.zeros(B * beams, steps, dtype=torch.long, device=prompt.device)
        finished = None
        for t in range(steps):
            if t:
                logits = self(written[:, t - 1], states)[0].view(B, beams, -1)
            scores, parents, tokens, finished = self.ops.beam_select(logits, scores, finished=finished, eos=eos)
            self.ops.reorder_states([*states, written], parents)
            written[:, t] = tokens.flatten()
        return written.view(B, beams, steps), scores
