"""The gated feed-forward half of a layer on 8-bit activations, next to attention.SparseAttention: pre-norm, gated
projections and the output projection with the residual, three launches (a8.py)."""
from __future__ import annotations

import torch

from .a8 import ACTS, A8, gated_a8, linear_a8, norm_quant8
from .w8 import W8


class GatedFeedForward:
    """y = h + down(act(gate(q)) * up(q)), q = rmsnorm(h) * norm_w, h = x + residual (or x).

    Weights: norm_w [dim] (rounded to bf16 where it is not), gate and up W8 [F, dim], down W8 [dim, F]; F % 32 == 0.
    limit as gated_a8's.  Between the launches the activations are A8: q once per value, the gated product once."""

    def __init__(self, norm_w: torch.Tensor, gate: W8, up: W8, down: W8, *, eps: float = 1e-6, act: str = "silu",
                 limit: float = 0.0):
        F, dim = gate.shape
        if up.shape != (F, dim) or down.shape != (dim, F) or tuple(norm_w.shape) != (dim,) or F % 32:
            raise ValueError(f"GatedFeedForward: gate {gate.shape}, up {up.shape}, down {down.shape}, "
                             f"norm {tuple(norm_w.shape)}")
        if act not in ACTS:
            raise ValueError(f"GatedFeedForward: act {act!r} (one of {', '.join(ACTS)})")
        self.norm_w = norm_w if norm_w.dtype == torch.bfloat16 else norm_w.to(torch.bfloat16)
        self.gate, self.up, self.down = gate, up, down
        self.eps, self.act, self.limit = eps, act, limit

    def __call__(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        """x [..., dim] bf16 (e.g. the attention's output) and the stream it is added to -> the next stream [..., dim]."""
        if residual is None:
            q, h = norm_quant8(x, self.norm_w, self.eps), x
        else:
            q, h = norm_quant8(x, self.norm_w, self.eps, residual=residual)
        a = gated_a8(q, self.gate, self.up, act=self.act, limit=self.limit, out=A8)
        return linear_a8(a, self.down, residual=h)
