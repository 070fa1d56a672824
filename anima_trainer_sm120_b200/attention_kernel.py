"""Softmax attention as a fused autograd op on the sm_100a kernels of ``csrc/attention_fwd.cu`` and ``csrc/attention_bwd.cu``.

anima-trainer leaves this step of the DiT to a library (``F.scaled_dot_product_attention``; its
``tests/bench_attention.py:3-7`` compares several). Tensors are (batch, tokens, heads, head_dim) as the projections
make them, so nothing is transposed or copied on the way in.
"""
from __future__ import annotations

import torch

from ._lib import host


class FusedAttention:
    """``softmax(scale * q k^T) v`` over the keys a query sees (native node: ``csrc/host/attention.cpp``)."""

    @staticmethod
    def apply(q, k, v, kv_lengths, causal, scale, return_lse):
        return host().attention(q, k, v, kv_lengths, causal, scale, return_lse)


def fused_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, kv_lengths: torch.Tensor | None = None,
                    causal: bool = False, scale: float | None = None, return_lse: bool = False):
    """Attention of ``q`` (B, Lq, H, D) to ``k`` / ``v`` (B, Lk, Hk, D); bfloat16, D 64 or 128, H a multiple of Hk, any strides
    (what the kernels cannot read in place is copied). Returns a dense (B, Lq, H, D) tensor.

    ``kv_lengths`` (int32 or int64 [B], on the GPU): sample b has keys 0 .. kv_lengths[b] - 1; keys and values behind them
    may hold anything, NaN included, and get gradient 0. ``causal``: query i sees keys j <= i + Lk - Lq. A query that sees no key
    has output 0. ``scale`` defaults to D ** -0.5 and must be positive. ``return_lse``: also the natural logarithm of each
    row's sum, fp32 [B, H, Lq], -inf for such a query; it carries no gradient.

    Sums and statistics are fp32; the probabilities (and, backward, their gradients) enter the second product as bf16.
    Forward and backward are deterministic. The backward pass holds, while it runs, the scores' gradients of the heads that it goes
    through at a time in bf16: 2 bytes a (query, key) pair, 1 GiB where there are more, up to 4 where fewer parts run faster."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    out, lse = FusedAttention.apply(q, k, v, kv_lengths, bool(causal), float(scale), bool(return_lse))
    return (out, lse) if return_lse else out
