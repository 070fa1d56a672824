"""Patch the attention step of the DiT with the fused kernels: ``Attention._attend`` runs :func:`attention_kernel.fused_attention`.

anima-trainer's patches leave ``F.scaled_dot_product_attention`` in place (``adaln_patch.py:100-130`` calls the unpatched
attention modules); this one has the ``install(cls)`` / ``uninstall(cls)`` form of the others and falls through to the
original method for what the kernels do not take (CPU tensors, other types, heads of another width).
"""
from __future__ import annotations

import torch

from .attention_kernel import fused_attention

_PATCHED: dict[type, object] = {}


def _patched_attend(self, q, k, v, attn_params=None):
    if not (q.is_cuda and q.dtype == k.dtype == v.dtype == torch.bfloat16 and q.shape[-1] in (64, 128)):
        return next(_PATCHED[c] for c in type(self).__mro__ if c in _PATCHED)(self, q, k, v, attn_params)
    return fused_attention(q, k, v, kv_lengths=self._key_lengths(attn_params))


def install(attn_cls: type | None = None) -> None:
    """Patch ``attn_cls._attend`` (default: the stand-in ``anima_dit.Attention``). Idempotent."""
    if attn_cls is None:
        from .anima_dit import Attention as attn_cls
    if attn_cls in _PATCHED:
        return
    _PATCHED[attn_cls] = attn_cls._attend
    attn_cls._attend = _patched_attend


def uninstall(attn_cls: type | None = None) -> None:
    if attn_cls is None:
        from .anima_dit import Attention as attn_cls
    orig = _PATCHED.pop(attn_cls, None)
    if orig is not None:
        attn_cls._attend = orig
