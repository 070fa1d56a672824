"""Oracle: attention, and the per-head RMSNorm with rotary embedding before it (torch, fp64, any device).

anima-trainer calls libraries for both (``F.scaled_dot_product_attention``; Liger's RMSNorm, ``liger_patch.py:31-47``;
Transformer Engine's RoPE, ``rope_patch.py:28-56``); these are the textbook definitions. Beside each value the functions give
the bound on a kernel's error that follows from the roundings it is allowed (``*_bounds``): bf16 results and bf16
probabilities (half a step: 2^-8), fp32 products, sums and statistics, and an exponential good to ``EXP_REL``.
"""
from __future__ import annotations

import math

import torch

BF16_HALF = 2.0 ** -8       # torch.finfo(torch.bfloat16).eps / 2
F32_HALF = 2.0 ** -24
EXP_REL = 2.0 ** -16        # relative error of one exponential


def visible(B, Lq, Lk, lengths=None, causal=False, device="cpu"):
    """bool [B, 1, Lq, Lk]: query i sees key j."""
    j, i = torch.arange(Lk, device=device), torch.arange(Lq, device=device)[:, None]
    seen = torch.ones(B, 1, Lq, Lk, dtype=torch.bool, device=device)
    if lengths is not None:
        seen &= (j < lengths.to(device).view(B, 1, 1, 1))
    if causal:
        seen &= (j <= i + Lk - Lq)
    return seen


def _wide(x, heads):
    """(B, L, Hk, D) -> fp64 (B, heads, L, D), a key head repeated for the queries' heads it serves."""
    return x.double().permute(0, 2, 1, 3).repeat_interleave(heads // x.shape[2], dim=1)


def _narrow(x, kv_heads):
    """(B, H, L, D) -> (B, L, kv_heads, D), summed over the heads of a group."""
    B, H, L, D = x.shape
    return x.view(B, kv_heads, H // kv_heads, L, D).sum(2).permute(0, 2, 1, 3)


def attention(q, k, v, *, lengths=None, causal=False, scale=None, dout=None):
    """Values and bounds: {"out", "lse"[, "dq", "dk", "dv"]} -> (fp64 value, fp64 bound), layouts as the package's."""
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    seen = visible(B, Lq, Lk, lengths, causal, q.device)
    hidden = ~seen[:, 0].any(1)                                       # [B, Lk]: keys nobody sees may hold anything
    k, v = (torch.where(hidden[:, :, None, None], torch.zeros_like(t), t) for t in (k, v))
    q, k, v = _wide(q, H), _wide(k, H), _wide(v, H)
    s = (q @ k.mT * scale).masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True) if Lk else s.new_full((B, H, Lq, 1), -math.inf)
    some = m > -math.inf
    e = torch.exp(s - torch.where(some, m, 0.0))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(some, total, 1.0)
    out = p @ v
    lse = (m + torch.log(total)).squeeze(-1)
    # relative error of one unnormalised probability: the score's absolute error (D products summed in fp32, its scaling, the
    # difference to the row's maximum, whose size is that of the scores) and the exponential's own
    size = q.abs() @ k.abs().mT * scale
    top = torch.where(seen, size, 0.0).amax(-1, keepdim=True) if Lk else torch.zeros_like(m)
    d_s = (2 * D + 16) * F32_HALF * top + EXP_REL
    d_sum = d_s + 2 * Lk * F32_HALF
    av = p @ v.abs()
    e_out = BF16_HALF * out.abs() + (BF16_HALF + d_s + d_sum + 2 * Lk * F32_HALF) * av * (1 + BF16_HALF)
    found = {"out": (out, e_out), "lse": (lse, (d_sum + 4 * F32_HALF * lse.abs().nan_to_num(posinf=0.0)[..., None]).squeeze(-1))}
    if dout is not None:
        g = _wide(dout, H)
        dp = g @ v.mT
        delta = (g * out).sum(-1, keepdim=True)
        ds = torch.where(seen, p * (dp - delta), 0.0)
        e_p = 2 * d_s + d_sum + 4 * F32_HALF * lse.abs().nan_to_num(posinf=0.0)[..., None]       # of the recomputed p, relative
        e_dp = (D + 4) * F32_HALF * (g.abs() @ v.abs().mT + (g * out).abs().sum(-1, keepdim=True)) \
            + (g.abs() * e_out).sum(-1, keepdim=True)
        e_ds = p * e_dp * (1 + e_p) + ds.abs() * (BF16_HALF + e_p)
        n = 2 * max(Lq, Lk) * (H // Hk) * F32_HALF
        e_dv = (BF16_HALF + n + e_p) * p
        found["dv"] = _pair(p.mT @ g, e_dv.mT @ g.abs(), Hk)
        found["dq"] = _pair(ds @ k * scale, (e_ds + n * ds.abs()) @ k.abs() * scale, None)
        found["dk"] = _pair(ds.mT @ q * scale, (e_ds + n * ds.abs()).mT @ q.abs() * scale, Hk)
    found["out"] = tuple(t.permute(0, 2, 1, 3) for t in found["out"])
    return found


def _pair(value, err, kv_heads):
    """(value, bound) in the package's layout; the result itself is rounded to bf16 once more."""
    value, err = (t.permute(0, 2, 1, 3) if kv_heads is None else _narrow(t, kv_heads) for t in (value, err))
    return value, err * (1 + BF16_HALF) + BF16_HALF * value.abs()


def norm_rope(x, w, cos=None, sin=None, eps=1e-6, dout=None):
    """Values and bounds {"out"[, "dx", "dw"]} of rope(rmsnorm(x) * w) over (B, L, H, D); dw in fp32 (no rounding to bf16)."""
    D = x.shape[-1]
    x, w = x.double(), w.double()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * r * w
    if cos is None:
        c, s = torch.ones_like(n), torch.zeros_like(n)
    else:
        c, s = (t.double().expand(x.shape[0], -1, -1)[:, :, None] if t.dim() == 3 else t.double()[None, :, None] for t in (cos, sin))
        c, s = c.expand_as(n), s.expand_as(n)

    def turn(t):
        a, b = t.chunk(2, -1)
        return torch.cat((-b, a), -1)

    few = (D + 24) * F32_HALF                    # the mean of D squares, its root, and a handful of products
    out = n * c + turn(n) * s
    found = {"out": (out, BF16_HALF * out.abs() + few * ((n * c).abs() + (turn(n) * s).abs()) * (1 + BF16_HALF))}
    if dout is not None:
        g = dout.double()
        dn = g * c - turn(g * s)
        adn = (g * c).abs() + turn(g * s).abs()
        gw, xh = dn * w, x * r
        mean = (gw * xh).mean(-1, keepdim=True)
        dx = r * (gw - xh * mean)
        size = r * (adn * w.abs() + xh.abs() * (adn * w.abs() * xh.abs()).mean(-1, keepdim=True))
        found["dx"] = (dx, BF16_HALF * dx.abs() + 2 * few * size * (1 + BF16_HALF))
        vectors = x[..., 0].numel()
        found["dw"] = ((dn * xh).sum((0, 1, 2)), (few + 2 * vectors * F32_HALF) * (adn * xh.abs()).sum((0, 1, 2)))
    return found
