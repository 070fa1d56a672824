"""The attention operators of the package as timeable passes: the per-head RMSNorm of q and k with the rotary embedding,
attention over padded or causal keys, and the training step of each.

``own`` picks what ``run`` does: the plain statement in elementary torch operations (fp32, rounded once), or the calls a
user makes of ``qk_norm_rope.fused_qk_norm_rope`` and ``attention_kernel.fused_attention``. Sizes are those of the
package's model (16 heads of 128, 4096 latent tokens, 512 text tokens, batch 8; 4 heads of 64 in its small configuration)
and generic ones around them.

A case: ``op`` "norm_rope" | "attend" | "layer" (both in a row, as an attention layer runs them); ``train``: gradients too;
``batch``, ``lq``, ``lk``, ``heads``, ``kv_heads``, ``dim``; ``rope``: with tables ("shared" by the samples, one per
"sample", or "none"); ``weights``: type of the norm weights
(the model's own is bf16: a layer has no other); ``packed``: q, k and v are slices of one projection's output;
``causal``; ``ragged``: the samples have keys of different lengths; ``empty``: the last sample has none.
"""
from __future__ import annotations

import math

import torch

own = False

BF16 = torch.bfloat16
EPS = 1e-6


def _case(op, name=None, train=False, batch=1, lq=1, lk=None, heads=16, kv_heads=None, dim=128, rope="none", weights="bf16",
          packed=False, causal=False, ragged=False, empty=False):
    case = dict(op=op, train=train, batch=batch, lq=lq, lk=lq if lk is None else lk, heads=heads,
                kv_heads=heads if kv_heads is None else kv_heads, dim=dim, rope=rope, weights=weights, packed=packed,
                causal=causal, ragged=ragged, empty=empty)
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # q and k of one self-attention layer in a training step of the model: latents of 128 x 128, batch 8
        _case("norm_rope", "norm_rope_step", train=True, batch=8, lq=4096, rope="shared"),
        # one new token a sample with shared key heads, each at its own position: latency
        _case("norm_rope", "norm_rope_one_token", batch=4, lq=1, kv_heads=4, rope="sample"),
        # slices of one packed projection, narrow heads, an odd number of tokens, fp32 norm weights that are trained
        _case("norm_rope", "norm_rope_packed", train=True, batch=3, lq=1021, heads=12, kv_heads=4, dim=64, rope="shared",
              weights="fp32", packed=True),
        # sampling, self-attention: the conditioned and the unconditioned image together
        _case("attend", "attend_sample_self", batch=2, lq=4096),
        # sampling, cross-attention onto a padded text of up to 512 tokens
        _case("attend", "attend_sample_text", batch=2, lq=4096, lk=512, ragged=True),
        # one query token against a long sequence of keys shared by groups of heads
        _case("attend", "attend_one_query", batch=8, lq=1, lk=16384, kv_heads=4, ragged=True),
        # the smallest call: one small image of the small configuration
        _case("attend", "attend_small", batch=1, lq=64, heads=4, dim=64),
        # a long sequence (a video, a large image), forward only
        _case("attend", "attend_long", batch=1, lq=16384),
        # training step of the model, self-attention: the largest
        _case("attend", "attend_train_self", train=True, batch=8, lq=4096),
        # training step of the model, cross-attention onto padded texts
        _case("attend", "attend_train_text", train=True, batch=8, lq=4096, lk=512, ragged=True),
        # causal, odd length, shared key heads, narrow heads, padded, one sample without any key
        _case("attend", "attend_train_causal", train=True, batch=4, lq=2047, heads=16, kv_heads=4, dim=64, causal=True,
              ragged=True, empty=True),
        # norm, rotation and attention in a row, forward and backward, as one attention layer trains them: one small image
        _case("layer", "layer_train", train=True, batch=2, lq=1024, rope="shared"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm_rope", "attend", "attend", "attend", "layer"))
    train = rng.random() < 0.6
    batch = rng.randint(1, 8)
    kv_heads = rng.choice((1, 2, 4, 8, 16))
    heads = min(16, kv_heads * rng.choice((1, 1, 2, 4)))
    dim = rng.choice((64, 128, 128))
    weights = rng.choice(("bf16", "fp32"))
    if op == "norm_rope":
        lq = _log(rng, 1, 4096)
        rope = rng.choice(("none", "shared", "sample"))
        return _case(op, None, train, batch, lq, None if rope != "none" else _log(rng, 1, 4096), heads, kv_heads, dim, rope,
                     weights, packed=rope != "none" and rng.random() < 0.3)
    if op == "layer":
        return _case(op, None, train, min(batch, 4), _log(rng, 16, 4096), None, heads, kv_heads, dim,
                     rng.choice(("shared", "sample")), "bf16", causal=rng.random() < 0.3)
    lq = _log(rng, 1, 4096)
    lk = lq if rng.random() < 0.5 else _log(rng, 1, 4096)
    if not train and rng.random() < 0.3:            # few queries, many keys
        lq, lk = rng.randint(1, 16), _log(rng, 1024, 16384)
    ragged = rng.random() < 0.4
    return _case(op, None, train, batch, lq, lk, heads, kv_heads, dim, "none", weights, packed=lq == lk and rng.random() < 0.3,
                 causal=rng.random() < 0.3, ragged=ragged, empty=ragged and batch > 1 and rng.random() < 0.3)


def _lengths(case):
    """Keys of each sample: all, or from all down to an eighth of them, odd numbers among them."""
    B, L = case["batch"], case["lk"]
    if not case["ragged"]:
        return [L] * B
    found = [max(1, L - (7 * L * b) // (8 * B) - (b % 2 if L > 8 else 0)) for b in range(B)]
    if case["empty"]:
        found[-1] = 0
    return found


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, Lq, Lk, H, Hk, D = (case[n] for n in ("batch", "lq", "lk", "heads", "kv_heads", "dim"))

    def rand(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(BF16)

    s = {"case": case}
    if case["packed"]:
        both = rand(B, Lq, H + 2 * Hk, D)
        s["q"], s["k"], s["v"] = both[:, :, :H], both[:, :, H:H + Hk], both[:, :, H + Hk:]
    else:
        s["q"], s["k"], s["v"] = rand(B, Lq, H, D), rand(B, Lk, Hk, D), rand(B, Lk, Hk, D)
    if case["op"] != "norm_rope":
        s["grad"] = rand(B, Lq, H, D, std=0.1)
    else:
        s["grad_q"], s["grad_k"] = rand(B, Lq, H, D, std=0.1), rand(B, Lk, Hk, D, std=0.1)
    if case["op"] != "attend":
        dtype = BF16 if case["weights"] == "bf16" else torch.float32
        s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2))
        s["cos"] = s["sin"] = None
        if case["rope"] != "none":
            pos = torch.arange(Lq, device="cuda", dtype=torch.float64)
            if case["rope"] == "sample":
                pos = pos + torch.randint(0, 4096, (B, 1), generator=g, device="cuda").double()
            inv = 10000.0 ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2))
            ang = pos[..., None] * inv
            ang = torch.cat((ang, ang), dim=-1)
            s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
    leaves = [n for n in ("q", "k", "v", "wq", "wk") if n in s] if case["train"] else []
    for n in leaves:
        s[n] = s[n].detach().requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------- plain forms
def _per_sample(table):
    return table[None, :, None, :] if table.dim() == 2 else table[:, :, None, :]


def _half_turn(x):
    a, b = x.chunk(2, dim=-1)
    return torch.cat((-b, a), dim=-1)


def _norm_rope(x, w, cos, sin):
    """(result, x / rms, 1 / rms) in fp32."""
    x = x.detach().float()
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = x * r * w.detach().float()
    if cos is not None:
        n = n * _per_sample(cos) + _half_turn(n) * _per_sample(sin)
    return n, x * r, r


def _norm_rope_back(g, xhat, r, w, cos, sin):
    """Gradients of x and of the weight, fp32."""
    g = g.float()
    if cos is not None:
        g = g * _per_sample(cos) - _half_turn(g * _per_sample(sin))
    gw = g * w.detach().float()
    return r * (gw - xhat * (gw * xhat).mean(-1, keepdim=True)), (g * xhat).sum((0, 1, 2))


def _visible(case, device):
    """[batch or 1, lq, lk]: key j is seen by query i; None: every key by every query."""
    Lq, Lk = case["lq"], case["lk"]
    seen = None
    j = torch.arange(Lk, device=device)
    if case["ragged"]:
        seen = (j < torch.tensor(_lengths(case), device=device)[:, None])[:, None, :]
    if case["causal"]:
        low = (j <= torch.arange(Lq, device=device)[:, None] + (Lk - Lq))[None]
        seen = low if seen is None else seen & low
    return seen


def _heads_first(x, kv_heads):
    """(B, L, H, D) -> fp32 (B, kv_heads, H / kv_heads, L, D)."""
    B, L, H, D = x.shape
    return x.detach().float().reshape(B, L, kv_heads, H // kv_heads, D).permute(0, 2, 3, 1, 4)


def _heads_last(x):
    B, Hk, G, L, D = x.shape
    return x.permute(0, 3, 1, 2, 4).reshape(B, L, Hk * G, D)


def _probabilities(q, k, scale, seen):
    p = q @ k.transpose(-1, -2)
    p *= scale
    if seen is not None:
        p.masked_fill_(~seen[:, None, None], -math.inf)
    m = p.amax(-1, keepdim=True)
    p -= torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = p.exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total == 0, torch.ones_like(total), total)
    return p


def _attend(case, q, k, v, grad=None):
    """The output and, with `grad`, the gradients of q, k and v; all fp32."""
    Hk, scale = case["kv_heads"], case["dim"] ** -0.5
    q, k, v = _heads_first(q, Hk), _heads_first(k, Hk), _heads_first(v, Hk)
    p = _probabilities(q, k, scale, _visible(case, q.device))
    out = p @ v
    if grad is None:
        return (_heads_last(out),)
    g = _heads_first(grad, Hk)
    dv = (p.transpose(-1, -2) @ g).sum(2, keepdim=True)
    ds = g @ v.transpose(-1, -2)
    ds -= (g * out).sum(-1, keepdim=True)
    ds *= p
    ds *= scale
    dq = ds @ k
    dk = (ds.transpose(-1, -2) @ q).sum(2, keepdim=True)
    return _heads_last(out), _heads_last(dq), _heads_last(dk), _heads_last(dv)


def _plain(s):
    case = s["case"]
    if case["op"] == "norm_rope":
        (q, qh, rq), (k, kh, rk) = (_norm_rope(s[n], s["w" + n], s["cos"], s["sin"]) for n in "qk")
        if not case["train"]:
            return {"q": q.to(BF16), "k": k.to(BF16)}
        dq, dwq = _norm_rope_back(s["grad_q"], qh, rq, s["wq"], s["cos"], s["sin"])
        dk, dwk = _norm_rope_back(s["grad_k"], kh, rk, s["wk"], s["cos"], s["sin"])
        return {"q": q.to(BF16), "k": k.to(BF16), "dq": dq.to(BF16), "dk": dk.to(BF16), "dwq": dwq.to(s["wq"].dtype),
                "dwk": dwk.to(s["wk"].dtype)}
    if case["op"] == "attend":
        found = _attend(case, s["q"], s["k"], s["v"], s["grad"] if case["train"] else None)
        return dict(zip(("out", "dq", "dk", "dv"), (t.to(BF16) for t in found)))
    (q, qh, rq), (k, kh, rk) = (_norm_rope(s[n], s["w" + n], s["cos"], s["sin"]) for n in "qk")
    if not case["train"]:
        return {"out": _attend(case, q, k, s["v"])[0].to(BF16)}
    out, gq, gk, dv = _attend(case, q, k, s["v"], s["grad"])
    dq, dwq = _norm_rope_back(gq, qh, rq, s["wq"], s["cos"], s["sin"])
    dk, dwk = _norm_rope_back(gk, kh, rk, s["wk"], s["cos"], s["sin"])
    return {"out": out.to(BF16), "dq": dq.to(BF16), "dk": dk.to(BF16), "dv": dv.to(BF16), "dwq": dwq.to(s["wq"].dtype),
            "dwk": dwk.to(s["wk"].dtype)}


# ---------------------------------------------------------------------------------------- the package's calls
def _own(s):
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    from anima_trainer_sm120_b200.qk_norm_rope import fused_qk_norm_rope

    case, train = s["case"], s["case"]["train"]
    q, k, v = s["q"], s["k"], s["v"]
    if case["op"] != "attend":
        q, k = fused_qk_norm_rope(q, k, s["wq"], s["wk"], s["cos"], s["sin"], EPS)
        if case["op"] == "norm_rope":
            if not train:
                return {"q": q, "k": k}
            grads = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["grad_q"], s["grad_k"]))
            return dict(zip(("q", "k", "dq", "dk", "dwq", "dwk"), (q.detach(), k.detach(), *grads)))
    out = fused_attention(q, k, v, kv_lengths=s["lengths"], causal=case["causal"])
    if not train:
        return {"out": out}
    names = ("q", "k", "v") if case["op"] == "attend" else ("q", "k", "v", "wq", "wk")
    grads = torch.autograd.grad(out, [s[n] for n in names], s["grad"])
    return dict(zip(["out"] + ["d" + n for n in names], (out.detach(), *grads)))


def run(s):
    if own:
        return _own(s)
    return _plain(s)


# ---------------------------------------------------------------------------------------- what a pass cannot do without
def _pairs(case):
    """(query, key) pairs that see each other, over samples and heads."""
    Lq, Lk, total = case["lq"], case["lk"], 0
    for n in _lengths(case):
        if not case["causal"]:
            total += Lq * n
            continue
        # query i sees min(n, max(0, i + Lk - Lq + 1)) keys
        first, last = max(0, Lk - Lq + 1), Lk                   # keys seen by the first and the last query, before the length
        rising = min(n, last) - first + 1                      # queries with first .. min(n, last) keys
        if rising > 0:
            total += (first + min(n, last)) * rising // 2
        total += (last - max(n, first - 1)) * n if n < last else 0
    return total * case["heads"]


def work(case):
    B, Lq, Lk, H, Hk, D = (case[n] for n in ("batch", "lq", "lk", "heads", "kv_heads", "dim"))
    q, k = 2 * B * Lq * H * D, 2 * B * Lk * Hk * D              # bytes of a tensor like q, like k
    table = 0 if case["rope"] == "none" else 8 * Lq * D * (B if case["rope"] == "sample" else 1)
    small = 2 * D * (2 if case["weights"] == "bf16" else 4)
    if case["op"] == "norm_rope":
        # forward: q and k in and out; backward: the gradients in, q and k once more, the gradients out
        flops = (q + k) // 2 * 8
        if not case["train"]:
            return {"bytes": 2 * (q + k) + table + small, "flops": flops}
        return {"bytes": 5 * (q + k) + table + 2 * small, "flops": 3 * flops}
    seen = 2 * sum(_lengths(case)) * Hk * D                     # bytes of the keys that count
    pairs = _pairs(case)
    if not case["train"]:
        bytes_, flops = 2 * q + 2 * seen, 4 * D * pairs
    else:
        # q, k, v and the gradient in; the output and three gradients out (all of them: zeros for keys nobody sees)
        bytes_, flops = 4 * q + 2 * seen + 2 * k, 14 * D * pairs
    if case["op"] == "layer":
        bytes_ += table + small * (2 if case["train"] else 1)
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_norm_rope(x, w, cos, sin):
    y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w
    if cos is None:
        return y
    half = x.shape[-1] // 2
    cos, sin = cos.double(), sin.double()
    if cos.dim() == 2:
        cos, sin = cos[None], sin[None]
    cos, sin = cos.unsqueeze(2), sin.unsqueeze(2)
    first = y[..., :half] * cos[..., :half] - y[..., half:] * sin[..., :half]
    second = y[..., half:] * cos[..., half:] + y[..., :half] * sin[..., half:]
    return torch.cat((first, second), dim=-1)


def _exact_attend(case, q, k, v, grad):
    """Sample by sample and key head by key head: softmax over the keys that are seen. fp64 (out, dq, dk, dv)."""
    B, Lq, Lk, H, Hk, D = (case[n] for n in ("batch", "lq", "lk", "heads", "kv_heads", "dim"))
    group, lengths = H // Hk, _lengths(case)
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        n = lengths[b]
        lo = max(0, Lq - Lk) if case["causal"] else 0           # the queries before it see nothing
        if n == 0 or lo >= Lq:
            continue
        hide = None
        if case["causal"]:
            hide = torch.ones(Lq, Lk, dtype=torch.bool, device=q.device).triu(Lk - Lq + 1)[lo:, :n]
        for h in range(H):
            a, c, e = q[b, lo:, h], k[b, :n, h // group], v[b, :n, h // group]
            s = a @ c.T / math.sqrt(D)
            if hide is not None:
                s = s.masked_fill(hide, float("-inf"))
            p = torch.softmax(s, dim=-1)
            o = p @ e
            out[b, lo:, h] = o
            if grad is None:
                continue
            g = grad[b, lo:, h]
            dv[b, :n, h // group] += p.T @ g
            t = p * (g @ e.T - (o * g).sum(-1, keepdim=True)) / math.sqrt(D)
            dq[b, lo:, h] = t @ c
            dk[b, :n, h // group] += t.T @ a
    return out, dq, dk, dv


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        wide = {n: s[n].detach().double() for n in ("q", "k", "v", "wq", "wk", "grad", "grad_q", "grad_k") if n in s}
    if case["op"] == "attend":
        found = _exact_attend(case, wide["q"], wide["k"], wide["v"], wide["grad"] if case["train"] else None)
        return dict(zip(("out", "dq", "dk", "dv"), found if case["train"] else found[:1]))
    leaves = [wide[n].requires_grad_(True) for n in ("q", "k", "wq", "wk")]
    q = _exact_norm_rope(leaves[0], leaves[2], s["cos"], s["sin"])
    k = _exact_norm_rope(leaves[1], leaves[3], s["cos"], s["sin"])
    if case["op"] == "norm_rope":
        if not case["train"]:
            return {"q": q.detach(), "k": k.detach()}
        grads = torch.autograd.grad((q, k), leaves, (wide["grad_q"], wide["grad_k"]))
        return dict(zip(("q", "k", "dq", "dk", "dwq", "dwk"), (q.detach(), k.detach(), *grads)))
    out, gq, gk, dv = _exact_attend(case, q.detach(), k.detach(), wide["v"], wide["grad"] if case["train"] else None)
    if not case["train"]:
        return {"out": out}
    dq, dk, dwq, dwk = torch.autograd.grad((q, k), leaves, (gq, gk))
    return {"out": out, "dq": dq, "dk": dk, "dv": dv, "dwq": dwq, "dwk": dwk}
