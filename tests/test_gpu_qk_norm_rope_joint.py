"""GPU parity of the joint q / k RMSNorm + rotary embedding (forward, input and weight gradients) with its definition in 64
bits within the bounds ``oracle.attention.norm_rope`` derives, and of the patched attention layer and trainer that use it."""
from __future__ import annotations

import pytest
import torch

from oracle import attention as OA

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
DEV = "cuda"


def _rand(seed, *shape, std=1.0, dtype=BF16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * std).to(dtype)


def _tables(seed, *shape):
    ang = torch.rand(shape, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)) * 50     # halves not equal
    return ang.cos(), ang.sin()


def _within(name, got, pair, extra=0.0):
    want, bound = pair
    off = (got.double() - want).abs() - bound - extra
    assert got.shape == want.shape and bool((off <= 1e-30).all()), f"{name}: off by up to {float(off.max())} beyond its bound"


def _check(q, k, wq, wk, cos, sin, gq, gk, eps=1e-6):
    from anima_trainer_sm120_b200.qk_norm_rope import fused_qk_norm_rope
    leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    out = fused_qk_norm_rope(*leaves, cos, sin, eps)
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(out, fused_qk_norm_rope(q, k, wq, wk, cos, sin, eps)))
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        want = OA.norm_rope(x, w, cos, sin, eps, dout=g)
        _within("out", out[i].detach(), want["out"])
        _within("dx", grads[i], want["dx"])
        assert grads[2 + i].dtype == w.dtype and grads[2 + i].shape == w.shape
        _within("dw", grads[2 + i], want["dw"], extra=OA.BF16_HALF * want["dw"][0].abs() if w.dtype == BF16 else 0.0)


@pytest.mark.parametrize("B,L,H,Hk,D", [(1, 1, 1, 1, 64), (4, 1, 16, 4, 128), (2, 37, 3, 3, 128), (3, 33, 6, 2, 64),
                                        (2, 300, 16, 16, 128), (1, 1021, 12, 4, 64), (5, 7, 5, 1, 128)])
@pytest.mark.parametrize("rope", ["none", "shared", "sample"])
@pytest.mark.parametrize("wdtype", [BF16, torch.float32])
def test_forward_and_gradients(B, L, H, Hk, D, rope, wdtype):
    q, k, gq, gk = _rand(1, B, L, H, D, std=1.7), _rand(2, B, L, Hk, D), _rand(3, B, L, H, D), _rand(4, B, L, Hk, D)
    wq, wk = (1 + 0.2 * _rand(s, D, dtype=torch.float32) for s in (5, 6))
    cos, sin = (None, None) if rope == "none" else _tables(7, *((B, L, D) if rope == "sample" else (L, D)))
    _check(q, k, wq.to(wdtype), wk.to(wdtype), cos, sin, gq, gk)


def test_queries_and_keys_of_different_lengths_without_tables():
    for Lq, Lk in [(100, 7), (1, 513), (64, 0), (0, 64)]:
        _check(_rand(1, 2, Lq, 4, 128), _rand(2, 2, Lk, 2, 128), _rand(3, 128), _rand(4, 128), None, None,
               _rand(5, 2, Lq, 4, 128), _rand(6, 2, Lk, 2, 128))


def test_zero_vectors_zero_weights_and_large_values():
    q, k, gq, gk = (_rand(s, 2, 20, 4, 64) for s in range(4))
    q[:, 3] = 0
    k[:, :, 1] *= 1000
    w = _rand(5, 64, dtype=torch.float32)
    w[::3] = 0
    _check(q, k, w, w.clone(), *_tables(1, 20, 64), gq, gk)


def test_slices_of_a_packed_projection_and_other_strides_give_the_same_bits():
    from anima_trainer_sm120_b200.qk_norm_rope import fused_qk_norm_rope
    B, L, H, Hk, D = 2, 50, 6, 2, 128
    packed = _rand(1, B, L, H + 2 * Hk, D)
    wq, wk = _rand(2, D), _rand(3, D)
    cos, sin = _tables(4, L, D)
    forms = [(packed[:, :, :H], packed[:, :, H:H + Hk]),
             tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (packed[:, :, :H], packed[:, :, H:H + Hk])),
             (packed[:, :, :H].contiguous(), packed[:, :, H:H + Hk].contiguous())]
    odd = torch.empty(B, L, H, D + 1, device=DEV, dtype=BF16)[..., :D].copy_(packed[:, :, :H])       # copied inside
    forms.append((odd, forms[2][1]))
    grads = _rand(5, B, L, H, D), _rand(6, B, L, Hk, D)
    seen = []
    for q, k in forms:
        leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
        out = fused_qk_norm_rope(*leaves, cos, sin)
        seen.append([*(t.detach() for t in out), *torch.autograd.grad(out, leaves, grads)])
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))


def test_gradient_subsets_and_missing_output_gradients():
    from anima_trainer_sm120_b200.qk_norm_rope import fused_qk_norm_rope
    ts = [_rand(1, 1, 30, 4, 64), _rand(2, 1, 30, 4, 64), _rand(3, 64), _rand(4, 64)]
    cos, sin = _tables(5, 30, 64)
    gq, gk = _rand(6, 1, 30, 4, 64), _rand(7, 1, 30, 4, 64)

    def go(subset):
        leaves = [t.clone().requires_grad_(i in subset) for i, t in enumerate(ts)]
        torch.autograd.backward([o for o in fused_qk_norm_rope(*leaves, cos, sin)], [gq, gk])
        return [t.grad for t in leaves]

    full = go({0, 1, 2, 3})
    for subset in ({0}, {1}, {2}, {3}, {0, 1}, {2, 3}, {0, 3}):
        for i, (a, b) in enumerate(zip(go(subset), full)):
            assert (a is None) == (i not in subset)
            # dx alone runs with more threads a block: the same arithmetic per vector
            assert a is None or torch.equal(a, b)
    leaves = [t.clone().requires_grad_(True) for t in ts]
    q, _ = fused_qk_norm_rope(*leaves, cos, sin)
    q.backward(gq)
    assert torch.equal(leaves[0].grad, full[0]) and not leaves[1].grad.any() and not leaves[3].grad.any()


def test_gradient_against_differences():
    from anima_trainer_sm120_b200.qk_norm_rope import fused_qk_norm_rope
    ts = [_rand(1, 1, 9, 2, 64), _rand(2, 1, 9, 2, 64), _rand(3, 64, dtype=torch.float32), _rand(4, 64, dtype=torch.float32)]
    cos, sin = _tables(5, 9, 64)
    gq, gk = _rand(6, 1, 9, 2, 64), _rand(7, 1, 9, 2, 64)
    leaves = [t.clone().requires_grad_(True) for t in ts]
    grads = torch.autograd.grad(fused_qk_norm_rope(*leaves, cos, sin), leaves, (gq, gk))

    def loss(q, k, wq, wk):
        return sum((OA.norm_rope(x, w, cos, sin)["out"][0] * g.double()).sum() for x, w, g in ((q, wq, gq), (k, wk, gk)))

    for i, (x, w, g) in enumerate(((ts[0], ts[2], gq), (ts[1], ts[3], gk)) * 2):
        d = _rand(20 + i, *ts[i].shape, dtype=torch.float64)
        ends = [loss(*(t.double() + (s * 1e-4 * d if j == i else 0) for j, t in enumerate(ts))) for s in (1, -1)]
        value, bound = OA.norm_rope(x, w, cos, sin, dout=g)["dx" if i < 2 else "dw"]
        slack = (bound * d.abs()).sum() + 1e-5 * (value * d).abs().sum()
        assert float(((grads[i].double() * d).sum() - (ends[0] - ends[1]) / 2e-4).abs()) <= float(slack)


def test_refusals():
    from anima_trainer_sm120_b200.qk_norm_rope import fused_qk_norm_rope
    q, k, w = _rand(1, 2, 8, 4, 64), _rand(2, 2, 8, 2, 64), _rand(3, 64)
    cos, sin = _tables(4, 8, 64)
    with pytest.raises(TypeError):
        fused_qk_norm_rope(q.float(), k, w, w)
    with pytest.raises(ValueError):
        fused_qk_norm_rope(q, k, w[:32], w)
    with pytest.raises(ValueError):
        fused_qk_norm_rope(q, k[:1], w, w)
    with pytest.raises(ValueError):
        fused_qk_norm_rope(q, k, w, w, cos)
    with pytest.raises(ValueError):
        fused_qk_norm_rope(q, k[:, :4], w, w, cos, sin)
    with pytest.raises(ValueError):
        fused_qk_norm_rope(q, k, w, w, cos[:4], sin[:4])
    with pytest.raises(ValueError):
        fused_qk_norm_rope(q, k, w, w, cos.expand(3, 8, 64), sin.expand(3, 8, 64))
    with pytest.raises(NotImplementedError):
        fused_qk_norm_rope(q[..., :32], k[..., :32], w[:32], w[:32])
    with pytest.raises(NotImplementedError):
        fused_qk_norm_rope(q, k, w, w, cos.clone().requires_grad_(True), sin)
    with pytest.raises(RuntimeError):
        fused_qk_norm_rope(q.cpu(), k.cpu(), w.cpu(), w.cpu())
    x = q.clone().requires_grad_(True)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(fused_qk_norm_rope(x, k, w, w)[0].sum(), x, create_graph=True)
    wt = w.clone().requires_grad_(True)
    out = fused_qk_norm_rope(q, k, wt, w)
    with torch.no_grad():
        wt.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out[0].sum().backward()


def test_many_vectors_keep_their_weight_gradient_exact_and_the_same():
    """Thousands of partial sums, and the same bits each time."""
    from anima_trainer_sm120_b200.qk_norm_rope import fused_qk_norm_rope
    B, L, H, D = 2, 2500, 8, 128
    leaves = [_rand(s, B, L, H, D).requires_grad_(True) for s in (1, 2)] + [
        _rand(s, D, dtype=torch.float32).requires_grad_(True) for s in (3, 4)]
    cos, sin = _tables(5, L, D)
    g = _rand(6, B, L, H, D), _rand(7, B, L, H, D)
    runs = [torch.autograd.grad(fused_qk_norm_rope(*leaves, cos, sin), leaves, g) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    _within("dw", runs[0][2], OA.norm_rope(leaves[0].detach(), leaves[2].detach(), cos, sin, dout=g[0])["dw"])


def test_thin_wrappers_give_the_nodes_bits():
    from anima_trainer_sm120_b200 import ops
    from anima_trainer_sm120_b200.qk_norm_rope import fused_qk_norm_rope
    q, k, gq, gk = _rand(1, 2, 30, 6, 64), _rand(2, 2, 30, 2, 64), _rand(3, 2, 30, 6, 64), _rand(4, 2, 30, 2, 64)
    wq, wk = _rand(5, 64), _rand(6, 64)
    cos, sin = _tables(7, 2, 30, 64)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, wq, wk)]
    want = fused_qk_norm_rope(*leaves, cos, sin)
    grads = torch.autograd.grad(want, leaves, (gq, gk))
    assert all(torch.equal(a, b) for a, b in zip(ops.qk_norm_rope_fwd(q, k, wq, wk, cos, sin, 1e-6), want))
    assert all(torch.equal(a, b) for a, b in zip(ops.qk_norm_rope_bwd(gq, gk, q, k, wq, wk, cos, sin, 1e-6), grads))
    some = ops.qk_norm_rope_bwd(gq, gk, q, k, wq, wk, cos, sin, 1e-6, weights=False)
    assert torch.equal(some[0], grads[0]) and torch.equal(some[1], grads[1]) and some[2] is None
    with pytest.raises(TypeError):
        ops.qk_norm_rope_fwd(q, k, wq, wk.float(), None, None, 1e-6)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_fwd(q, k, wq, wk, cos[:, :5], sin[:, :5], 1e-6)


# ---------------------------------------------------------------------------------------- the layer, the model, the trainer
@pytest.mark.parametrize("heads", [2, 4])          # head widths 128 and 64
@pytest.mark.parametrize("cross", [False, True])
def test_patched_attention_layer_matches_the_eager_one(heads, cross):
    """Forward, input gradient and norm weight gradients: within 3 % of the largest value, as the eager layer rounds to bf16
    after every step (norm, product with the weight, rotation: five half steps of 2^-8 each on q and on k, and the same
    again backward)."""
    from anima_trainer_sm120_b200 import attention_patch, qk_norm_rope
    from anima_trainer_sm120_b200.anima_dit import Attention, AttentionParams, tiny_config
    cfg = tiny_config(heads=heads)
    torch.manual_seed(1)
    attn = Attention(cfg, cfg.context_dim if cross else None).to(DEV, BF16)
    x, gy = _rand(1, 2, 96, cfg.dim), _rand(2, 2, 96, cfg.dim)
    ctx = _rand(3, 2, 24, cfg.context_dim) if cross else None
    params = AttentionParams(torch.tensor([24, 7], device=DEV, dtype=torch.int32)) if cross else None
    rope = torch.rand(96, 1, 1, cfg.head_dim, device=DEV, generator=torch.Generator(DEV).manual_seed(4)) * 30
    results = []
    for fused in (False, True):
        if fused:
            qk_norm_rope.install(Attention, joint=True)
            attention_patch.install(Attention)
        try:
            xi = x.clone().requires_grad_(True)
            attn.zero_grad()
            y = attn(xi, params, ctx, rope_emb=rope)
            if fused:
                assert y.grad_fn is not None
            y.backward(gy)
            results.append([y.detach(), xi.grad, attn.q_norm.weight.grad.clone(), attn.k_norm.weight.grad.clone()])
        finally:
            qk_norm_rope.uninstall(Attention)
            attention_patch.uninstall(Attention)
    for a, b in zip(*results):
        assert float((a.float() - b.float()).abs().max() / a.float().abs().max()) < 3e-2


def test_layer_in_a_row_matches_the_definition():
    """Norm, rotation and attention as a layer runs them, against the 64-bit composition. q and k are rounded to bf16 between
    the two: each score is off by up to 2 * 2^-8 of scale * sum |q||k| (both factors), which bounds the change of every
    probability and, backward, of every gradient; taken at the largest score of the tensors."""
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    from anima_trainer_sm120_b200.qk_norm_rope import fused_qk_norm_rope
    B, L, H, Hk, D = 1, 150, 4, 2, 64
    q, k, v, g = _rand(1, B, L, H, D), _rand(2, B, L, Hk, D), _rand(3, B, L, Hk, D), _rand(4, B, L, H, D)
    wq, wk = (1 + 0.1 * _rand(s, D, dtype=torch.float32) for s in (5, 6))
    cos, sin = _tables(7, L, D)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, wq, wk)]
    a, b = fused_qk_norm_rope(leaves[0], leaves[1], leaves[3], leaves[4], cos, sin)
    out = fused_attention(a, b, leaves[2])
    grads = torch.autograd.grad(out, leaves, g)
    # exactly the composition of the two operators on the rounded q and k
    assert torch.equal(out, fused_attention(a.detach(), b.detach(), v))
    want = OA.attention(a.detach(), b.detach(), v, dout=g)
    for i, (x, w, d, n) in enumerate(((q, wq, "dq", a), (k, wk, "dk", b))):
        up, e_up = want[d]
        back = OA.norm_rope(x, w, cos, sin, dout=up)
        # the bound of the incoming gradient goes through the same linear map, with absolute values
        r = torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-6)
        c, s = (t.double()[None, :, None].abs() for t in (cos, sin))
        turned = e_up * c + torch.cat([(e_up * s).chunk(2, -1)[1], (e_up * s).chunk(2, -1)[0]], -1)
        gw, xh = turned * w.double().abs(), (x.double() * r).abs()
        extra = r * (gw + xh * (gw * xh).mean(-1, keepdim=True))
        _within("dx", grads[i], back["dx"], extra=extra * (1 + OA.BF16_HALF))
        _within("dw", grads[3 + i], back["dw"], extra=(turned * xh).sum((0, 1, 2)))
    _within("dv", grads[2], want["dv"])


def test_model_with_padded_texts_and_trainer_run_on_the_kernels():
    """The whole model with the fused attention: the loss agrees with the same arm on SDPA (bf16 roundings in between) and the
    adapters get gradients; text behind a sample's length has no influence. With and without graph capture."""
    from anima_trainer_sm120_b200 import _lib
    from anima_trainer_sm120_b200.anima_dit import tiny_config
    from anima_trainer_sm120_b200.train_step import StepConfig, Trainer
    dev = torch.device(DEV, 0)
    losses = {}
    for attention, graph in (("sdpa", False), ("fused", False), ("fused", True)):
        tr = Trainer(tiny_config(), StepConfig(precision="bf16_fused", lokr_dim=8, lokr_factor=4, attention=attention,
                                               cuda_graph=graph, cuda_graph_warmup=2), dev)
        before = _lib.load().anima_kernel_launches()
        losses[attention, graph] = [tr.step(*tr.synthetic_batch(2, 16, 24, s)) for s in range(4)]
        assert _lib.load().anima_kernel_launches() > before
        assert tr.flat_grad.abs().sum() > 0 and bool(torch.isfinite(tr.flat_grad).all())
    for key in (("fused", False), ("fused", True)):
        for a, b in zip(losses["sdpa", False], losses[key]):
            assert abs(a - b) < 2e-2 * abs(a)
    tr = Trainer(tiny_config(), StepConfig(precision="bf16_fused", lokr_dim=8, lokr_factor=4, attention="fused"), dev)
    lat, ctx, _ = tr.synthetic_batch(2, 16, 24, 0)
    t = torch.tensor([0.3, 0.6], device=dev)
    n = torch.tensor([24, 5], device=dev, dtype=torch.int32)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        y = tr.dit(lat, t, ctx, context_lengths=n)
        ctx2 = ctx.clone()
        ctx2[1, 5:] = 7.0
        assert torch.equal(y, tr.dit(lat, t, ctx2, context_lengths=n))
        assert not torch.equal(y, tr.dit(lat, t, ctx2))
    Trainer(tiny_config(), StepConfig(precision="bf16", lokr_dim=8, lokr_factor=4), dev)       # puts the patches back
    with pytest.raises(ValueError):
        Trainer(tiny_config(), StepConfig(precision="bf16", attention="fused"), dev)
    with pytest.raises(ValueError):
        Trainer(tiny_config(), StepConfig(attention="flash"), dev)
