"""CPU-side checks of the attention operators: the oracle against autograd of the textbook softmax, the model's padded texts,
and the refusals of the C ABI, which answer before anything touches a device."""
from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import attention as OA


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Lq,Lk", [(5, 9), (9, 5), (7, 7)])
def test_oracle_matches_autograd_of_softmax(Lq, Lk, causal):
    g = torch.Generator().manual_seed(Lq)
    B, H, Hk, D = 2, 4, 2, 8
    q, k, v, dout = (torch.randn(B, L, h, D, generator=g, dtype=torch.float64) for L, h in ((Lq, H), (Lk, Hk), (Lk, Hk), (Lq, H)))
    n = torch.tensor([Lk, Lk - 2])
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    a, b, c = (t.repeat_interleave(H // t.shape[2], 2).transpose(1, 2) for t in leaves)
    seen = OA.visible(B, Lq, Lk, n, causal)
    s = (a @ b.mT * D ** -0.5).masked_fill(~seen, -1e30)
    out = torch.where(seen.any(-1, keepdim=True), torch.softmax(s, -1), 0.0) @ c
    grads = torch.autograd.grad(out, leaves, dout.transpose(1, 2))
    want = OA.attention(q, k, v, lengths=n, causal=causal, dout=dout)
    for x, name in zip((out.transpose(1, 2), *grads), ("out", "dq", "dk", "dv")):
        torch.testing.assert_close(want[name][0], x, rtol=1e-10, atol=1e-12)
        assert bool((want[name][1] >= 0).all())
    torch.testing.assert_close(want["lse"][0], torch.logsumexp(s.masked_fill(~seen, -torch.inf), -1), rtol=1e-12, atol=0)


def test_oracle_of_norm_and_rotation_matches_autograd_and_the_model():
    from anima_trainer_sm120_b200.anima_dit import RMSNorm, apply_rotary_pos_emb
    g = torch.Generator().manual_seed(1)
    x, dout = (torch.randn(2, 5, 3, 8, generator=g, dtype=torch.float64) for _ in range(2))
    norm = RMSNorm(8).double()
    norm.weight.data = torch.randn(8, generator=g, dtype=torch.float64)
    ang = torch.rand(5, 1, 1, 8, generator=g, dtype=torch.float64)
    xi = x.clone().requires_grad_(True)
    xf = xi * torch.rsqrt(xi.pow(2).mean(-1, keepdim=True) + 1e-6) * norm.weight
    out = apply_rotary_pos_emb(xf, ang)
    dx, dw = torch.autograd.grad(out, (xi, norm.weight), dout)
    want = OA.norm_rope(x, norm.weight.detach(), ang.flatten(1).cos(), ang.flatten(1).sin(), dout=dout)
    for a, n in ((out, "out"), (dx, "dx"), (dw, "dw")):
        torch.testing.assert_close(want[n][0], a.detach(), rtol=1e-10, atol=1e-12)


def test_model_hides_the_text_behind_a_samples_length():
    from anima_trainer_sm120_b200.anima_dit import AnimaDiT, tiny_config
    torch.manual_seed(0)
    dit = AnimaDiT(tiny_config(depth=1))
    x, t, ctx = torch.randn(2, 16, 1, 4, 4), torch.tensor([0.2, 0.7]), torch.randn(2, 6, 128)
    with torch.no_grad():
        full = dit(x, t, ctx)
        assert torch.allclose(full, dit(x, t, ctx, context_lengths=torch.tensor([6, 6])), atol=1e-5)
        cut = dit(x, t, ctx, context_lengths=torch.tensor([6, 2]))
        ctx[1, 2:] = 100.0
        assert torch.equal(cut, dit(x, t, ctx, context_lengths=torch.tensor([6, 2])))
        assert torch.allclose(cut[0], full[0], atol=1e-5) and not torch.allclose(cut[1], full[1], atol=1e-5)


def test_patches_leave_cpu_tensors_to_the_eager_methods():
    from anima_trainer_sm120_b200 import attention_patch, qk_norm_rope
    from anima_trainer_sm120_b200.anima_dit import Attention, tiny_config
    torch.manual_seed(0)
    attn, x = Attention(tiny_config(), None), torch.randn(1, 5, 256)
    rope = torch.rand(5, 1, 1, 64)
    want = attn(x, rope_emb=rope)
    before = Attention._attend, Attention._prepare_qk
    try:
        attention_patch.install(Attention)
        attention_patch.install(Attention)
        qk_norm_rope.install(Attention, joint=True)
        assert torch.equal(want, attn(x, rope_emb=rope))
    finally:
        attention_patch.uninstall(Attention)
        qk_norm_rope.uninstall(Attention)
    assert (Attention._attend, Attention._prepare_qk) == before


def _ptr(offset=0):
    buf = (ctypes.c_uint8 * 4096)()
    _ptr.keep = buf
    return ((ctypes.addressof(buf) + 15) & ~15) + offset


def _attention(lib, name="fwd", q=None, qs=(512, 128, 64), ks=(512, 128, 64), sizes=(1, 4, 4, 2, 2, 64), scale=1.0, ws=0):
    p = _ptr() if q is None else q
    o = _ptr()
    three = lambda s: (ctypes.c_int64 * 3)(*s) if s else None
    if name == "fwd":
        return lib.anima_attention_fwd(p, three(qs), o, three(ks), o, three(ks), None, *sizes, scale, 0, o, None, None, 0, None, None)
    return lib.anima_attention_bwd(p, three(qs), o, three(qs), o, three(ks), o, three(ks), o, o, None, *sizes, scale, 0, o, o, o,
                                   o if ws else None, ws, None, None)


@pytest.mark.parametrize("name", ["fwd", "bwd"])
def test_attention_entries_refuse_before_any_launch(lib, name):
    go = lambda **kw: _attention(lib, name, **kw)
    assert go(q=0) == -1 and b"null" in lib.anima_last_error()
    assert go(qs=None) == -1
    assert go(q=_ptr(2)) == -2
    assert go(qs=(512, 127, 64)) == -2 and go(ks=(512, 128, 4)) == -2
    assert go(qs=(512, -128, 64)) == -1
    assert go(sizes=(1, 4, 4, 2, 2, 96)) == -5
    assert go(sizes=(1, 4, 4, 3, 2, 64)) == -3
    assert go(sizes=(-1, 4, 4, 2, 2, 64)) == -1 and go(sizes=(1, 4, 4, 0, 2, 64)) == -1
    assert go(sizes=(1 << 20, 4, 4, 2, 2, 64)) == -7 and go(sizes=(1, 1 << 31, 4, 2, 2, 64)) == -7
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert go(scale=scale) == -1
    if name == "bwd":
        assert go(ws=0) == -6 and go(ws=8) == -6
    size = getattr(lib, f"anima_attention_{name}_workspace_bytes")
    assert size(1, 4, 4, 2, 2, 64, 0) >= 0 and size(1, 4, 4, 3, 2, 64, 0) == -3 and size(1, 4, 4, 2, 2, 32, 0) == -5


def test_qk_norm_rope_entries_refuse_before_any_launch(lib):
    p = _ptr()

    def fwd(q=p, qs=(512, 128, 64), w=p, cos=None, sin=None, samples=1, sizes=(1, 4, 4, 2, 2, 64)):
        s = (ctypes.c_int64 * 3)(*qs)
        return lib.anima_qk_norm_rope_fwd(q, s, p, s, w, p, 1, cos, sin, samples, 1e-6, *sizes, p, p, None)

    assert fwd(q=None) == -1 and fwd(w=None) == -1
    assert fwd(q=p + 2) == -2 and fwd(w=p + 8) == -2 and fwd(qs=(512, 128, 4)) == -2
    assert fwd(cos=p) == -1
    assert fwd(cos=p, sin=p, samples=3) == -3 and fwd(cos=p, sin=p, sizes=(1, 4, 5, 2, 2, 64)) == -3
    assert fwd(cos=p + 4, sin=p) == -2
    assert fwd(sizes=(1, 4, 4, 2, 2, 80)) == -5 and fwd(sizes=(1, 4, 4, 0, 2, 64)) == -1
    assert fwd(sizes=(1 << 20, 1 << 20, 4, 2, 2, 64)) == -7
    s = (ctypes.c_int64 * 3)(512, 128, 64)
    bwd = lambda dw, ws: lib.anima_qk_norm_rope_bwd(p, p, p, s, p, s, p, p, 1, None, None, 1, 1e-6, 1, 4, 4, 2, 2, 64, p, p, dw, None,
                                                    p if ws else None, ws, None)
    assert bwd(p, 0) == -6 and bwd(p, 16) == -6
    assert lib.anima_qk_norm_rope_bwd_workspace_bytes(1, 4, 4, 2, 2, 64) > 0
    assert lib.anima_qk_norm_rope_bwd_workspace_bytes(1, 4, 4, 2, 2, 32) == -5


def test_python_entries_refuse_cpu_tensors():
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    from anima_trainer_sm120_b200.qk_norm_rope import fused_qk_norm_rope
    x = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_attention(x, x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_qk_norm_rope(x, x, x[0, 0, 0], x[0, 0, 0])


def test_trainer_options_are_checked_before_anything_is_built():
    from anima_trainer_sm120_b200.anima_dit import tiny_config
    from anima_trainer_sm120_b200.train_step import StepConfig, Trainer
    cpu = torch.device("cpu")
    with pytest.raises(ValueError, match="attention"):
        Trainer(tiny_config(), StepConfig(precision="bf16", attention="fused"), cpu)
    with pytest.raises(ValueError, match="attention"):
        Trainer(tiny_config(), StepConfig(precision="bf16", attention="other"), cpu)
    with pytest.raises(RuntimeError, match="CUDA"):
        Trainer(tiny_config(), StepConfig(precision="bf16_fused", attention="fused"), cpu)
    Trainer(tiny_config(), StepConfig(precision="bf16", lokr_dim=8, lokr_factor=4), cpu)


def test_ops_wrappers_refuse_what_they_cannot_pass_on():
    from anima_trainer_sm120_b200 import ops
    x = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.attention_fwd(x, x, x), lambda: ops.attention_bwd(x, x, x, x, x, x),
                 lambda: ops.qk_norm_rope_fwd(x, x, x[0, 0, 0], x[0, 0, 0], None, None, 1e-6),
                 lambda: ops.qk_norm_rope_bwd(x, x, x, x, x[0, 0, 0], x[0, 0, 0], None, None, 1e-6)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_patch_reaches_a_class_derived_from_the_patched_one():
    from anima_trainer_sm120_b200 import attention_patch
    from anima_trainer_sm120_b200.anima_dit import AnimaConfig, Attention

    class Derived(Attention):
        pass

    cfg = AnimaConfig(dim=128, heads=2, depth=1)
    module = Derived(cfg, None)
    q, k, v = (torch.randn(1, 5, 2, cfg.head_dim) for _ in range(3))
    want = module._attend(q, k, v)
    attention_patch.install(Attention)
    try:
        assert torch.equal(module._attend(q, k, v), want)          # CPU tensors: the original method
    finally:
        attention_patch.uninstall(Attention)
