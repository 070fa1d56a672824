#include "attention.h"

namespace anima_host {

using torch::autograd::set_history;

namespace {

// Nothing here has a gradient of its own: a backward pass that is itself recorded would lose it without notice.
void refuse_second_order(const char* who) {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), who, ": the backward pass cannot be differentiated (create_graph)");
}

// A (batch, token, head, D) tensor as the kernels take it: the head vector dense, the other strides multiples of 16 bytes.
// What does not fit (also an expanded dimension) is copied; the stride of a dimension of size 1 counts for nothing.
struct Heads {
  Tensor t;
  int64_t s[3];
  const void* ptr() const { return t.data_ptr(); }
};
bool usable(const Tensor& t) {
  if (t.size(3) > 1 && t.stride(3) != 1) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && (t.stride(i) <= 0 || t.stride(i) % 8 != 0)) return false;
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}
Heads heads_of(const Tensor& x) {
  Heads h{x, {}};
  if (h.t.scalar_type() != BF16) h.t = h.t.detach().to(BF16);
  if (!usable(h.t)) h.t = h.t.detach().clone(at::MemoryFormat::Contiguous);
  int64_t dense = h.t.size(3);
  for (int i = 2; i >= 0; --i) {
    h.s[i] = h.t.size(i) > 1 ? h.t.stride(i) : dense;
    dense *= std::max<int64_t>(1, h.t.size(i));
  }
  // the order of the strides is (batch, token, head): sizes (B, L, H, D)
  return h;
}
Tensor dense_like(const Tensor& t, const at::Device& dev) { return at::detail::empty_cuda(t.sizes(), BF16, dev, std::nullopt); }
Tensor scratch(int64_t bytes, const at::Device& dev) { return bytes ? empty({bytes}, U8, dev) : Tensor(); }

void check_qk(const char* who, const Tensor& q, const Tensor& k) {
  TORCH_CHECK_TYPE(q.scalar_type() == BF16 && k.scalar_type() == BF16, who, " needs bfloat16, got ", q.scalar_type(), " and ",
                   k.scalar_type());
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4, who, ": tensors must be (batch, tokens, heads, head_dim), got ", q.sizes(), " and ",
                    k.sizes());
  TORCH_CHECK_VALUE(q.size(0) == k.size(0) && q.size(3) == k.size(3), who, ": q ", q.sizes(), " does not go with k ", k.sizes());
}

// ------------------------------------------------------------------------------------------------ attention
struct AttentionNode : public HostNode {
  Kept lengths;
  double scale = 0;
  bool causal = false;

  variable_list apply(variable_list&& g) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const bool want[3] = {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2)};
    if (!(want[0] || want[1] || want[2])) return variable_list(3);
    refuse_second_order("fused_attention");
    const Tensor dout = grad_of(g, 0);
    const Heads q = heads_of(get(0)), k = heads_of(get(1)), v = heads_of(get(2));
    const Tensor out_ = get(3), lse = get(4);
    const Launch l(q.t);
    Below below;
    const Heads go = heads_of(dout);
    const Tensor out = bf16_contiguous(out_);
    Tensor d[3];
    for (int i = 0; i < 3; ++i)
      if (want[i]) d[i] = dense_like(i == 0 ? q.t : k.t, l.dev);
    const Tensor& n = lengths.get();
    const int64_t B = q.t.size(0), lq = q.t.size(1), H = q.t.size(2), D = q.t.size(3), lk = k.t.size(1), Hk = k.t.size(2);
    const int64_t bytes = check(anima_attention_bwd_workspace_bytes(B, lq, lk, H, Hk, D, causal));
    const Tensor ws = scratch(bytes, l.dev);
    check(anima_attention_bwd(go.ptr(), go.s, q.ptr(), q.s, k.ptr(), k.s, v.ptr(), v.s, out.data_ptr(), lse.data_ptr<float>(),
                              n.defined() ? n.data_ptr<int32_t>() : nullptr, B, lq, lk, H, Hk, D, static_cast<float>(scale), causal,
                              ptr(d[0]), ptr(d[1]), ptr(d[2]), ptr(ws), bytes, status_word(l.dev), l.stream));
    return {d[0], d[1], d[2]};
  }
  std::string name() const override { return "FusedAttentionBackward"; }
};

// ------------------------------------------------------------------------------------------------ q / k norm and rotation
struct Tables {
  Tensor cos, sin;
  int64_t samples = 1;
  const float* c() const { return cos.defined() ? cos.data_ptr<float>() : nullptr; }
  const float* s() const { return sin.defined() ? sin.data_ptr<float>() : nullptr; }
};
Tensor table_of(const Tensor& t) {
  Tensor d = cast(t.detach(), F32);
  if (!d.is_contiguous() || (reinterpret_cast<uintptr_t>(d.data_ptr()) & 15)) d = d.clone(at::MemoryFormat::Contiguous);
  return d;
}
Tables tables_of(const OptTensor& cos, const OptTensor& sin, const Tensor& q, const Tensor& k) {
  Tables t;
  const bool has = cos && cos->defined();
  TORCH_CHECK_VALUE(has == (sin && sin->defined()), "fused_qk_norm_rope: give both tables or neither");
  if (!has) return t;
  TORCH_CHECK_VALUE(q.size(1) == k.size(1), "fused_qk_norm_rope: one table for ", q.size(1), " queries and ", k.size(1), " keys");
  TORCH_CHECK_VALUE(cos->sizes() == sin->sizes(), "fused_qk_norm_rope: tables of different shapes ", cos->sizes(), " and ", sin->sizes());
  TORCH_CHECK_VALUE((cos->dim() == 2 || (cos->dim() == 3 && (cos->size(0) == 1 || cos->size(0) == q.size(0)))) &&
                        cos->size(-2) == q.size(1) && cos->size(-1) == q.size(3),
                    "fused_qk_norm_rope: rope tables ", cos->sizes(), " for q ", q.sizes());
  t.cos = table_of(*cos);
  t.sin = table_of(*sin);
  t.samples = cos->dim() == 3 ? cos->size(0) : 1;
  return t;
}
// both norm weights as the kernels read them: bf16 or fp32, one type for the two
struct Weights {
  Tensor q, k;
  bool bf16;
};
Weights weights_of(const Tensor& wq, const Tensor& wk) {
  const bool bf16 = wq.scalar_type() == BF16 && wk.scalar_type() == BF16;
  auto one = [&](const Tensor& w) {
    Tensor d = bf16 || w.scalar_type() == F32 ? w : w.detach().to(F32);
    if (!d.is_contiguous() || (reinterpret_cast<uintptr_t>(d.data_ptr()) & 15)) d = d.detach().clone(at::MemoryFormat::Contiguous);
    return d;
  };
  return {one(wq), one(wk), bf16};
}

struct QkNormRopeNode : public HostNode {
  Kept cos, sin;
  int64_t samples = 1;
  double eps = 0;

  variable_list apply(variable_list&& g) override {
    std::lock_guard<std::mutex> lock(mutex_);
    bool want[4];
    for (int i = 0; i < 4; ++i) want[i] = task_should_compute_output(i);
    if (!(want[0] || want[1] || want[2] || want[3])) return variable_list(4);
    refuse_second_order("fused_qk_norm_rope");
    const Tensor gq_ = grad_of(g, 0), gk_ = grad_of(g, 1);
    const Heads q = heads_of(get(0)), k = heads_of(get(1));
    const Tensor wq = get(2), wk = get(3);
    const Launch l(q.t);
    Below below;
    const Tensor gq = aligned(gq_), gk = aligned(gk_);
    const Weights w = weights_of(wq, wk);
    const int64_t B = q.t.size(0), lq = q.t.size(1), H = q.t.size(2), D = q.t.size(3), lk = k.t.size(1), Hk = k.t.size(2);
    Tensor dq = dense_like(q.t, l.dev), dk = dense_like(k.t, l.dev), dw[2];
    for (int i = 0; i < 2; ++i)
      if (want[2 + i]) dw[i] = empty({D}, w.bf16 ? BF16 : F32, l.dev);
    const int64_t bytes = dw[0].defined() || dw[1].defined() ? check(anima_qk_norm_rope_bwd_workspace_bytes(B, lq, lk, H, Hk, D)) : 0;
    const Tensor ws = scratch(bytes, l.dev), &c = cos.get(), &s = sin.get();
    check(anima_qk_norm_rope_bwd(gq.data_ptr(), gk.data_ptr(), q.ptr(), q.s, k.ptr(), k.s, w.q.data_ptr(), w.k.data_ptr(), w.bf16,
                                 static_cast<float*>(ptr(c)), static_cast<float*>(ptr(s)), samples, static_cast<float>(eps), B, lq, lk,
                                 H, Hk, D, dq.data_ptr(), dk.data_ptr(), ptr(dw[0]), ptr(dw[1]), ptr(ws), bytes, l.stream));
    auto back = [](const Tensor& t, const Tensor& w) { return t.defined() ? cast(t, w.scalar_type()).view(w.sizes()) : t; };
    return {dq, dk, back(dw[0], wq), back(dw[1], wk)};
  }
  static Tensor aligned(const Tensor& t) {
    const Tensor d = bf16_contiguous(t);
    return reinterpret_cast<uintptr_t>(d.data_ptr()) & 15 ? d.detach().clone(at::MemoryFormat::Contiguous) : d;
  }
  std::string name() const override { return "FusedQKNormRoPEBackward"; }
};

}  // namespace

std::tuple<Tensor, OptTensor> attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const OptTensor& lengths_, bool causal,
                                        double scale, bool want_lse) {
  check_qk("fused_attention", q_, k_);
  TORCH_CHECK_TYPE(v_.scalar_type() == BF16, "fused_attention needs bfloat16, got ", v_.scalar_type());
  TORCH_CHECK_VALUE(v_.sizes() == k_.sizes(), "fused_attention: v ", v_.sizes(), " does not go with k ", k_.sizes());
  const Launch l(q_);
  admit(l, q_, k_, v_, lengths_);
  const int64_t B = q_.size(0), lq = q_.size(1), H = q_.size(2), D = q_.size(3), lk = k_.size(1), Hk = k_.size(2);
  const bool grad = any_wants(q_, k_, v_);
  Tensor out, lse, lengths;
  Heads q, k, v;
  {
    Below below;
    if (lengths_ && lengths_->defined()) {
      TORCH_CHECK_TYPE(lengths_->scalar_type() == at::kInt || lengths_->scalar_type() == at::kLong,
                       "fused_attention: kv_lengths must be int32 or int64, got ", lengths_->scalar_type());
      TORCH_CHECK_VALUE(lengths_->dim() == 1 && lengths_->size(0) == B, "fused_attention: kv_lengths must be [", B, "], got ",
                        lengths_->sizes());
      lengths = cast(*lengths_, at::kInt).contiguous();
    }
    q = heads_of(q_);
    k = heads_of(k_);
    v = heads_of(v_);
    out = dense_like(q.t, l.dev);
    if (grad || want_lse) lse = empty({B, H, lq}, F32, l.dev);
    const int64_t bytes = check(anima_attention_fwd_workspace_bytes(B, lq, lk, H, Hk, D, causal));
    const Tensor ws = scratch(bytes, l.dev);
    check(anima_attention_fwd(q.ptr(), q.s, k.ptr(), k.s, v.ptr(), v.s, lengths.defined() ? lengths.data_ptr<int32_t>() : nullptr, B,
                              lq, lk, H, Hk, D, static_cast<float>(scale), causal, out.data_ptr(),
                              lse.defined() ? lse.data_ptr<float>() : nullptr, ptr(ws), bytes, status_word(l.dev), l.stream));
  }
  if (grad) {
    auto node = make_node<AttentionNode>(q_, k_, v_);
    set_history(out, node);
    node->save(q.t);
    node->save(k.t);
    node->save(v.t);
    node->save(out, true);
    node->save(lse);
    node->lengths = Kept(lengths);
    node->scale = scale;
    node->causal = causal;
  }
  return {out, want_lse ? OptTensor(lse) : OptTensor()};
}

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q_, const Tensor& k_, const Tensor& wq, const Tensor& wk, const OptTensor& cos,
                                        const OptTensor& sin, double eps) {
  check_qk("fused_qk_norm_rope", q_, k_);
  const int64_t B = q_.size(0), lq = q_.size(1), H = q_.size(2), D = q_.size(3), lk = k_.size(1), Hk = k_.size(2);
  TORCH_CHECK_VALUE(wq.numel() == D && wk.numel() == D, "fused_qk_norm_rope: norm weights of ", wq.numel(), " and ", wk.numel(),
                    " elements for heads of ", D);
  TORCH_CHECK_TYPE(wq.is_floating_point() && wk.is_floating_point(), "fused_qk_norm_rope: norm weights must be floating point");
  const Launch l(q_);
  admit(l, q_, k_, wq, wk, cos, sin);
  TORCH_CHECK_NOT_IMPLEMENTED(!wants(cos) && !wants(sin), "fused_qk_norm_rope: no gradient for the rope tables");
  const bool grad = any_wants(q_, k_, wq, wk);
  Tensor oq, ok;
  Heads q, k;
  Tables t;
  {
    Below below;
    t = tables_of(cos, sin, q_, k_);
    q = heads_of(q_);
    k = heads_of(k_);
    const Weights w = weights_of(wq, wk);
    oq = dense_like(q.t, l.dev);
    ok = dense_like(k.t, l.dev);
    check(anima_qk_norm_rope_fwd(q.ptr(), q.s, k.ptr(), k.s, w.q.data_ptr(), w.k.data_ptr(), w.bf16, t.c(), t.s(), t.samples,
                                 static_cast<float>(eps), B, lq, lk, H, Hk, D, oq.data_ptr(), ok.data_ptr(), l.stream));
  }
  if (grad) {
    auto node = make_node<QkNormRopeNode>(q_, k_, wq, wk);
    set_history(oq, node);
    set_history(ok, node);
    node->save(q.t);
    node->save(k.t);
    node->save(wq);
    node->save(wk);
    node->cos = Kept(t.cos);
    node->sin = Kept(t.sin);
    node->samples = t.samples;
    node->eps = eps;
  }
  return {oq, ok};
}

}  // namespace anima_host
