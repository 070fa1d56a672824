// Softmax attention over (batch, token, head, head_dim) tensors, forward and backward, bf16 in and out.
//
//   s[i, j] = scale * q[i] . k[j],  p[i, j] = exp(s[i, j]) / sum over seen j' of exp(s[i, j']),  out[i] = sum_j p[i, j] v[j]
//   lse[i]  = ln(sum_j exp(s[i, j]))
//   delta[i] = out[i] . dout[i],    ds[i, j] = p[i, j] (dout[i] . v[j] - delta[i])
//   dq[i] = scale * sum_j ds[i, j] k[j],  dk[j] = scale * sum_i ds[i, j] q[i],  dv[j] = sum_i p[i, j] dout[i]
//
// A key is seen by a query if it lies before the sample's length and, causal, at most lk - lq places after the query. A
// query that sees no key has output 0 and lse -inf and takes no part in the gradients. kv_heads may divide heads.
//
// Plain form: one warp a query (or a key, for dk and dv), its head vector spread over the lanes, fp32 throughout.
#include "common.cuh"

namespace anima {
namespace {

constexpr int kWarps = 8;

struct Strided {       // element strides of (batch, token, head); the head vector is dense
  int64_t b, l, h;
};
struct AttnParams {
  const __nv_bfloat16 *q, *k, *v, *out, *dout;
  Strided sq, sk, sv, sdo;
  const int32_t* lengths;
  int lq, lk, heads, kv_heads, causal;
  float scale;
  float* lse;          // [batch, heads, lq]
  float* delta;        // [batch, heads, lq]
  __nv_bfloat16 *o, *dq, *dk, *dv;   // dense
};

template <int D>
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, int lane, float (&x)[D / 32]) {
#pragma unroll
  for (int e = 0; e < D / 32; e += 2) {
    const float2 t = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p + lane * (D / 32) + e));
    x[e] = t.x;
    x[e + 1] = t.y;
  }
}
template <int D>
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, int lane, const float (&x)[D / 32]) {
#pragma unroll
  for (int e = 0; e < D / 32; e += 2)
    *reinterpret_cast<__nv_bfloat162*>(p + lane * (D / 32) + e) = __floats2bfloat162_rn(x[e], x[e + 1]);
}
template <int D>
__device__ __forceinline__ float dot(const float (&a)[D / 32], const float (&b)[D / 32]) {
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) s = fmaf(a[e], b[e], s);
  return warp_sum(s);
}
__device__ __forceinline__ int keys_of(const AttnParams& p, int b) {
  return p.lengths ? max(0, min(p.lk, p.lengths[b])) : p.lk;
}

// grid (ceil(lq / kWarps), heads, batch)
template <int D>
__global__ void __launch_bounds__(kWarps * 32) attention_rows_kernel(const AttnParams p) {
  const int lane = threadIdx.x & 31, i = blockIdx.x * kWarps + (threadIdx.x >> 5), h = blockIdx.y, b = blockIdx.z;
  if (i >= p.lq) return;
  const int hk = h / (p.heads / p.kv_heads);
  int n = keys_of(p, b);
  if (p.causal) n = max(0, min(n, i + p.lk - p.lq + 1));
  const int64_t row = (static_cast<int64_t>(b) * p.heads + h) * p.lq + i;
  const int64_t dense = ((static_cast<int64_t>(b) * p.lq + i) * p.heads + h) * D;
  float q[D / 32], acc[D / 32] = {}, k[D / 32], v[D / 32];
  load_vec<D>(p.q + b * p.sq.b + i * p.sq.l + h * p.sq.h, lane, q);
  const __nv_bfloat16* kp = p.k + b * p.sk.b + hk * p.sk.h;
  const __nv_bfloat16* vp = p.v + b * p.sv.b + hk * p.sv.h;
  {
    float g[D / 32], o[D / 32];
    load_vec<D>(p.dout + b * p.sdo.b + i * p.sdo.l + h * p.sdo.h, lane, g);
    load_vec<D>(p.out + dense, lane, o);
    const float delta = dot<D>(g, o), lse = p.lse[row];
    if (lane == 0) p.delta[row] = delta;
    for (int j = 0; j < n; ++j) {
      load_vec<D>(kp + j * p.sk.l, lane, k);
      load_vec<D>(vp + j * p.sv.l, lane, v);
      const float ds = __expf(dot<D>(q, k) * p.scale - lse) * (dot<D>(g, v) - delta) * p.scale;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) acc[c] = fmaf(ds, k[c], acc[c]);
    }
    if (p.dq) store_vec<D>(p.dq + dense, lane, acc);
  }
}

// grid (ceil(lk / kWarps), kv_heads, batch)
template <int D>
__global__ void __launch_bounds__(kWarps * 32) attention_keys_kernel(const AttnParams p) {
  const int lane = threadIdx.x & 31, j = blockIdx.x * kWarps + (threadIdx.x >> 5), hk = blockIdx.y, b = blockIdx.z;
  if (j >= p.lk) return;
  float k[D / 32], v[D / 32], dk[D / 32] = {}, dv[D / 32] = {}, q[D / 32], g[D / 32];
  const int group = p.heads / p.kv_heads;
  if (j < keys_of(p, b)) {
    load_vec<D>(p.k + b * p.sk.b + j * p.sk.l + hk * p.sk.h, lane, k);
    load_vec<D>(p.v + b * p.sv.b + j * p.sv.l + hk * p.sv.h, lane, v);
    for (int h = hk * group; h < (hk + 1) * group; ++h) {
      const int64_t row = (static_cast<int64_t>(b) * p.heads + h) * p.lq;
      for (int i = p.causal ? max(0, j - (p.lk - p.lq)) : 0; i < p.lq; ++i) {
        load_vec<D>(p.q + b * p.sq.b + i * p.sq.l + h * p.sq.h, lane, q);
        load_vec<D>(p.dout + b * p.sdo.b + i * p.sdo.l + h * p.sdo.h, lane, g);
        const float e = __expf(dot<D>(q, k) * p.scale - p.lse[row + i]);
        const float ds = e * (dot<D>(g, v) - p.delta[row + i]) * p.scale;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          dk[c] = fmaf(ds, q[c], dk[c]);
          dv[c] = fmaf(e, g[c], dv[c]);
        }
      }
    }
  }
  const int64_t dense = ((static_cast<int64_t>(b) * p.lk + j) * p.kv_heads + hk) * D;
  if (p.dk) store_vec<D>(p.dk + dense, lane, dk);
  if (p.dv) store_vec<D>(p.dv + dense, lane, dv);
}

int check_sizes(const char* who, int64_t batch, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  ANIMA_REQUIRE(batch >= 0 && lq >= 0 && lk >= 0 && heads > 0 && kv_heads > 0, ANIMA_E_ARG, "%s: bad sizes", who);
  ANIMA_REQUIRE(head_dim == 64 || head_dim == 128, ANIMA_E_UNSUPPORTED, "%s: head_dim=%lld is not supported (64 or 128)", who,
                (long long)head_dim);
  ANIMA_REQUIRE(heads % kv_heads == 0, ANIMA_E_SHAPE, "%s: heads=%lld is not a multiple of kv_heads=%lld", who,
                (long long)heads, (long long)kv_heads);
  ANIMA_REQUIRE(batch < 65536 && heads < 65536 && lq < (1ll << 30) && lk < (1ll << 30) && batch * heads * lq < (1ll << 40),
                ANIMA_E_TOO_LARGE, "%s: too large", who);
  return ANIMA_OK;
}
int check_tensor(const char* who, const char* name, const void* p, const int64_t* s, bool empty) {
  ANIMA_REQUIRE(s, ANIMA_E_ARG, "%s: strides of %s are missing", who, name);
  ANIMA_REQUIRE(p || empty, ANIMA_E_ARG, "%s: null pointer (%s)", who, name);
  ANIMA_REQUIRE(s[0] >= 0 && s[1] >= 0 && s[2] >= 0, ANIMA_E_ARG, "%s: negative stride of %s", who, name);
  ANIMA_REQUIRE(aligned16(p) && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0, ANIMA_E_ALIGN,
                "%s: %s must be 16-byte aligned, its strides multiples of 8 elements", who, name);
  return ANIMA_OK;
}
Strided strided(const int64_t* s) { return {s[0], s[1], s[2]}; }

}  // namespace
}  // namespace anima

using namespace anima;

extern "C" int64_t anima_attention_bwd_workspace_bytes(int64_t batch, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads,
                                                       int64_t head_dim, int causal) {
  (void)causal;
  if (int rc = check_sizes("attention_bwd", batch, lq, lk, heads, kv_heads, head_dim)) return rc;
  return batch * heads * lq * 4;
}

extern "C" int anima_attention_bwd(const void* dout, const int64_t* dout_strides, const void* q, const int64_t* q_strides,
                                   const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                   const void* out, const float* lse, const int32_t* kv_lengths, int64_t batch, int64_t lq,
                                   int64_t lk, int64_t heads, int64_t kv_heads, int64_t head_dim, float scale, int causal,
                                   void* dq, void* dk, void* dv, void* workspace, int64_t workspace_bytes, int32_t* status,
                                   void* stream) {
  const char* who = "attention_bwd";
  (void)status;
  const int64_t need = anima_attention_bwd_workspace_bytes(batch, lq, lk, heads, kv_heads, head_dim, causal);
  if (need < 0) return (int)need;
  ANIMA_REQUIRE(scale > 0.f && scale < INFINITY, ANIMA_E_ARG, "%s: scale must be positive and finite", who);
  const bool no_q = batch * lq == 0, no_k = batch * lk == 0;
  if (int rc = check_tensor(who, "dout", dout, dout_strides, no_q)) return rc;
  if (int rc = check_tensor(who, "q", q, q_strides, no_q)) return rc;
  if (int rc = check_tensor(who, "k", k, k_strides, no_k)) return rc;
  if (int rc = check_tensor(who, "v", v, v_strides, no_k)) return rc;
  ANIMA_REQUIRE(no_q || (out && lse), ANIMA_E_ARG, "%s: null pointer", who);
  ANIMA_REQUIRE(aligned16(out) && aligned16(dq) && aligned16(dk) && aligned16(dv) && aligned16(workspace), ANIMA_E_ALIGN,
                "%s: tensors must be 16-byte aligned", who);
  ANIMA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), ANIMA_E_WORKSPACE, "%s: workspace of %lld bytes, %lld needed",
                who, (long long)workspace_bytes, (long long)need);
  AttnParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.out = static_cast<const __nv_bfloat16*>(out);
  p.dout = static_cast<const __nv_bfloat16*>(dout);
  p.sq = strided(q_strides);
  p.sk = strided(k_strides);
  p.sv = strided(v_strides);
  p.sdo = strided(dout_strides);
  p.lengths = kv_lengths;
  p.lq = (int)lq; p.lk = (int)lk; p.heads = (int)heads; p.kv_heads = (int)kv_heads; p.causal = causal;
  p.scale = scale;
  p.lse = const_cast<float*>(lse);
  p.delta = static_cast<float*>(workspace);
  p.dq = static_cast<__nv_bfloat16*>(dq);
  p.dk = static_cast<__nv_bfloat16*>(dk);
  p.dv = static_cast<__nv_bfloat16*>(dv);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!no_q) {
    const dim3 grid((unsigned)ceil_div(lq, kWarps), (unsigned)heads, (unsigned)batch);
    if (head_dim == 64) attention_rows_kernel<64><<<grid, kWarps * 32, 0, s>>>(p);
    else attention_rows_kernel<128><<<grid, kWarps * 32, 0, s>>>(p);
    ANIMA_CHECK_LAUNCH(who);
  }
  if (!no_k && (dk || dv)) {
    const dim3 grid((unsigned)ceil_div(lk, kWarps), (unsigned)kv_heads, (unsigned)batch);
    if (head_dim == 64) attention_keys_kernel<64><<<grid, kWarps * 32, 0, s>>>(p);
    else attention_keys_kernel<128><<<grid, kWarps * 32, 0, s>>>(p);
    ANIMA_CHECK_LAUNCH(who);
  }
  return ANIMA_OK;
}
