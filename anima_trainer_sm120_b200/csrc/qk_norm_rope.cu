// Per-head RMSNorm of the queries AND the keys with the rotary embedding, in one launch; backward with the gradients of both
// norm weights.
//
//   r = rsqrt(mean(x^2) + eps),  n = x r w,  out1 = n1 c1 - n2 s1,  out2 = n2 c2 + n1 s2     (1 / 2: halves of a head vector)
//   dn1 = g1 c1 + g2 s2,  dn2 = g2 c2 - g1 s1,  gw = dn w,  dx = r (gw - x r mean(gw x r)),  dw = sum over vectors of dn x r
//
// Bound by memory: forward reads and writes each element once (4 bytes), backward reads the gradient and x and writes dx (6);
// 1 / rms is made again from x in backward, so forward leaves nothing but its result.
// A token's lanes walk its heads with the folded rotation in registers (head_vectors.cuh), loads run ahead through the
// cp.async ring; q and k differ in pointers, strides, heads and weight only, so the CTAs of q come first and those of k
// after them, and the tail of one overlaps the start of the other.
// The weight's gradient needs no rotation per head: sum over heads of dn1 x1 r = c1 sum(g1 x1 r) + s2 sum(g2 x1 r) (and
// likewise dn2), so four products are summed over a token's heads and rotated once. Per-CTA partials, then one CTA a column
// block adds them in ascending order: reproducible, no atomics.
#include "head_vectors.cuh"

namespace anima {
namespace {

using namespace headvec;

constexpr int kThreads = 256;
constexpr int kFwdStages = 6, kBwdStages = 4;

struct Side {                  // queries or keys
  const __nv_bfloat16* x;
  const __nv_bfloat16* g;      // backward: dense gradient of the result
  __nv_bfloat16* out;          // dense result, or dx
  const void* w;
  float* partial;              // [ctas, D], null: no weight gradient
  void* dw;
  int64_t sb, sl, sh;          // strides of x (elements)
  int64_t len, tokens;         // tokens a sample, in all
  int heads, heads_per_group, groups, ctas;
};
struct PairParams {
  Side side[2];
  const float *cos, *sin;
  int64_t table_step;          // rows from one sample's table to the next
  float eps;
};

template <int D, int THREADS>
struct Place {                 // where a thread works
  static constexpr int kLanes = D / 16, kTokens = THREADS / kLanes;
  int64_t x_at, dense_at, pos;
  int h0, h1, lane, cta;
  unsigned mask;
  bool live;
  __device__ __forceinline__ Place(const Side& s, int cta_, int64_t table_step) : cta(cta_) {
    lane = threadIdx.x & (kLanes - 1);
    mask = ((1u << kLanes) - 1) << (threadIdx.x & 31 & ~(kLanes - 1));
    const int64_t token = static_cast<int64_t>(cta / s.groups) * kTokens + threadIdx.x / kLanes;
    const int group = cta % s.groups;
    live = token < s.tokens;
    const int64_t t = live ? token : 0, b = t / s.len, at = t - b * s.len;
    h0 = group * s.heads_per_group;
    h1 = live ? min(s.heads, h0 + s.heads_per_group) : h0;
    pos = b * table_step + at;
    x_at = b * s.sb + at * s.sl + lane * 8;
    dense_at = t * s.heads * D + lane * 8;
  }
};

template <int D, bool ROPE, bool WBF16>
__global__ void __launch_bounds__(kThreads, 2) qk_norm_rope_fwd_kernel(const __grid_constant__ PairParams p) {
  after_previous();
  const bool second = static_cast<int>(blockIdx.x) >= p.side[0].ctas;
  const Side& s = p.side[second];
  const Place<D, kThreads> at(s, static_cast<int>(blockIdx.x) - (second ? p.side[0].ctas : 0), p.table_step);
  if (!at.live) return;        // a token's lanes leave together; shuffles below stay inside them
  const __nv_bfloat16* x = after_previous(s.x);
  Rotation r;
  load_rotation<D, ROPE, WBF16>(r, after_previous(s.w), after_previous(p.cos), after_previous(p.sin), at.pos, at.lane);
  extern __shared__ uint4 ring_smem[];
  const Ring<2, kFwdStages, kThreads> ring(ring_smem);
  auto start = [&](int h, int slot) {
    if (h < at.h1) {
      ring.copy(slot, 0, x + at.x_at + h * s.sh);
      ring.copy(slot, 1, x + at.x_at + h * s.sh + D / 2);
    }
    ring.commit();
  };
#pragma unroll
  for (int i = 0; i < kFwdStages - 1; ++i) start(at.h0 + i, i);
  int slot = 0;
#pragma unroll 1
  for (int h = at.h0; h < at.h1; ++h) {
    ring.wait();
    f2 v1[4], v2[4];
    widen(ring.read(slot, 0), v1);
    widen(ring.read(slot, 1), v2);
    start(h + kFwdStages - 1, slot == 0 ? kFwdStages - 1 : slot - 1);   // the slot used one head ago
    slot = slot + 1 == kFwdStages ? 0 : slot + 1;
    f2 q0 = f2_mul(v1[0], v1[0]), q1 = f2_mul(v2[0], v2[0]);
#pragma unroll
    for (int e = 1; e < 4; ++e) {
      q0 = f2_fma(v1[e], v1[e], q0);
      q1 = f2_fma(v2[e], v2[e], q1);
    }
    const f2 rs = f2_dup(rsqrtf(lanes_sum<D / 16>(f2_sum(f2_add(q0, q1)), at.mask) / D + p.eps));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f2 o1 = f2_mul(v1[e], r.a1[e]), o2 = f2_mul(v2[e], r.a2[e]);
      if (ROPE) {
        o1 = f2_fma(v2[e], r.b1[e], o1);
        o2 = f2_fma(v1[e], r.b2[e], o2);
      }
      v1[e] = f2_mul(o1, rs);
      v2[e] = f2_mul(o2, rs);
    }
    stg_stream16(s.out + at.dense_at + h * D, narrow(v1));
    stg_stream16(s.out + at.dense_at + h * D + D / 2, narrow(v2));
  }
}

// DW: also the weight's gradient, as a partial of this CTA. Its four products take 32 more registers, so such a CTA has
// half the threads.
template <int D, bool ROPE, bool WBF16, bool DW>
__global__ void __launch_bounds__(DW ? kThreads / 2 : kThreads, DW ? 3 : 2)
qk_norm_rope_bwd_kernel(const __grid_constant__ PairParams p) {
  constexpr int THREADS = DW ? kThreads / 2 : kThreads;
  after_previous();
  const bool second = static_cast<int>(blockIdx.x) >= p.side[0].ctas;
  const Side& s = p.side[second];
  const Place<D, THREADS> at(s, static_cast<int>(blockIdx.x) - (second ? p.side[0].ctas : 0), p.table_step);
  const __nv_bfloat16 *x = after_previous(s.x), *g = after_previous(s.g);
  Rotation r;
  load_rotation<D, ROPE, WBF16>(r, after_previous(s.w), after_previous(p.cos), after_previous(p.sin), at.pos, at.lane);
  extern __shared__ uint4 ring_smem[];
  const Ring<4, kBwdStages, THREADS> ring(ring_smem);
  auto start = [&](int h, int slot) {
    if (h < at.h1) {
      ring.copy(slot, 0, g + at.dense_at + h * D);
      ring.copy(slot, 1, g + at.dense_at + h * D + D / 2);
      ring.copy(slot, 2, x + at.x_at + h * s.sh);
      ring.copy(slot, 3, x + at.x_at + h * s.sh + D / 2);
    }
    ring.commit();
  };
#pragma unroll
  for (int i = 0; i < kBwdStages - 1; ++i) start(at.h0 + i, i);
  f2 u11[4], u21[4], u22[4], u12[4];     // sums over the heads of g1 x1 r, g2 x1 r, g2 x2 r, g1 x2 r
  if (DW) {
#pragma unroll
    for (int e = 0; e < 4; ++e) u11[e] = u21[e] = u22[e] = u12[e] = 0ull;
  }
  int slot = 0;
#pragma unroll 1
  for (int h = at.h0; h < at.h1; ++h) {
    ring.wait();
    f2 g1[4], g2[4], v1[4], v2[4];
    widen(ring.read(slot, 0), g1);
    widen(ring.read(slot, 1), g2);
    widen(ring.read(slot, 2), v1);
    widen(ring.read(slot, 3), v2);
    start(h + kBwdStages - 1, slot == 0 ? kBwdStages - 1 : slot - 1);
    slot = slot + 1 == kBwdStages ? 0 : slot + 1;
    f2 q0 = f2_mul(v1[0], v1[0]), q1 = f2_mul(v2[0], v2[0]);
#pragma unroll
    for (int e = 1; e < 4; ++e) {
      q0 = f2_fma(v1[e], v1[e], q0);
      q1 = f2_fma(v2[e], v2[e], q1);
    }
    const float rstd = rsqrtf(lanes_sum<D / 16>(f2_sum(f2_add(q0, q1)), at.mask) / D + p.eps);
    const f2 rs = f2_dup(rstd);
    f2 d0 = f2_dup(0.f), d1 = d0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (DW) {
        const f2 n1 = f2_mul(v1[e], rs), n2 = f2_mul(v2[e], rs);
        u11[e] = f2_fma(g1[e], n1, u11[e]);
        u22[e] = f2_fma(g2[e], n2, u22[e]);
        if (ROPE) {
          u21[e] = f2_fma(g2[e], n1, u21[e]);
          u12[e] = f2_fma(g1[e], n2, u12[e]);
        }
      }
      f2 w1 = f2_mul(g1[e], r.a1[e]), w2 = f2_mul(g2[e], r.a2[e]);
      if (ROPE) {
        w1 = f2_fma(g2[e], r.b2[e], w1);
        w2 = f2_fma(g1[e], r.b1[e], w2);
      }
      d0 = f2_fma(w1, v1[e], d0);
      d1 = f2_fma(w2, v2[e], d1);
      g1[e] = w1;
      g2[e] = w2;
    }
    const float mean = lanes_sum<D / 16>(f2_sum(f2_add(d0, d1)), at.mask) * rstd / D;   // mean(gw x r)
    const f2 nm = f2_dup(-mean * rstd);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      g1[e] = f2_mul(rs, f2_fma(v1[e], nm, g1[e]));
      g2[e] = f2_mul(rs, f2_fma(v2[e], nm, g2[e]));
    }
    stg_stream16(s.out + at.dense_at + h * D, narrow(g1));
    stg_stream16(s.out + at.dense_at + h * D + D / 2, narrow(g2));
  }
  if (!DW) return;
  if (s.partial == nullptr) return;      // the same for the whole CTA
  if (ROPE) {                            // rotate the token's sums
    f2 c1[4], c2[4], s1[4], s2[4];
    load8<false>(p.cos + at.pos * D, at.lane * 8, c1);
    load8<false>(p.cos + at.pos * D, D / 2 + at.lane * 8, c2);
    load8<false>(p.sin + at.pos * D, at.lane * 8, s1);
    load8<false>(p.sin + at.pos * D, D / 2 + at.lane * 8, s2);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u11[e] = f2_fma(c1[e], u11[e], f2_mul(s2[e], u21[e]));
      u22[e] = f2_fma(c2[e], u22[e], f2_mul(f2_mul(s1[e], f2_dup(-1.f)), u12[e]));
    }
  }
  // over the tokens of a warp, then over the warps in order
  constexpr int kLanes = D / 16, kWarps = THREADS / 32;
  __shared__ float sums[kWarps][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const f2 u = half ? u22[e] : u11[e];
      float lo = f2_lo(u), hi = f2_hi(u);
#pragma unroll
      for (int o = 16; o >= kLanes; o >>= 1) {
        lo += __shfl_xor_sync(0xffffffffu, lo, o);
        hi += __shfl_xor_sync(0xffffffffu, hi, o);
      }
      if (lane < kLanes) {
        sums[warp][half * (D / 2) + lane * 8 + 2 * e] = lo;
        sums[warp][half * (D / 2) + lane * 8 + 2 * e + 1] = hi;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < D) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) t += sums[w][threadIdx.x];
    s.partial[static_cast<int64_t>(at.cta) * D + threadIdx.x] = t;
  }
}

// dw[c] = sum over the CTAs of partial[cta][c]; blockIdx.x = group of 32 columns, blockIdx.y = side. Warp w adds its
// contiguous share in ascending order, then the 32 shares are added in ascending order.
template <int D>
__global__ void __launch_bounds__(1024) qk_norm_rope_dw_kernel(const __grid_constant__ PairParams p, int bf16) {
  after_previous();
  const Side& s = p.side[blockIdx.y];
  if (s.partial == nullptr) return;
  __shared__ float sums[32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  const int per = (s.ctas + 31) / 32, a = warp * per, b = min(s.ctas, a + per);
  const float* partial = after_previous(s.partial);
  float t = 0.f;
#pragma unroll 8
  for (int i = a; i < b; ++i) t += partial[static_cast<int64_t>(i) * D + c];
  sums[warp][lane] = t;
  __syncthreads();
  if (warp != 0) return;
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < 32; ++w) total += sums[w][lane];
  if (bf16) static_cast<__nv_bfloat16*>(s.dw)[c] = __float2bfloat16_rn(total);
  else static_cast<float*>(s.dw)[c] = total;
}

// Heads a token's lanes walk: all of them once the token blocks alone fill the GPU (four CTAs a SM), fewer, down to 2, below
// that: one token of 16 heads is then eight CTAs' work instead of one's.
void plan(Side& s, int tokens_per_cta) {
  const int64_t blocks = ceil_div(s.tokens, tokens_per_cta);
  int64_t groups = std::max<int64_t>(1, 4LL * sm_count() / std::max<int64_t>(1, blocks));
  groups = std::min<int64_t>(groups, std::max<int64_t>(1, s.heads / 2));
  s.heads_per_group = static_cast<int>(ceil_div(s.heads, groups));
  s.groups = static_cast<int>(ceil_div(s.heads, s.heads_per_group));
  s.ctas = static_cast<int>(blocks * s.groups);
}
int bwd_tokens_per_cta(int64_t head_dim, bool dw) { return static_cast<int>((dw ? kThreads / 2 : kThreads) / (head_dim / 16)); }

int check_sizes(const char* who, int64_t batch, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  ANIMA_REQUIRE(batch >= 0 && lq >= 0 && lk >= 0 && heads > 0 && kv_heads > 0, ANIMA_E_ARG, "%s: bad sizes", who);
  ANIMA_REQUIRE(head_dim == 64 || head_dim == 128, ANIMA_E_UNSUPPORTED, "%s: head_dim=%lld is not supported (64 or 128)", who,
                (long long)head_dim);
  ANIMA_REQUIRE(heads < (1ll << 16) && kv_heads < (1ll << 16) && batch < (1ll << 31) && lq < (1ll << 31) && lk < (1ll << 31) &&
                    batch * lq * heads < (1ll << 34) && batch * lk * kv_heads < (1ll << 34),
                ANIMA_E_TOO_LARGE, "%s: too many vectors", who);
  return ANIMA_OK;
}
int check_input(const char* who, const char* name, const void* x, const int64_t* s, const void* w, const void* out, bool empty) {
  ANIMA_REQUIRE(s && w, ANIMA_E_ARG, "%s: null pointer (%s)", who, name);
  ANIMA_REQUIRE(empty || (x && out), ANIMA_E_ARG, "%s: null pointer (%s)", who, name);
  ANIMA_REQUIRE(aligned16(x) && aligned16(out) && aligned16(w) && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0, ANIMA_E_ALIGN,
                "%s: %s and its weight must be 16-byte aligned, strides multiples of 8 elements", who, name);
  return ANIMA_OK;
}
int check_tables(const char* who, const float* cos_tab, const float* sin_tab, int64_t table_samples, int64_t batch, int64_t lq,
                 int64_t lk) {
  ANIMA_REQUIRE((cos_tab == nullptr) == (sin_tab == nullptr), ANIMA_E_ARG, "%s: give both tables or neither", who);
  if (!cos_tab) return ANIMA_OK;
  ANIMA_REQUIRE(lq == lk, ANIMA_E_SHAPE, "%s: one table for %lld queries and %lld keys", who, (long long)lq, (long long)lk);
  ANIMA_REQUIRE(table_samples == 1 || table_samples == batch, ANIMA_E_SHAPE, "%s: tables of %lld samples for a batch of %lld", who,
                (long long)table_samples, (long long)batch);
  ANIMA_REQUIRE(aligned16(cos_tab) && aligned16(sin_tab), ANIMA_E_ALIGN, "%s: tables must be 16-byte aligned", who);
  return ANIMA_OK;
}
Side side_of(const void* x, const int64_t* strides, const void* w, void* out, int64_t batch, int64_t len, int64_t heads) {
  Side s = {};
  s.x = static_cast<const __nv_bfloat16*>(x);
  s.out = static_cast<__nv_bfloat16*>(out);
  s.w = w;
  s.sb = strides[0];
  s.sl = strides[1];
  s.sh = strides[2];
  s.len = std::max<int64_t>(1, len);
  s.tokens = batch * len;
  s.heads = static_cast<int>(heads);
  return s;
}

// f(kernel) for the kernel of this call
template <int D, class F>
void pick_fwd(bool rope, bool wbf16, F&& f) {
  if (rope) wbf16 ? f(qk_norm_rope_fwd_kernel<D, true, true>) : f(qk_norm_rope_fwd_kernel<D, true, false>);
  else wbf16 ? f(qk_norm_rope_fwd_kernel<D, false, true>) : f(qk_norm_rope_fwd_kernel<D, false, false>);
}
template <int D, bool DW, class F>
void pick_bwd(bool rope, bool wbf16, F&& f) {
  if (rope) wbf16 ? f(qk_norm_rope_bwd_kernel<D, true, true, DW>) : f(qk_norm_rope_bwd_kernel<D, true, false, DW>);
  else wbf16 ? f(qk_norm_rope_bwd_kernel<D, false, true, DW>) : f(qk_norm_rope_bwd_kernel<D, false, false, DW>);
}
template <int D, class F>
void pick_bwd(bool rope, bool wbf16, bool dw, F&& f) {
  dw ? pick_bwd<D, true>(rope, wbf16, f) : pick_bwd<D, false>(rope, wbf16, f);
}

}  // namespace
}  // namespace anima

using namespace anima;

extern "C" int anima_qk_norm_rope_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                      const void* q_weight, const void* k_weight, int weights_are_bf16, const float* cos_tab,
                                      const float* sin_tab, int64_t table_samples, float eps, int64_t batch, int64_t lq,
                                      int64_t lk, int64_t heads, int64_t kv_heads, int64_t head_dim, void* q_out, void* k_out,
                                      void* stream) {
  const char* who = "qk_norm_rope_fwd";
  if (int rc = check_sizes(who, batch, lq, lk, heads, kv_heads, head_dim)) return rc;
  if (int rc = check_input(who, "q", q, q_strides, q_weight, q_out, batch * lq == 0)) return rc;
  if (int rc = check_input(who, "k", k, k_strides, k_weight, k_out, batch * lk == 0)) return rc;
  if (int rc = check_tables(who, cos_tab, sin_tab, table_samples, batch, lq, lk)) return rc;
  PairParams p = {};
  p.side[0] = side_of(q, q_strides, q_weight, q_out, batch, lq, heads);
  p.side[1] = side_of(k, k_strides, k_weight, k_out, batch, lk, kv_heads);
  for (Side& s : p.side) plan(s, static_cast<int>(kThreads / (head_dim / 16)));
  p.cos = cos_tab;
  p.sin = sin_tab;
  p.table_step = table_samples == 1 ? 0 : lq;
  p.eps = eps;
  const int64_t ctas = static_cast<int64_t>(p.side[0].ctas) + p.side[1].ctas;
  if (ctas == 0) return ANIMA_OK;
  constexpr int kSmem = kFwdStages * 2 * kThreads * 16;
  auto go = [&](auto kernel) {
    launch_after(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), kSmem, static_cast<cudaStream_t>(stream), p);
  };
  head_dim == 64 ? pick_fwd<64>(cos_tab != nullptr, weights_are_bf16 != 0, go) : pick_fwd<128>(cos_tab != nullptr, weights_are_bf16 != 0, go);
  ANIMA_CHECK_LAUNCH(who);
  return ANIMA_OK;
}

extern "C" int64_t anima_qk_norm_rope_bwd_workspace_bytes(int64_t batch, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads,
                                                          int64_t head_dim) {
  if (int rc = check_sizes("qk_norm_rope_bwd", batch, lq, lk, heads, kv_heads, head_dim)) return rc;
  Side q = {}, k = {};
  q.tokens = batch * lq; q.heads = static_cast<int>(heads);
  k.tokens = batch * lk; k.heads = static_cast<int>(kv_heads);
  plan(q, bwd_tokens_per_cta(head_dim, true));
  plan(k, bwd_tokens_per_cta(head_dim, true));
  return (static_cast<int64_t>(q.ctas) + k.ctas) * head_dim * 4;
}

extern "C" int anima_qk_norm_rope_bwd(const void* dq_out, const void* dk_out, const void* q, const int64_t* q_strides,
                                      const void* k, const int64_t* k_strides, const void* q_weight, const void* k_weight,
                                      int weights_are_bf16, const float* cos_tab, const float* sin_tab, int64_t table_samples,
                                      float eps, int64_t batch, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads,
                                      int64_t head_dim, void* dq, void* dk, void* dq_weight, void* dk_weight, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const char* who = "qk_norm_rope_bwd";
  if (int rc = check_sizes(who, batch, lq, lk, heads, kv_heads, head_dim)) return rc;
  if (int rc = check_input(who, "q", q, q_strides, q_weight, dq, batch * lq == 0)) return rc;
  if (int rc = check_input(who, "k", k, k_strides, k_weight, dk, batch * lk == 0)) return rc;
  if (int rc = check_tables(who, cos_tab, sin_tab, table_samples, batch, lq, lk)) return rc;
  ANIMA_REQUIRE((batch * lq == 0 || dq_out) && (batch * lk == 0 || dk_out), ANIMA_E_ARG, "%s: null pointer", who);
  ANIMA_REQUIRE(aligned16(dq_out) && aligned16(dk_out), ANIMA_E_ALIGN, "%s: gradients must be 16-byte aligned", who);
  const bool dw = dq_weight || dk_weight;
  const int64_t need = dw ? anima_qk_norm_rope_bwd_workspace_bytes(batch, lq, lk, heads, kv_heads, head_dim) : 0;
  ANIMA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), ANIMA_E_WORKSPACE, "%s: workspace of %lld bytes, %lld needed",
                who, (long long)workspace_bytes, (long long)need);
  PairParams p = {};
  p.side[0] = side_of(q, q_strides, q_weight, dq, batch, lq, heads);
  p.side[1] = side_of(k, k_strides, k_weight, dk, batch, lk, kv_heads);
  p.side[0].g = static_cast<const __nv_bfloat16*>(dq_out);
  p.side[1].g = static_cast<const __nv_bfloat16*>(dk_out);
  p.side[0].dw = dq_weight;
  p.side[1].dw = dk_weight;
  float* partial = static_cast<float*>(workspace);
  for (Side& s : p.side) {
    plan(s, bwd_tokens_per_cta(head_dim, dw));
    // a side without tokens has no partials: its sum, over none, is still to be written
    if (s.dw) s.partial = need ? partial : static_cast<float*>(s.dw);
    partial += static_cast<int64_t>(s.ctas) * head_dim;
  }
  p.cos = cos_tab;
  p.sin = sin_tab;
  p.table_step = table_samples == 1 ? 0 : lq;
  p.eps = eps;
  const int64_t ctas = static_cast<int64_t>(p.side[0].ctas) + p.side[1].ctas;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool rope = cos_tab != nullptr, wb = weights_are_bf16 != 0;
  if (ctas) {
    const int threads = dw ? kThreads / 2 : kThreads;
    constexpr int kSmem = kBwdStages * 4 * kThreads * 16;
    static PerDeviceOnce once;
    const cudaError_t rc = per_device_once(once, [] {
      cudaError_t e = cudaSuccess;
      auto opt_in = [&](auto kernel) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
      };
      for (bool r : {false, true})
        for (bool w : {false, true}) {
          pick_bwd<64>(r, w, false, opt_in);
          pick_bwd<128>(r, w, false, opt_in);
        }
      return e;
    });
    ANIMA_REQUIRE(rc == cudaSuccess, ANIMA_E_CUDA, "%s: cannot reserve %d bytes of shared memory: %s", who, kSmem,
                  cudaGetErrorString(rc));
    auto go = [&](auto kernel) {
      launch_after(kernel, dim3(static_cast<unsigned>(ctas)), dim3(threads), static_cast<size_t>(kSmem / kThreads * threads), st, p);
    };
    head_dim == 64 ? pick_bwd<64>(rope, wb, dw, go) : pick_bwd<128>(rope, wb, dw, go);
    ANIMA_CHECK_LAUNCH(who);
  }
  if (dw) {
    const dim3 grid(static_cast<unsigned>(head_dim / 32), 2);
    if (head_dim == 64) launch_after(qk_norm_rope_dw_kernel<64>, grid, dim3(1024), 0, st, p, weights_are_bf16);
    else launch_after(qk_norm_rope_dw_kernel<128>, grid, dim3(1024), 0, st, p, weights_are_bf16);
    ANIMA_CHECK_LAUNCH(who);
  }
  return ANIMA_OK;
}
