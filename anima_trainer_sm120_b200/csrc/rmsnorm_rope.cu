// Per-head RMSNorm with optional rotary embedding, forward and backward, for the q / k
// projections of the attention layers (head width 128, bf16).
//
// In anima-trainer these two steps are third-party kernels (Liger RMSNorm, liger_patch.py:31-47, and
// Transformer Engine's fused RoPE, rope_patch.py:28-56); the stand-in DiT of this package would
// otherwise run them as ~10 eager elementwise launches per call. HBM-bound: 4 B/elem forward
// (+ 4 B per vector for rstd), 6 B/elem backward.
//   n   = x * rsqrt(mean(x^2) + eps) * w
//   out = n * cos + rotate_half(n) * sin   (cos / sin: fp32 tables [seq_len, 128], L2-resident)
//           rotate_half(n)[i] = -n[i+64] (i < 64), n[i-64] (i >= 64)
// The norm weight is treated as frozen (no weight gradient), which is the LoKr training setting.
#include "common.cuh"
#include "head_vectors.cuh"

namespace anima {
namespace {

constexpr int kHeadDim = 128;
constexpr int kThreads = 256;
constexpr int kLanesPerToken = 8;                        // 8 lanes x (8 + 8) elements = one 128-wide head vector
constexpr int kTokensPerCta = kThreads / kLanesPerToken;

constexpr int kFwdStages = 6, kBwdStages = 4;
using namespace headvec;   // the layout of a token in its lanes

// blockIdx.y = group of heads (a grid of token blocks alone would leave SMs idle on short sequences)
template <bool ROPE, bool WBF16>
__global__ void __launch_bounds__(kThreads, 2)
rmsnorm_rope_fwd_kernel(const __nv_bfloat16* __restrict__ x, const void* __restrict__ w, const float* __restrict__ cos_tab,
                        const float* __restrict__ sin_tab, float eps, int64_t tokens, int heads, int heads_per_group,
                        int64_t seq_len, __nv_bfloat16* __restrict__ out, float* __restrict__ rstd_out,
                        uint4* __restrict__ w_copy) {
  after_previous();
  w = after_previous(w);
  if (w_copy != nullptr && blockIdx.x + blockIdx.y == 0 && threadIdx.x < kHeadDim * (WBF16 ? 2 : 4) / 16)
    w_copy[threadIdx.x] = static_cast<const uint4*>(w)[threadIdx.x];
  cos_tab = after_previous(cos_tab);
  sin_tab = after_previous(sin_tab);
  const int l = threadIdx.x & (kLanesPerToken - 1);
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kTokensPerCta + threadIdx.x / kLanesPerToken;
  if (token >= tokens) return;   // the eight lanes of a token leave together; shuffles below stay inside them
  const unsigned mask = 0xffu << (threadIdx.x & 24);
  const int h0 = blockIdx.y * heads_per_group, h1 = min(heads, h0 + heads_per_group);
  Rotation r;
  load_rotation<kHeadDim, ROPE, WBF16>(r, w, cos_tab, sin_tab, ROPE ? token % seq_len : 0, l);
  const int64_t base = token * heads * kHeadDim + l * 8;
  extern __shared__ uint4 ring_smem[];
  const Ring<2, kFwdStages, kThreads> ring(ring_smem);
  auto start = [&](int h, int slot) {
    if (h < h1) {
      ring.copy(slot, 0, x + base + h * kHeadDim);
      ring.copy(slot, 1, x + base + h * kHeadDim + 64);
    }
    ring.commit();
  };
#pragma unroll
  for (int i = 0; i < kFwdStages - 1; ++i) start(h0 + i, i);
  int slot = 0;
#pragma unroll 1
  for (int h = h0; h < h1; ++h) {
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
    const float rstd = rsqrtf(lanes_sum<kLanesPerToken>(f2_sum(f2_add(q0, q1)), mask) / kHeadDim + eps);
    const f2 rs = f2_dup(rstd);
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
    stg_stream16(out + base + h * kHeadDim, narrow(v1));
    stg_stream16(out + base + h * kHeadDim + 64, narrow(v2));
    if (l == 0) rstd_out[token * heads + h] = rstd;
  }
}

template <bool ROPE, bool WBF16>
__global__ void __launch_bounds__(kThreads, 2)
rmsnorm_rope_bwd_kernel(const __nv_bfloat16* __restrict__ dout, const __nv_bfloat16* __restrict__ x,
                        const void* __restrict__ w, const float* __restrict__ cos_tab, const float* __restrict__ sin_tab,
                        const float* __restrict__ rstd_in, int64_t tokens, int heads, int heads_per_group, int64_t seq_len,
                        __nv_bfloat16* __restrict__ dx) {
  after_previous();
  w = after_previous(w);
  cos_tab = after_previous(cos_tab);
  sin_tab = after_previous(sin_tab);
  const int l = threadIdx.x & (kLanesPerToken - 1);
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kTokensPerCta + threadIdx.x / kLanesPerToken;
  if (token >= tokens) return;
  const unsigned mask = 0xffu << (threadIdx.x & 24);
  const int h0 = blockIdx.y * heads_per_group, h1 = min(heads, h0 + heads_per_group);
  Rotation r;
  load_rotation<kHeadDim, ROPE, WBF16>(r, w, cos_tab, sin_tab, ROPE ? token % seq_len : 0, l);
  const int64_t base = token * heads * kHeadDim + l * 8;
  extern __shared__ uint4 ring_smem[];
  const Ring<4, kBwdStages, kThreads> ring(ring_smem);
  auto start = [&](int h, int slot) {
    if (h < h1) {
      const int64_t at = base + h * kHeadDim;
      ring.copy(slot, 0, dout + at);
      ring.copy(slot, 1, dout + at + 64);
      ring.copy(slot, 2, x + at);
      ring.copy(slot, 3, x + at + 64);
    }
    ring.commit();
  };
#pragma unroll
  for (int i = 0; i < kBwdStages - 1; ++i) start(h0 + i, i);
  rstd_in = after_previous(rstd_in);
  float rstd_next = rstd_in[token * heads + h0];
  int slot = 0;
#pragma unroll 1
  for (int h = h0; h < h1; ++h) {
    const int64_t at = base + h * kHeadDim;
    const float rstd = rstd_next;
    if (h + 1 < h1) rstd_next = rstd_in[token * heads + h + 1];
    ring.wait();
    f2 g1[4], g2[4], v1[4], v2[4];
    widen(ring.read(slot, 0), g1);
    widen(ring.read(slot, 1), g2);
    widen(ring.read(slot, 2), v1);
    widen(ring.read(slot, 3), v2);
    start(h + kBwdStages - 1, slot == 0 ? kBwdStages - 1 : slot - 1);
    slot = slot + 1 == kBwdStages ? 0 : slot + 1;
    // dx = rstd * (gw - xhat * mean(gw * xhat)), xhat = x * rstd
    f2 d0 = f2_dup(0.f), d1 = d0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
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
    const float dot = lanes_sum<kLanesPerToken>(f2_sum(f2_add(d0, d1)), mask) * rstd / kHeadDim;   // mean(gw * xhat)
    const f2 nm = f2_dup(-dot * rstd), rs = f2_dup(rstd);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      g1[e] = f2_mul(rs, f2_fma(v1[e], nm, g1[e]));
      g2[e] = f2_mul(rs, f2_fma(v2[e], nm, g2[e]));
    }
    stg_stream16(dx + at, narrow(g1));
    stg_stream16(dx + at + 64, narrow(g2));
  }
}

// Heads one CTA walks: all of them once the token blocks alone fill the GPU, fewer (down to 2) below that.
int heads_per_group(int64_t token_blocks, int64_t heads) {
  int64_t groups = std::max<int64_t>(1, 4LL * sm_count() / std::max<int64_t>(1, token_blocks));
  groups = std::min<int64_t>(groups, std::max<int64_t>(1, heads / 2));
  return static_cast<int>(ceil_div(heads, groups));
}

int check(const char* who, int64_t tokens, int64_t heads, int64_t head_dim, int64_t seq_len, const void* cos_tab, const void* sin_tab) {
  ANIMA_REQUIRE(tokens >= 0 && heads > 0, ANIMA_E_ARG, "%s: bad sizes", who);
  ANIMA_REQUIRE(head_dim == kHeadDim, ANIMA_E_UNSUPPORTED, "%s: head_dim=%lld is not supported (only %d)", who,
                (long long)head_dim, kHeadDim);
  ANIMA_REQUIRE(heads < (1ll << 31) && tokens * heads < (1ll << 40), ANIMA_E_TOO_LARGE, "%s: too many vectors", who);
  ANIMA_REQUIRE((cos_tab == nullptr) == (sin_tab == nullptr), ANIMA_E_ARG, "%s: give both tables or neither", who);
  ANIMA_REQUIRE(!cos_tab || (seq_len > 0 && tokens % seq_len == 0), ANIMA_E_SHAPE,
                "%s: tokens=%lld is not a multiple of seq_len=%lld", who, (long long)tokens, (long long)seq_len);
  return ANIMA_OK;
}

}  // namespace
}  // namespace anima

using namespace anima;

extern "C" int anima_rmsnorm_rope_fwd_keep(const void* x, const void* weight, int weight_is_bf16, const float* cos_tab,
                                           const float* sin_tab, float eps, int64_t tokens, int64_t heads, int64_t head_dim,
                                           int64_t seq_len, void* out, float* rstd, void* weight_copy, void* stream) {
  ANIMA_REQUIRE(x && weight && out && rstd, ANIMA_E_ARG, "rmsnorm_rope_fwd: null pointer");
  if (int rc = check("rmsnorm_rope_fwd", tokens, heads, head_dim, seq_len, cos_tab, sin_tab)) return rc;
  ANIMA_REQUIRE(aligned16(x) && aligned16(out) && aligned16(weight) && aligned16(weight_copy) && (!cos_tab || (aligned16(cos_tab) && aligned16(sin_tab))), ANIMA_E_ALIGN,
                "rmsnorm_rope_fwd: tensors must be 16-byte aligned");
  if (tokens * heads == 0) return ANIMA_OK;
  const int64_t blocks = ceil_div(tokens, kTokensPerCta);
  const int hpg = heads_per_group(blocks, heads);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(ceil_div(heads, hpg)));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto* xp = static_cast<const __nv_bfloat16*>(x);
  auto* op = static_cast<__nv_bfloat16*>(out);
  constexpr int kSmem = kFwdStages * 2 * kThreads * 16;
  auto go = [&](auto kernel) { launch_after(kernel, grid, kThreads, kSmem, s, xp, weight, cos_tab, sin_tab, eps, tokens, (int)heads, hpg, seq_len, op, rstd, static_cast<uint4*>(weight_copy)); };
  if (cos_tab) weight_is_bf16 ? go(rmsnorm_rope_fwd_kernel<true, true>) : go(rmsnorm_rope_fwd_kernel<true, false>);
  else weight_is_bf16 ? go(rmsnorm_rope_fwd_kernel<false, true>) : go(rmsnorm_rope_fwd_kernel<false, false>);
  ANIMA_CHECK_LAUNCH("rmsnorm_rope_fwd");
  return ANIMA_OK;
}

extern "C" int anima_rmsnorm_rope_fwd_ex(const void* x, const void* weight, int weight_is_bf16, const float* cos_tab,
                                         const float* sin_tab, float eps, int64_t tokens, int64_t heads, int64_t head_dim,
                                         int64_t seq_len, void* out, float* rstd, void* stream) {
  return anima_rmsnorm_rope_fwd_keep(x, weight, weight_is_bf16, cos_tab, sin_tab, eps, tokens, heads, head_dim, seq_len, out,
                                     rstd, nullptr, stream);
}

extern "C" int anima_rmsnorm_rope_bwd_ex(const void* dout, const void* x, const void* weight, int weight_is_bf16,
                                         const float* cos_tab, const float* sin_tab, const float* rstd, int64_t tokens,
                                         int64_t heads, int64_t head_dim, int64_t seq_len, void* dx, void* stream) {
  ANIMA_REQUIRE(dout && x && weight && rstd && dx, ANIMA_E_ARG, "rmsnorm_rope_bwd: null pointer");
  if (int rc = check("rmsnorm_rope_bwd", tokens, heads, head_dim, seq_len, cos_tab, sin_tab)) return rc;
  ANIMA_REQUIRE(aligned16(dout) && aligned16(x) && aligned16(dx) && aligned16(weight) && (!cos_tab || (aligned16(cos_tab) && aligned16(sin_tab))),
                ANIMA_E_ALIGN, "rmsnorm_rope_bwd: tensors must be 16-byte aligned");
  if (tokens * heads == 0) return ANIMA_OK;
  const int64_t blocks = ceil_div(tokens, kTokensPerCta);
  const int hpg = heads_per_group(blocks, heads);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(ceil_div(heads, hpg)));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto* gp = static_cast<const __nv_bfloat16*>(dout);
  const auto* xp = static_cast<const __nv_bfloat16*>(x);
  auto* dp = static_cast<__nv_bfloat16*>(dx);
  constexpr int kSmem = kBwdStages * 4 * kThreads * 16;
  static PerDeviceOnce once;
  const cudaError_t rc = per_device_once(once, [] {
    for (auto k : {rmsnorm_rope_bwd_kernel<true, true>, rmsnorm_rope_bwd_kernel<true, false>, rmsnorm_rope_bwd_kernel<false, true>,
                   rmsnorm_rope_bwd_kernel<false, false>})
      if (cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem)) return e;
    return cudaSuccess;
  });
  ANIMA_REQUIRE(rc == cudaSuccess, ANIMA_E_CUDA, "rmsnorm_rope_bwd: cannot reserve %d bytes of shared memory: %s", kSmem,
                cudaGetErrorString(rc));
  auto go = [&](auto kernel) { launch_after(kernel, grid, kThreads, kSmem, s, gp, xp, weight, cos_tab, sin_tab, rstd, tokens, (int)heads, hpg, seq_len, dp); };
  if (cos_tab) weight_is_bf16 ? go(rmsnorm_rope_bwd_kernel<true, true>) : go(rmsnorm_rope_bwd_kernel<true, false>);
  else weight_is_bf16 ? go(rmsnorm_rope_bwd_kernel<false, true>) : go(rmsnorm_rope_bwd_kernel<false, false>);
  ANIMA_CHECK_LAUNCH("rmsnorm_rope_bwd");
  return ANIMA_OK;
}

extern "C" int anima_rmsnorm_rope_fwd(const void* x, const float* weight, const float* cos_tab, const float* sin_tab, float eps,
                                      int64_t tokens, int64_t heads, int64_t head_dim, int64_t seq_len,
                                      void* out, float* rstd, void* stream) {
  return anima_rmsnorm_rope_fwd_ex(x, weight, 0, cos_tab, sin_tab, eps, tokens, heads, head_dim, seq_len, out, rstd, stream);
}

extern "C" int anima_rmsnorm_rope_bwd(const void* dout, const void* x, const float* weight, const float* cos_tab,
                                      const float* sin_tab, const float* rstd, int64_t tokens, int64_t heads, int64_t head_dim,
                                      int64_t seq_len, void* dx, void* stream) {
  return anima_rmsnorm_rope_bwd_ex(dout, x, weight, 0, cos_tab, sin_tab, rstd, tokens, heads, head_dim, seq_len, dx, stream);
}
