// Attention, forward (formulas: attention_common.cuh): one pass over the keys with each row's running maximum and sum.
//
// A CTA owns a tile of 128 queries of one head and walks the keys, 64 at a time. Per step
//   S = Q K^T     tcgen05, both operands in shared memory, fp32 scores in tensor memory (lane = query, column = key);
//   softmax       one warpgroup, one thread a row: 64 scores into registers, row maximum without shuffles,
//                 p = 2^(s scale log2 e - m), rounded to bf16 for the second product (the sum takes the unrounded values), written
//                 over the scores;
//   O += P V      tcgen05 with P read from tensor memory, V as it lies (keys along rows: the MN-major form), fp32.
// The scores have two buffers: S of the step after next is issued behind O += P V, which frees its buffer, so the warpgroup
// finds its next scores ready. One warp issues the products, one feeds K and V through a ring of TMA boxes of 64 keys.
// Two CTAs share an SM (half of its tensor memory and shared memory each): the maxima, sums, loads and waits of one fill the
// special-function unit's and the tensor cores' pauses of the other, and so do a CTA's set-up, first loads and way out, 6000
// cycles or four steps. One CTA with two query tiles reads K and V half as often, but was slower nearly everywhere
// ([8, 4096 x 512, 16, 128] 224 against 206 us, [8, 4096 x 1024] 275 / 261, [2, 4096 x 4096] 245 / 240, [8, 4096 x 4096] 869 / 884,
// [4, 4096 x 4096, 16, 64] 396 / 363).
// O leaves through the query tile's shared memory and TMA stores (each thread holds a row: its own 16-byte stores took 3000
// cycles a tile).
// The running maximum of a row is only raised once a score exceeds it by 2^8: until then p is at most 256, which costs neither
// bf16 (relative) nor the fp32 sums anything, and O, which lies in tensor memory, need not be rescaled.
// Few rows (one token, a short text) leave SMs idle: the keys are then cut into ranges, whose normalised fp32 outputs and
// log-sums a second kernel joins in order. One query token per sample: the heads that share a key head become the rows of a
// tile, so that each key is read once.
// Bound: 4 D flop a (query, key) pair on the tensor cores and one exponential, of which an SM makes 16 a cycle: a tile pair
// of D = 128 takes 1024 cycles of either.
#include "attention_common.cuh"

namespace anima {
namespace attn {
namespace {

constexpr int kStep = 64;                // keys of a step
constexpr float kMaxSlack = 8.f;         // log2 of how far a score may exceed the maximum in use
constexpr int kPoly = 1;                 // of four pairs of exponentials, those made on the multiply-add pipes

template <int D>
struct FwdCfg {
  static constexpr int kMmaWarp = 4, kTmaWarp = 5, kThreads = 192;
  static constexpr uint32_t kBytes = tile_bytes<D>(), kStepBytes = kBytes / 2;
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kBars = 2 * kStages + 7;
  static constexpr int kSmem = static_cast<int>(kBytes + kStages * kStepBytes) + kBars * 8 + 24;
  static_assert(2 * (kSmem + 1024) <= 228 * 1024, "shared memory of two CTAs");
  // tensor-memory columns: scores of buffer x at 64 x
  static constexpr uint32_t kS = 0, kO = kTile, kCols = 256;
};

struct FwdParams {
  Sizes z;
  float c;                               // scale * log2 e
  __nv_bfloat16* out;
  Strided so;                            // of out
  float* lse;                            // [batch, heads, lq] or null
  int q_blocks, splits, tiles_per_split;
  float* part_o;                         // [split][batch, heads, lq][D], null: no split
  float* part_lse;                       // [split][batch, heads, lq], base 2
  int64_t rows;                          // batch * heads * lq
  int32_t* status;
};

// grid (q_blocks * splits, heads, batch)
template <int D>
__global__ void __launch_bounds__(FwdCfg<D>::kThreads, 2)
attention_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o,
                     const __grid_constant__ FwdParams p) {
  using C = FwdCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t q_smem = base;
  auto kv_smem = [&](int s) { return base + C::kBytes + s * C::kStepBytes; };
  const uint32_t bars = base + C::kBytes + C::kStages * C::kStepBytes;
  auto full = [&](int s) { return bars + 8 * s; };
  auto empty = [&](int s) { return bars + 8 * (C::kStages + s); };
  const uint32_t q_full = bars + 8 * (2 * C::kStages);
  auto s_full = [&](int x) { return q_full + 8 * (1 + x); };
  auto o_done = [&](int x) { return q_full + 8 * (3 + x); };
  auto p_full = [&](int x) { return q_full + 8 * (5 + x); };
  volatile int& abort_flag = *reinterpret_cast<volatile int*>(smem + (bars - base) + C::kBars * 8 + 8);
  uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(smem + (bars - base) + C::kBars * 8 + 16);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < C::kBars; ++i) mbar_init(bars + 8 * i, i >= 2 * C::kStages + 5 ? 4 : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_o) : "memory");
  }
  if (warp == C::kMmaWarp) tc_alloc(smem_u32(&tmem_slot), C::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  after_previous();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);

  const Sizes& z = p.z;
  const int split = blockIdx.x / p.q_blocks, qb = blockIdx.x - split * p.q_blocks, h = blockIdx.y, b = blockIdx.z;
  const int hk = h / z.group;
  const int q0 = qb * kTile;
  const int n = keys_of(z, b);
  // this CTA's keys start at k0, in `count` steps
  const int j0 = split * p.tiles_per_split, k0 = j0 * kTile;
  const int lim_tile = min(key_limit(z, n, min(z.lq, q0 + kTile) - 1), k0 + p.tiles_per_split * kTile);
  const int count = max(0, lim_tile - k0 + kStep - 1) / kStep;
  // the order of the ring: K0, K1, V0, K2, V1, ...
  auto k_at = [](int u) { return u == 0 ? 0 : 2 * u - 1; };
  auto v_at = [&](int u) { return 2 * u + (u + 1 < count ? 2 : 1); };

  if (warp == C::kTmaWarp) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0 && count > 0) {
      mbar_expect_tx(q_full, C::kBytes);
      load_rows<D, kTile>(q_smem, &map_q, q_full, q0, h, b);
      for (int i = 0; i < 2 * count; ++i) {
        const int s = i % C::kStages;
        const bool value = i == 2 * count - 1 || (i > 0 && !(i & 1));
        const int u = value ? (i - 1) / 2 : (i + 1) / 2;
        if (!mbar_wait(empty(s), ((i / C::kStages) & 1) ^ 1, &abort_flag)) break;
        mbar_expect_tx(full(s), C::kStepBytes);
        load_rows<D, kStep>(kv_smem(s), value ? &map_v : &map_k, full(s), k0 + u * kStep, hk, b);
      }
    }
  } else if (warp == C::kMmaWarp) {
    // ------------------------------------------------------------ MMA issuer
    const uint64_t q_desc = tc_desc_sw128(q_smem);
    auto arrived = [&](int i) { return warp_wait(full(i % C::kStages), (i / C::kStages) & 1, &abort_flag); };
    auto scores = [&](int u) {                 // S of step u
      const int s = k_at(u) % C::kStages;
      const uint64_t k = tc_desc_sw128(kv_smem(s));
#pragma unroll
      for (int i = 0; i < D / 16; ++i)         // 16 bytes a unit
        tc_mma_ss(tmem + C::kS + (u & 1) * kStep, q_desc + (i >> 2) * (kTile * 128 / 16) + (i & 3) * 2,
                  k + (i >> 2) * (kStep * 128 / 16) + (i & 3) * 2, tc_idesc_bf16(kTile, kStep), i > 0);
      tc_commit_warp(s_full(u & 1));
      tc_commit_warp(empty(s));
    };
    bool ok = count > 0 && warp_wait(q_full, 0, &abort_flag);
    for (int u = 0; u < min(2, count) && ok; ++u) {
      ok = arrived(k_at(u));
      tc_fence_after();
      if (ok) scores(u);
    }
    for (int u = 0; u < count && ok; ++u) {
      const int vs = v_at(u) % C::kStages;
      const bool next = u + 2 < count;
      // keys of the step that exist; the product over the others is left out, up to the next multiple of 16
      const int keys = min(kStep, n - k0 - u * kStep), steps = (keys + 15) / 16;
      ok = arrived(v_at(u)) && (!next || arrived(k_at(u + 2)));
      if (!ok) break;
      if (keys & 15) zero_rows<D>(kv_smem(vs), kStep * 128, keys, steps * 16);
      const uint64_t v = tc_desc_sw128(kv_smem(vs), kStep * 128);
      ok = warp_wait(p_full(u & 1), (u >> 1) & 1, &abort_flag);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < kStep / 16; ++i)
        if (i < steps)
          tc_mma_ts(tmem + C::kO, tmem + C::kS + (u & 1) * kStep + i * 8, v + i * (16 * 128 / 16), tc_idesc_bf16(kTile, D, true), u > 0 || i > 0);
      tc_commit_warp(o_done(u & 1));
      tc_commit_warp(empty(vs));
      if (next) scores(u + 2);
    }
  } else {
    // ------------------------------------------------------------ softmax: thread = row
    const int row = q0 + threadIdx.x;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t s_at = tmem + lanes + C::kS, o_at = tmem + lanes + C::kO;
    const int lim = key_limit(z, n, row);
    // the warp's first row sees the fewest keys: steps that end before that need no mask
    const int lim_all = __shfl_sync(0xffffffffu, lim, 0);
    float m = -INFINITY, used = 0.f;     // maximum in use (raw scores), m * c (0 while there is none)
    f2 sum[4] = {0ull, 0ull, 0ull, 0ull};
    bool ok = true;
    // 32 rows behind the last query (a few queries against many keys): nothing is made of their scores, and what lies in their
    // place in tensor memory only reaches rows of O that nobody stores
    const bool idle = row - lane >= z.lq;
    for (int u = 0; u < count; ++u) {
      const uint32_t at = s_at + (u & 1) * kStep;
      ok = warp_wait(s_full(u & 1), (u >> 1) & 1, &abort_flag);
      if (!ok) break;
      if (idle) {
        if (lane == 0) mbar_arrive(p_full(u & 1));
        continue;
      }
      tc_fence_after();
      uint32_t s[2][32];
      tc_ld32(at, s[0]);
      tc_ld32(at + 32, s[1]);
      tc_wait_ld();
      const int key = k0 + u * kStep;
      if (key + kStep > lim_all) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (key + i * 32 + e >= lim) s[i][e] = 0xff800000u;
      }
      float mx[4] = {m, m, m, m};
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 32; e += 2) mx[(e >> 1) & 3] = max3(mx[(e >> 1) & 3], __uint_as_float(s[i][e]), __uint_as_float(s[i][e + 1]));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const bool grow = (top - m) * p.c > kMaxSlack;
      if (__any_sync(0xffffffffu, grow)) {
        const float f = grow ? exp2_approx((m - top) * p.c) : 1.f;      // 0 where there was no maximum yet
        if (grow) {
          m = top;
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] = f2_mul(sum[i], f2_dup(f));
          used = m * p.c;
        }
        if (u > 0) {                       // the product of the step before is the last one under way: S(u) came behind the others
          ok = warp_wait(o_done((u - 1) & 1), ((u - 1) >> 1) & 1, &abort_flag);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int i = 0; i < D / 32; ++i) {
            uint32_t o[32];
            tc_ld32(o_at + i * 32, o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tc_st32(o_at + i * 32, o);
          }
        }
      }
      const f2 c2 = f2_dup(p.c), u2 = f2_dup(-used);
      f2 y[32];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const f2 x = f2_fma(f2_make(__uint_as_float(s[i][2 * e]), __uint_as_float(s[i][2 * e + 1])), c2, u2);
          y[i * 16 + e] = (e & 3) < kPoly ? exp2_poly(x) : exp2_pair(x);
          w[e] = bf16_of_f2(y[i * 16 + e]);
        }
        tc_st16(at + i * 16, w);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full(u & 1));
      // the row's sum, behind what the tensor cores wait for
#pragma unroll
      for (int e = 0; e < 32; ++e) sum[e & 3] = f2_add(sum[e & 3], y[e]);
    }
    // ------------------------------------------------------------ epilogue
    if (ok && count > 0) {
      ok = warp_wait(o_done((count - 1) & 1), ((count - 1) >> 1) & 1, &abort_flag);
      tc_fence_after();
    }
    const float l = f2_sum(f2_add(f2_add(sum[0], sum[1]), f2_add(sum[2], sum[3])));
    const float inv = l == 0.f ? 0.f : 1.f / l;        // a row without keys has no sum
    const bool live = row < z.lq && ok;
    const int64_t at = (static_cast<int64_t>(b) * z.heads + h) * z.lq + row;
    const float total = l == 0.f ? -INFINITY : used + log2_approx(l);      // base 2
    if (p.part_o != nullptr) {
      if (live) p.part_lse[split * p.rows + at] = total;
      if (count > 0) {
#pragma unroll 1
        for (int i = 0; i < D / 32; ++i) {
          uint32_t o[32];
          __syncwarp();
          tc_ld32(o_at + i * 32, o);
          tc_wait_ld();
          if (!live) continue;
          float4* dst = reinterpret_cast<float4*>(p.part_o + (split * p.rows + at) * D + i * 32);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dst[e] = make_float4(__uint_as_float(o[4 * e]) * inv, __uint_as_float(o[4 * e + 1]) * inv,
                                 __uint_as_float(o[4 * e + 2]) * inv, __uint_as_float(o[4 * e + 3]) * inv);
        }
      }
    } else {
      if (live && p.lse) p.lse[at] = total * kLn2;
      // through the query tile's memory, which no product reads any more, swizzled as TMA wants it; rows behind the last query
      // are left out by the store
      const int r = threadIdx.x;
      const uint32_t to = q_smem + r * 128;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        uint32_t o[32];
        __syncwarp();
        if (count > 0) {
          tc_ld32(o_at + i * 32, o);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float f[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) f[x] = __uint_as_float(o[8 * e + x]) * inv;
          const uint4 w = pack8(f);
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                       ::"r"(to + (i >> 1) * (kTile * 128) + ((((i & 1) * 4 + e) ^ (r & 7)) << 4)), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
                       : "memory");
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      const int first = row - lane;              // of the warp's 32 rows
      if (lane == 0 && ok && first < z.lq) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) tma_store_4d(&map_o, to + c * (kTile * 128), c * 64, first, h, b);
        asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
      }
      __syncwarp();
    }
  }

  __syncwarp();
  if (abort_flag) {
    // Copies still in flight land before shared memory is released.
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::kMmaWarp) {
    tc_fence_after();
    tc_dealloc(tmem, C::kCols);
  }
}

// out[row] = sum over splits of part_o[split][row] 2^(part_lse[split][row] - total), one warp a row, splits in ascending order.
template <int D>
__global__ void __launch_bounds__(256) attention_join_kernel(const __grid_constant__ FwdParams p) {
  after_previous();
  const int lane = threadIdx.x & 31;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (at >= p.rows) return;
  const float* part_lse = after_previous(p.part_lse);
  const float* part_o = after_previous(p.part_o);
  float top = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) top = fmaxf(top, part_lse[s * p.rows + at]);
  top = warp_max(top);
  const float ref = top == -INFINITY ? 0.f : top;
  float acc[D / 32] = {}, l = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float w = part_lse[s * p.rows + at] - ref;
    if (w == -INFINITY) continue;             // this range saw nothing and wrote nothing
    const float f = exp2_approx(w);
    l += f;
    const float* src = part_o + (s * p.rows + at) * D + lane * (D / 32);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = fmaf(f, src[e], acc[e]);
  }
  const int64_t bh = at / p.z.lq, row = at - bh * p.z.lq, b = bh / p.z.heads, h = bh - b * p.z.heads;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* dst = p.out + b * p.so.b + row * p.so.l + h * p.so.h + lane * (D / 32);
#pragma unroll
  for (int e = 0; e < D / 32; e += 2) *reinterpret_cast<__nv_bfloat162*>(dst + e) = __floats2bfloat162_rn(acc[e] * inv, acc[e + 1] * inv);
  if (p.lse && lane == 0) p.lse[at] = l == 0.f ? -INFINITY : (ref + log2_approx(l)) * kLn2;
}

struct Plan {
  int q_blocks, splits, tiles_per_split;
  explicit Plan(const Shape& s) {
    q_blocks = static_cast<int>(ceil_div(s.lq, kTile));
    // Ranges the keys are cut into where there are fewer CTAs than SMs: as many as fill every SM once (more only add to what is
    // joined: [8, 1 x 16384, 16 / 4 heads, 128] 43 us with twice as many, 35 so), none shorter than three tiles.
    const int64_t ctas = q_blocks * s.heads * s.batch, key_tiles = ceil_div(s.lk, kTile);
    splits = 1;
    if (ctas > 0 && ctas < sm_count()) splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(2LL * sm_count() / ctas, key_tiles / 3)));
    tiles_per_split = static_cast<int>(ceil_div(std::max<int64_t>(1, key_tiles), splits));
  }
};

template <int D>
int launch(const char* who, const CUtensorMap* maps, const FwdParams& p, const Shape& s, cudaStream_t st) {
  using C = FwdCfg<D>;
  static PerDeviceOnce once;
  const cudaError_t rc = per_device_once(once, [] {
    return cudaFuncSetAttribute(attention_fwd_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  ANIMA_REQUIRE(rc == cudaSuccess, ANIMA_E_CUDA, "%s: cannot reserve %d bytes of shared memory: %s", who, C::kSmem,
                cudaGetErrorString(rc));
  const dim3 grid(static_cast<unsigned>(p.q_blocks * p.splits), static_cast<unsigned>(s.heads), static_cast<unsigned>(s.batch));
  launch_after(attention_fwd_kernel<D>, grid, dim3(C::kThreads), C::kSmem, st, maps[0], maps[1], maps[2], maps[3], p);
  ANIMA_CHECK_LAUNCH(who);
  if (p.splits > 1) {
    launch_after(attention_join_kernel<D>, dim3(static_cast<unsigned>(ceil_div(p.rows, 8))), dim3(256), 0, st, p);
    ANIMA_CHECK_LAUNCH(who);
  }
  return ANIMA_OK;
}

}  // namespace
}  // namespace attn
}  // namespace anima

using namespace anima;

extern "C" int64_t anima_attention_fwd_workspace_bytes(int64_t batch, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads,
                                                       int64_t head_dim, int causal) {
  if (int rc = attn::check_sizes("attention_fwd", batch, lq, lk, heads, kv_heads, head_dim)) return rc;
  const int64_t splits = attn::Plan(attn::Shape(batch, lq, lk, heads, kv_heads, head_dim, causal)).splits;
  return splits > 1 ? splits * batch * heads * lq * (head_dim + 1) * 4 : 0;
}

extern "C" int anima_attention_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                   const void* v, const int64_t* v_strides, const int32_t* kv_lengths, int64_t batch,
                                   int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads, int64_t head_dim, float scale,
                                   int causal, void* out, float* lse, void* workspace, int64_t workspace_bytes,
                                   int32_t* status, void* stream) {
  const char* who = "attention_fwd";
  const int64_t need = anima_attention_fwd_workspace_bytes(batch, lq, lk, heads, kv_heads, head_dim, causal);
  if (need < 0) return static_cast<int>(need);
  ANIMA_REQUIRE(scale > 0.f && scale < INFINITY, ANIMA_E_ARG, "%s: scale must be positive and finite", who);
  const bool no_q = batch * lq == 0, no_k = batch * lk == 0;
  if (int rc = attn::check_tensor(who, "q", q, q_strides, no_q)) return rc;
  if (int rc = attn::check_tensor(who, "k", k, k_strides, no_k)) return rc;
  if (int rc = attn::check_tensor(who, "v", v, v_strides, no_k)) return rc;
  if (no_q) return ANIMA_OK;
  ANIMA_REQUIRE(out, ANIMA_E_ARG, "%s: null pointer", who);
  ANIMA_REQUIRE(aligned16(out) && aligned16(workspace), ANIMA_E_ALIGN, "%s: out and workspace must be 16-byte aligned", who);
  ANIMA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), ANIMA_E_WORKSPACE, "%s: workspace of %lld bytes, %lld needed",
                who, (long long)workspace_bytes, (long long)need);
  const attn::Shape s(batch, lq, lk, heads, kv_heads, head_dim, causal);
  attn::Strided sq = attn::strided(q_strides);
  attn::FwdParams p = {};
  p.so = {lq * heads * head_dim, heads * head_dim, head_dim};
  s.regroup(sq);
  s.regroup(p.so);
  p.z = s.sizes(kv_lengths);
  p.c = scale * attn::kLog2e;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.status = status;
  const attn::Plan plan(s);
  p.q_blocks = plan.q_blocks;
  p.splits = plan.splits;
  p.tiles_per_split = plan.tiles_per_split;
  p.rows = s.batch * s.heads * s.lq;
  if (p.splits > 1) {
    p.part_o = static_cast<float*>(workspace);
    p.part_lse = p.part_o + p.splits * p.rows * head_dim;
  }
  CUtensorMap maps[4];
  ANIMA_REQUIRE(attn::bind_context() && attn::encode_heads(&maps[0], q, sq, s.batch, s.lq, s.heads, s.d, q) &&
                    attn::encode_heads(&maps[1], k, attn::strided(k_strides), s.batch, s.lk, s.kv_heads, s.d, q, attn::kStep) &&
                    attn::encode_heads(&maps[2], v, attn::strided(v_strides), s.batch, s.lk, s.kv_heads, s.d, q, attn::kStep) &&
                    attn::encode_heads(&maps[3], out, p.so, s.batch, s.lq, s.heads, s.d, q, 32),
                ANIMA_E_CUDA, "%s: cuTensorMapEncodeTiled failed (driver entry point missing or bad operand)", who);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return head_dim == 64 ? attn::launch<64>(who, maps, p, s, st) : attn::launch<128>(who, maps, p, s, st);
}
