// Attention, forward (formulas: attention_common.cuh): one pass over the keys with each row's running maximum and sum.
//
// A CTA takes tiles of 128 queries of a head, one after the other, and walks the keys for each, 64 at a time. Per step
//   S = Q K^T     tcgen05, both operands in shared memory, fp32 scores in tensor memory (lane = query, column = key);
//   softmax       one warpgroup, one thread a row: 64 scores into registers, row maximum without shuffles,
//                 p = 2^(s scale log2 e - m), rounded to bf16 for the second product (the sum takes the unrounded values), written
//                 over the scores;
//   O += P V      tcgen05 with P read from tensor memory, V as it lies (keys along rows: the MN-major form), fp32.
// The scores have two buffers: S of the step after next is issued behind O += P V, which frees its buffer, so the warpgroup
// finds its next scores ready. One warp issues the products, one feeds K and V through a ring of TMA boxes of 64 keys.
// Two CTAs share an SM (half of its tensor memory and shared memory each): the maxima, sums, loads and waits of one fill the
// special-function unit's and the tensor cores' pauses of the other. One CTA with two query tiles reads K and V half as often,
// but was slower nearly everywhere ([8, 4096 x 512, 16, 128] 224 against 206 us, [8, 4096 x 1024] 275 / 261, [2, 4096 x 4096]
// 245 / 240, [8, 4096 x 4096] 869 / 884, [4, 4096 x 4096, 16, 64] 396 / 363).
// A CTA's set-up, first loads and way out are 6000 cycles, four steps. So, where walks are short, it stays for its next tile, whose
// Q, K and V are loaded and first scores made while the last one's output leaves: [8, 4096 x 512] 173 -> 141 us (run after run 202 ->
// 160), [2, 4096 x 512] 55 -> 46, [8, 4096 x 1024] 259 -> 244.
// O leaves through shared memory and TMA stores (each thread holds a row: its own 16-byte stores took 3000 cycles a tile): through
// Q's place, or, where that is the next tile's by then, through one of its own, 64 columns at a time, for which a stage of K and V
// goes (a fifth changes little; with three, and two places for Q, it took 1.25 x the time).
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

// STAY: the CTA goes on to another tile.
template <int D, bool STAY>
struct FwdCfg {
  static constexpr int kMmaWarp = 4, kTmaWarp = 5, kThreads = 192;
  static constexpr uint32_t kBytes = tile_bytes<D>(), kStepBytes = kBytes / 2;
  static constexpr int kStages = D == 64 ? 8 : STAY ? 4 : 5;
  static constexpr int kBars = 2 * kStages + 8;
  static constexpr int kStagesEnd = static_cast<int>(kBytes + kStages * kStepBytes), kBarsAt = kStagesEnd + (STAY ? kTile * 128 : 0);
  static constexpr int kOutAt = STAY ? kStagesEnd : 0, kSmem = kBarsAt + kBars * 8 + 24;      // on the way out: O
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
  int q_blocks, splits, tiles_per_split, items;
  int block, blocks, last;               // heads that the items go through together, how many such blocks, heads of the last
  Divisor by_block, by_here, by_last, by_split, by_sample, by_group;
  float* part_o;                         // [split][batch, heads, lq][D], null: no split
  float* part_lse;                       // [split][batch, heads, lq], base 2
  int64_t rows;                          // batch * heads * lq
  int32_t* status;
};

struct Walk {
  int split, b, h, hk, q0, n, k0, count;
};
// Item id's range of the keys, sample, heads and query tile. Causal, the tiles' walks differ in length: the items go through blocks
// of heads, the longest walks of all its heads first, so that the short ones fill what is left ([4, 2047, 16 / 4, 64] 81 -> 70 us,
// [1, 16384, 16 / 4, 64] 845 -> 744, [8, 2048, 16, 128] 174 -> 164); few enough heads that their K and V stay in L2.
__device__ __forceinline__ Walk place_of(const FwdParams& p, int id) {
  Walk w;
  const int block = p.by_block.of(id), r = id - block * p.block * p.q_blocks * p.splits;
  const int y = (block == p.blocks - 1 ? p.by_last : p.by_here).of(r), here = block == p.blocks - 1 ? p.last : p.block;
  const int bh = block * p.block + r - y * here, x = p.z.causal ? p.q_blocks * p.splits - 1 - y : y;
  w.split = p.by_split.of(x);
  w.b = p.by_sample.of(bh);
  w.h = bh - w.b * p.z.heads;
  w.hk = p.by_group.of(w.h);
  w.q0 = (x - w.split * p.q_blocks) * kTile;
  return w;
}
template <int D, bool STAY>
__global__ void __launch_bounds__(FwdCfg<D, STAY>::kThreads, 2)
attention_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o,
                     const __grid_constant__ FwdParams p) {
  using C = FwdCfg<D, STAY>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t q_smem = base;
  auto kv_smem = [&](int s) { return base + C::kBytes + s * C::kStepBytes; };
  const uint32_t bars = base + C::kBarsAt;
  // barriers behind the stages' full and empty; bit i of a role's `bits` is the phase of barrier i that it waits for next
  enum { kSFull = 2 * C::kStages, kODone = kSFull + 2, kQFull = kODone + 2, kQFree, kPFull };
  auto bar = [&](int i) { return bars + 8 * i; };
  volatile int& abort_flag = *reinterpret_cast<volatile int*>(smem + (bars - base) + C::kBars * 8 + 8);
  uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(smem + (bars - base) + C::kBars * 8 + 16);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < C::kBars; ++i) mbar_init(bars + 8 * i, i >= kPFull ? 4 : 1);
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
  auto walk_of = [&](int id) {           // this item's keys start at k0, in `count` steps
    Walk w = place_of(p, id);
    w.n = keys_of(z, w.b);
    w.k0 = w.split * p.tiles_per_split * kTile;
    const int lim = min(key_limit(z, w.n, min(z.lq, w.q0 + kTile) - 1), w.k0 + p.tiles_per_split * kTile);
    w.count = max(0, lim - w.k0 + kStep - 1) / kStep;
    return w;
  };
  uint32_t bits = 0;                     // phases of the barriers that a role waits for
  bool ok = true;
  int id = blockIdx.x;
  auto next_item = [&] { return STAY && ok && (id += gridDim.x) < p.items; };
  // the order of the ring: K0, K1, V0, K2, V1, ...
  auto k_at = [](int u) { return u == 0 ? 0 : 2 * u - 1; };
  auto v_at = [](int u, int count) { return 2 * u + (u + 1 < count ? 2 : 1); };

  if (warp == C::kTmaWarp) {
    // ------------------------------------------------------------ TMA producer
    ok = lane == 0;
    bits = ~0u;                          // all is free at first
    if (ok) do {
      const Walk w = walk_of(id);
      if (w.count == 0) continue;
      ok = mbar_wait(bar(kQFree), phase_of(bits, kQFree), &abort_flag);
      if (!ok) break;
      mbar_expect_tx(bar(kQFull), C::kBytes);
      load_rows<D, kTile>(q_smem, &map_q, bar(kQFull), w.q0, w.h, w.b);
      for (int i = 0; i < 2 * w.count && ok; ++i) {
        const int s = i % C::kStages;
        const bool value = i == 2 * w.count - 1 || (i > 0 && !(i & 1));
        const int u = value ? (i - 1) / 2 : (i + 1) / 2;
        ok = mbar_wait(bar(C::kStages + s), phase_of(bits, C::kStages + s), &abort_flag);
        if (!ok) break;
        mbar_expect_tx(bar(s), C::kStepBytes);
        load_rows<D, kStep>(kv_smem(s), value ? &map_v : &map_k, bar(s), w.k0 + u * kStep, w.hk, w.b);
      }
    } while (next_item());
  } else if (warp == C::kMmaWarp) {
    // ------------------------------------------------------------ MMA issuer
    const uint64_t q_desc = tc_desc_sw128(q_smem);
    do {
      const Walk w = walk_of(id);
      if (w.count == 0) continue;
      auto arrived = [&](int i) { return warp_wait(bar(i % C::kStages), phase_of(bits, i % C::kStages), &abort_flag); };
      auto scores = [&](int u) {               // S of step u
        const int s = k_at(u) % C::kStages;
        const uint64_t k = tc_desc_sw128(kv_smem(s));
#pragma unroll
        for (int i = 0; i < D / 16; ++i)       // 16 bytes a unit
          tc_mma_ss(tmem + C::kS + (u & 1) * kStep, q_desc + (i >> 2) * (kTile * 128 / 16) + (i & 3) * 2,
                    k + (i >> 2) * (kStep * 128 / 16) + (i & 3) * 2, tc_idesc_bf16(kTile, kStep), i > 0);
        tc_commit_warp(bar(kSFull + (u & 1)));
        tc_commit_warp(bar(C::kStages + s));
        if (u + 1 == w.count) tc_commit_warp(bar(kQFree));
      };
      ok = warp_wait(bar(kQFull), phase_of(bits, kQFull), &abort_flag);
      for (int u = 0; u < min(2, w.count) && ok; ++u) {
        ok = arrived(k_at(u));
        tc_fence_after();
        if (ok) scores(u);
      }
      for (int u = 0; u < w.count && ok; ++u) {
        const int vs = v_at(u, w.count) % C::kStages;
        const bool next = u + 2 < w.count;
        // keys of the step that exist; the product over the others is left out, up to the next multiple of 16
        const int keys = min(kStep, w.n - w.k0 - u * kStep), steps = (keys + 15) / 16;
        ok = arrived(v_at(u, w.count)) && (!next || arrived(k_at(u + 2)));
        if (!ok) break;
        if (keys & 15) zero_rows<D>(kv_smem(vs), kStep * 128, keys, steps * 16);
        const uint64_t v = tc_desc_sw128(kv_smem(vs), kStep * 128);
        ok = warp_wait(bar(kPFull + (u & 1)), phase_of(bits, kPFull + (u & 1)), &abort_flag);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < kStep / 16; ++i)
          if (i < steps)
            tc_mma_ts(tmem + C::kO, tmem + C::kS + (u & 1) * kStep + i * 8, v + i * (16 * 128 / 16), tc_idesc_bf16(kTile, D, true), u > 0 || i > 0);
        tc_commit_warp(bar(kODone + (u & 1)));
        tc_commit_warp(bar(C::kStages + vs));
        if (next) scores(u + 2);
      }
    } while (next_item());
  } else {
    // ------------------------------------------------------------ softmax: thread = row
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t s_at = tmem + lanes + C::kS, o_at = tmem + lanes + C::kO;
    // of barrier x of two, which every other step completes (not every one is waited for): its phase at step u
    auto phase_at = [&](int u) { return ((bits >> (u & 1)) ^ (u >> 1)) & 1u; };
    do {
      const Walk w = walk_of(id);
      const int count = w.count, k0 = w.k0, row = w.q0 + threadIdx.x;
      const int lim = key_limit(z, w.n, row);
      // the warp's first row sees the fewest keys: steps that end before that need no mask
      const int lim_all = __shfl_sync(0xffffffffu, lim, 0);
      float m = -INFINITY, used = 0.f;     // maximum in use (raw scores), m * c (0 while there is none)
      f2 sum[4] = {0ull, 0ull, 0ull, 0ull};
      // 32 rows behind the last query (a few queries against many keys): nothing is made of their scores, and what lies in their
      // place in tensor memory only reaches rows of O that nobody stores
      const bool idle = row - lane >= z.lq;
      for (int u = 0; u < count; ++u) {
        const uint32_t at = s_at + (u & 1) * kStep;
        ok = warp_wait(bar(kSFull + (u & 1)), phase_at(u), &abort_flag);
        if (!ok) break;
        if (idle) {
          if (lane == 0) mbar_arrive(bar(kPFull + (u & 1)));
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
            ok = warp_wait(bar(kODone + ((u - 1) & 1)), phase_at(u - 1), &abort_flag);
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
          uint32_t word[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const f2 x = f2_fma(f2_make(__uint_as_float(s[i][2 * e]), __uint_as_float(s[i][2 * e + 1])), c2, u2);
            y[i * 16 + e] = (e & 3) < kPoly ? exp2_poly(x) : exp2_pair(x);
            word[e] = bf16_of_f2(y[i * 16 + e]);
          }
          tc_st16(at + i * 16, word);
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kPFull + (u & 1)));
        // the row's sum, behind what the tensor cores wait for
#pragma unroll
        for (int e = 0; e < 32; ++e) sum[e & 3] = f2_add(sum[e & 3], y[e]);
      }
      // ------------------------------------------------------------ epilogue
      if (ok && count > 0) {
        ok = warp_wait(bar(kODone + ((count - 1) & 1)), phase_at(count - 1), &abort_flag);
        tc_fence_after();
      }
      bits ^= ((count + 1) >> 1 & 1) | (count >> 1 & 1) << 1;
      const float l = f2_sum(f2_add(f2_add(sum[0], sum[1]), f2_add(sum[2], sum[3])));
      const float inv = l == 0.f ? 0.f : 1.f / l;        // a row without keys has no sum
      const bool live = row < z.lq && ok;
      const int64_t at = (static_cast<int64_t>(w.b) * z.heads + w.h) * z.lq + row;
      const float total = l == 0.f ? -INFINITY : used + log2_approx(l);      // base 2
      if (!STAY && p.part_o != nullptr) {
        if (live) p.part_lse[w.split * p.rows + at] = total;
        if (count > 0) {
#pragma unroll 1
          for (int i = 0; i < D / 32; ++i) {
            uint32_t o[32];
            __syncwarp();
            tc_ld32(o_at + i * 32, o);
            tc_wait_ld();
            if (!live) continue;
            float4* dst = reinterpret_cast<float4*>(p.part_o + (w.split * p.rows + at) * D + i * 32);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              dst[e] = make_float4(__uint_as_float(o[4 * e]) * inv, __uint_as_float(o[4 * e + 1]) * inv,
                                   __uint_as_float(o[4 * e + 2]) * inv, __uint_as_float(o[4 * e + 3]) * inv);
          }
        }
      } else {
        if (live && p.lse) p.lse[at] = total * kLn2;
        // by way of shared memory, swizzled as TMA wants it; rows behind the last query are left out by the store
        const int first = row - lane;            // of the warp's 32 rows
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          uint32_t o[2][32];
          __syncwarp();
          if (count > 0) {
            tc_ld32(o_at + c * 64, o[0]);
            tc_ld32(o_at + c * 64 + 32, o[1]);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 64; ++e) o[e >> 5][e & 31] = 0u;
          }
          const uint32_t mine = base + C::kOutAt + (STAY ? 0 : c * kTile * 128) + warp * (32 * 128), to = mine + lane * 128;
          if (STAY) {
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // of what went out last
            __syncwarp();
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float f[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) f[x] = __uint_as_float(o[e >> 2][8 * (e & 3) + x]) * inv;
            const uint4 v = pack8(f);
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                         ::"r"(to + ((e ^ (lane & 7)) << 4)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                         : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && ok && first < z.lq) {
            tma_store_4d(&map_o, mine, c * 64, first, w.h, w.b);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        }
      }
      tc_fence_before();                 // O has been read before the next item's first probabilities are announced
    } while (next_item());
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
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

template <int D, bool STAY>
int launch_fwd(const char* who, const CUtensorMap* maps, const FwdParams& p, cudaStream_t st) {
  using C = FwdCfg<D, STAY>;
  static PerDeviceOnce once;
  const cudaError_t rc = per_device_once(once, [] {
    return cudaFuncSetAttribute(attention_fwd_kernel<D, STAY>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  ANIMA_REQUIRE(rc == cudaSuccess, ANIMA_E_CUDA, "%s: cannot reserve %d bytes of shared memory: %s", who, C::kSmem,
                cudaGetErrorString(rc));
  const dim3 grid(static_cast<unsigned>(STAY ? 2LL * sm_count() : p.items));
  launch_after(attention_fwd_kernel<D, STAY>, grid, dim3(C::kThreads), C::kSmem, st, maps[0], maps[1], maps[2], maps[3], p);
  ANIMA_CHECK_LAUNCH(who);
  return ANIMA_OK;
}
template <int D>
int launch(const char* who, const CUtensorMap* maps, const FwdParams& p, const Shape& s, cudaStream_t st) {
  // Where a tile has up to 32 steps, or there are six tiles a CTA, two CTAs a SM take all tiles in turn ([4, 4096 x 1536] 224 -> 204 us,
  // [4, 4096 x 4096, 16, 64] 407 -> 391). Else what that saves is less than what sharing the tiles out beforehand costs, when a SM
  // has two CTAs with one more than the others ([2, 4096 x 4096] run after run 290 instead of 267 us; causal, tiles of unequal
  // length, [4, 2047, 16 / 4, 64] 83 / 75): each has its own CTA, taken by the SM that is free first.
  const int64_t steps = ceil_div(ceil_div(s.lk, kStep), p.splits), slots = 2LL * sm_count();
  const bool stay = !p.z.causal && p.items > slots && (steps <= 32 || p.items >= 6 * slots);
  if (int e = stay ? launch_fwd<D, true>(who, maps, p, st) : launch_fwd<D, false>(who, maps, p, st)) return e;
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
  const int64_t items = plan.q_blocks * static_cast<int64_t>(plan.splits) * s.heads * s.batch;
  ANIMA_REQUIRE(items < (1ll << 30), ANIMA_E_TOO_LARGE, "%s: too many tiles", who);
  p.items = static_cast<int>(items);
  const int64_t all = s.batch * s.heads, per_head = plan.q_blocks * static_cast<int64_t>(plan.splits);
  p.block = p.z.causal ? static_cast<int>(std::min(all, ceil_div(8LL * sm_count(), per_head))) : 1;
  p.blocks = static_cast<int>(ceil_div(all, p.block));
  p.last = static_cast<int>(all - (p.blocks - 1LL) * p.block);
  p.by_block = attn::Divisor(p.block * per_head);
  p.by_here = attn::Divisor(p.block);
  p.by_last = attn::Divisor(p.last);
  p.by_split = attn::Divisor(plan.q_blocks);
  p.by_sample = attn::Divisor(s.heads);
  p.by_group = attn::Divisor(s.heads / s.kv_heads);
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
