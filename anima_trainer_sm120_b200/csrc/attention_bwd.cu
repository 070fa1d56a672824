// Attention, backward (formulas: attention_common.cuh): the probabilities are made again from q, k and the forward's log-sums.
//
// No atomics, every sum in a fixed order:
//   rows   -delta = -out . dout of each query, and minus its log-sum in base 2 (-inf for a query that saw nothing, and for the
//          rows that fill up the last tile: their probabilities come out as 0);
//   keys   a CTA takes tiles of 128 keys of a key head and walks, for each, the query tiles of all heads it serves:
//            S^T = K Q^T, dP^T = V dO^T (lane = key, column = query), dV += P^T dO, dK += dS^T Q; dS goes to memory in bf16;
//   dq     dQ = dS K, a CTA for each tile of 128 queries of a head.
// Where dS would be too large a kernel makes it again for itself instead of dq:
//   queries a CTA takes tiles of 128 queries of a head and walks the key tiles for each:
//            S = Q K^T, dP = dO V^T (lane = query), dQ += dS K.
// P^T, dS^T and dS are read by the tensor cores from tensor memory, where the threads that made them wrote them over the scores,
// and never cross shared memory (whose bandwidth a product with two operands there takes up whole); dQ needs no fp32 buffer that
// all CTAs add to (atomics whose order would change results, and 4 D bytes a query and key tile, twice those of dS at D = 128).
// dS costs 4 bytes of traffic a (query, key) pair and saves two products and an exponential (14 -> 10 D flop): [8, 4096, 16, 128]
// 3.52 -> 3.05 ms, [8, 4096 x 512] 642 -> 530 us, [2, 1024, 16, 128] 83 -> 71 us, [1, 64, 4, 64] 19.5 -> 17.4 us.
// Each tile of q, dO, K lies in shared memory once and serves as a K-major operand of one product and as an MN-major operand
// of another.
// Four warpgroups share a pair of tiles, 32 columns each. One warp issues all products, in the order in which they are waited for
// (a second one lets dK run between dV and the next S, which all warpgroups wait for: 3000 instead of 2600 cycles a pair): dV(i)
// and S(i+1) as soon as P(i) lies in tensor memory, dK(i) and dP(i+1) as soon as dS(i) does. A branch around a product that
// nobody asked for costs the others 10 %: all are made, whichever gradients are wanted.
// Products of 64 instead of 128 columns would let the halves of a tile take turns, but read their A operand from shared memory
// twice as often, which then bounds them (1.5 x the time of the same work in whole tiles).
// Bound: keys, shared memory, which the two products with both operands there and the loads of the others keep busy; dq, memory.
#include "attention_common.cuh"

namespace anima {
namespace attn {
namespace {

constexpr int kWorkers = 16;             // warps that make probabilities: four warpgroups
constexpr int kMmaWarp = kWorkers, kTmaWarp = kWorkers + 1, kThreads = (kWorkers + 2) * 32;
constexpr int kPoly = 1;                 // of four pairs of exponentials, those made on the multiply-add pipes

struct BwdParams {
  Sizes z;
  float c, scale;                        // scale * log2 e, scale
  const float *lse2, *delta;             // [batch, heads, lq_pad], both negated
  int lq_pad;
  __nv_bfloat16 *dq, *dk, *dv;
  Strided sdq;                           // dk, dv: dense
  int tiles, splits, per_split;          // key (query) tiles; ranges their walks are cut into, and how long these are
  int head0, heads_now, items;           // the launch's first head of those of all samples, their number; tiles * splits * heads_now
  int block, last_first;                 // heads that the items go through together; from the last tile on
  // dS as the tensor cores read it, in tiles [query head - ds_head][query tile][key tile] of kDsTile bytes, null: not stored. A tile:
  // [half of the keys][8 queries][key][query] bf16.
  uint8_t* ds;
  int ds_head, q_tiles, k_tiles;
  float *part0, *part1;                  // fp32 partial sums [split][elements], if splits > 1: dv and dk, or dq
  int64_t elements;
  int32_t* status;
};

struct RowsParams {
  const __nv_bfloat16 *out, *dout;
  Strided so, sdo;
  const float* lse;
  float *lse2, *delta;
  int lq, lq_pad, heads;
  Divisor by_heads;
};

// D / 8 lanes a row; a CTA takes rows_per_cta (token, head) rows of a sample in the order of memory, all loads first. grid (., batch).
// Bound: reading out and dout once, [8, 4096, 16, 128] 46.5 us, 5.8 TB/s (with the log-sums loaded last and a division a row 60).
constexpr int kRowsPerThread = 2;
template <int D>
constexpr int rows_per_cta() { return 256 / (D / 8) * kRowsPerThread; }
template <int D>
__global__ void __launch_bounds__(256) attention_rows_kernel(const __grid_constant__ RowsParams p) {
  after_previous();
  constexpr int kLanes = D / 8, kRows = 256 / kLanes;
  const int lane = threadIdx.x & (kLanes - 1), all = p.lq_pad * p.heads;
  const int64_t b = blockIdx.y;
  const int first = blockIdx.x * rows_per_cta<D>() + static_cast<int>(threadIdx.x) / kLanes;
  const __nv_bfloat16* out = after_previous(p.out) + b * p.so.b + lane * 8;
  const __nv_bfloat16* dout = after_previous(p.dout) + b * p.sdo.b + lane * 8;
  uint4 x[kRowsPerThread], y[kRowsPerThread];
  int l[kRowsPerThread], h[kRowsPerThread];
  float lse[kRowsPerThread];
  const float* lses = after_previous(p.lse);
#pragma unroll
  for (int i = 0; i < kRowsPerThread; ++i) {
    const int r = first + i * kRows;
    l[i] = p.by_heads.of(r);
    h[i] = r - l[i] * p.heads;
    x[i] = y[i] = make_uint4(0u, 0u, 0u, 0u);
    lse[i] = -INFINITY;
    if (l[i] < p.lq) {
      if (lane == 0) lse[i] = lses[(b * p.heads + h[i]) * p.lq + l[i]];
      x[i] = ldg_stream16(out + l[i] * p.so.l + h[i] * p.so.h);
      y[i] = *reinterpret_cast<const uint4*>(dout + l[i] * p.sdo.l + h[i] * p.sdo.h);      // read again by the next two kernels
    }
  }
#pragma unroll
  for (int i = 0; i < kRowsPerThread; ++i) {
    f2 s = f2_mul(f2_of_bf16(x[i].x), f2_of_bf16(y[i].x));
    s = f2_fma(f2_of_bf16(x[i].y), f2_of_bf16(y[i].y), s);
    s = f2_fma(f2_of_bf16(x[i].z), f2_of_bf16(y[i].z), s);
    s = f2_fma(f2_of_bf16(x[i].w), f2_of_bf16(y[i].w), s);
    float t = f2_sum(s);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane != 0 || first + i * kRows >= all) continue;
    const int64_t bh = b * p.heads + h[i], to = bh * p.lq_pad + l[i];
    p.lse2[to] = lse[i] == -INFINITY ? -INFINITY : lse[i] * -kLog2e;
    p.delta[to] = lse[i] == -INFINITY ? 0.f : -t;
  }
}

// Shared memory: two tiles that stay, a ring (keys: three tiles of q, two of dout with lse2 and delta; queries: five tiles of K
// and V), barriers.
// bytes: a tile, 64 keys of it, 8 queries of these
constexpr int kDsTile = kTile * kTile * 2, kDsHalf = kDsTile / 2, kDsGroup = kTile / 2 * 16;
__device__ __forceinline__ uint32_t ds_index(const BwdParams& p, int head, int qt, int kt) {       // of 4 GiB / kDsTile tiles at most
  return (static_cast<uint32_t>(head - p.ds_head) * p.q_tiles + qt) * p.k_tiles + kt;
}

template <int D>
struct BwdCfg {
  static constexpr uint32_t kBytes = tile_bytes<D>();
  static constexpr int kQ = 3, kG = 2, kStages = kQ + kG;              // tiles of q, of dout; of K and V
  static constexpr int kRowBytes = 2 * kTile * 4;                      // lse2 and delta of a tile
  static constexpr int kBars = 12 + 2 * kStages;
  static constexpr int kSmem = (2 + kStages) * kBytes + kG * kRowBytes + kBars * 8;
  static_assert(kSmem <= 227 * 1024, "shared memory");
  static constexpr uint32_t kS = 0, kDp = 128, kAcc0 = 256, kAcc1 = 256 + D;   // tensor-memory columns
};
template <int D>
struct Layout {
  using C = BwdCfg<D>;
  uint32_t base;
  __device__ __forceinline__ uint32_t fixed(int i) const { return base + i * C::kBytes; }
  __device__ __forceinline__ uint32_t stage(int s) const { return base + (2 + s) * C::kBytes; }        // keys: those of dout come first
  __device__ __forceinline__ uint32_t row_data(int s) const { return base + (2 + C::kStages) * C::kBytes + s * C::kRowBytes; }
  __device__ __forceinline__ uint32_t bar(int i) const { return row_data(C::kG) + 8 * i; }             // 10, 11: the abort flag, the tensor-memory address
  __device__ __forceinline__ uint32_t full(int s) const { return bar(12 + s); }
  __device__ __forceinline__ uint32_t empty(int s) const { return bar(12 + C::kStages + s); }
};
// (queries: kSFull one for each score buffer)
enum { kFixedFull = 0, kDone = 1, kSFull = 2, kDpFull = 4, kAccFree = 5, kPReady = 6, kFixedFree = 7, kDsReady = 8 };

// One item of a CTA's work: range `split` of the walk of one tile. The CTAs go through the items in turn, so that the loads and
// first products of an item overlap the last passes and the way out of the one before. Causal, the tiles' walks differ in
// length: the items go through blocks of heads, the longest walks of all its heads first, so that the short ones fill what is
// left ([4, 2047, 16 / 4, 64] 216 -> 170 us, [1, 16384, 16 / 4, 64] 3.03 -> 2.27 ms, [8, 2048, 16, 128] 498 -> 480 us). Few enough heads that
// what they read stays in L2. 32-bit arithmetic: a 64-bit division is a call, behind which the
// compiler takes nothing for uniform any more (see phase_of; 761 became 873 us).
struct Item {
  int split, tile, head, b;
};
__device__ __forceinline__ Item item_of(const BwdParams& p, int id, int heads) {
  Item it;
  it.split = id % p.splits;
  const int rest = id / p.splits;
  int bh = rest / p.tiles, x = rest - bh * p.tiles;
  if (p.block > 1) {
    const int block = bh / p.block, here = min(p.block, p.heads_now - block * p.block), r = rest - block * p.block * p.tiles;
    x = r / here;
    bh = block * p.block + r - x * here;
  }
  bh += p.head0;
  it.tile = p.last_first ? p.tiles - 1 - x : x;
  it.head = bh % heads;
  it.b = bh / heads;
  return it;
}

template <int D>
__device__ __forceinline__ void setup(const Layout<D>& m, volatile int* abort_flag, uint32_t* tmem_slot, int warp) {
  using C = BwdCfg<D>;
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < C::kBars; ++i)
      if (i < 10 || i >= 12) mbar_init(m.bar(i), i == kAccFree || i == kPReady || i == kDsReady ? kWorkers : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) tc_alloc(smem_u32(tmem_slot), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  after_previous();
}
__device__ __forceinline__ void teardown(volatile int* abort_flag, int32_t* status, uint32_t tmem, int warp) {
  __syncwarp();
  if (*abort_flag) {
    // Copies still in flight land before shared memory is released.
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
    if (threadIdx.x == 0 && status) atomicExch(status, 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tc_dealloc(tmem, 512);
  }
}

// D[tmem] = A . B^T of two tiles in shared memory, the head vector along K
template <int D>
__device__ __forceinline__ void product_ss(uint32_t d, uint32_t a_smem, uint32_t b_smem) {
  const uint64_t a = tc_desc_sw128(a_smem), b = tc_desc_sw128(b_smem);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const uint32_t at = (i >> 2) * (kTile * 128 / 16) + (i & 3) * 2;     // 16 bytes a unit
    tc_mma_ss(d, a + at, b + at, tc_idesc_bf16(kTile, kTile), i > 0);
  }
}
// D[tmem] += A . B over the first 16 `steps` rows of the tile B: A bf16 in tensor memory, elements 32 w .. 32 w + 31 of a row in
// columns a + 32 w .. + 15
template <int D>
__device__ __forceinline__ void product_ts(uint32_t d, uint32_t a, uint32_t b_smem, int steps, bool accumulate) {
  const uint64_t b = tc_desc_sw128(b_smem, kTile * 128);
#pragma unroll
  for (int i = 0; i < kTile / 16; ++i)
    if (i < steps) tc_mma_ts(d, a + (i >> 1) * 32 + (i & 1) * 8, b + i * (16 * 128 / 16), tc_idesc_bf16(kTile, D, true), accumulate || i > 0);
}

// N elements of a thread's row of an fp32 accumulator, scaled: bf16 to dst, or fp32 to part (either may be null)
template <int N>
__device__ __forceinline__ void store_row(uint32_t acc, bool has, float scale, bool live, __nv_bfloat16* dst, float* part) {
#pragma unroll
  for (int i = 0; i < N / 16; ++i) {
    uint32_t o[16];
    __syncwarp();
    if (has) {
      tc_ld16(acc + i * 16, o);
      tc_wait_ld();
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] = 0u;
    }
    if (!live) continue;
    if (part) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        reinterpret_cast<float4*>(part + i * 16)[e] =
            make_float4(__uint_as_float(o[4 * e]) * scale, __uint_as_float(o[4 * e + 1]) * scale,
                        __uint_as_float(o[4 * e + 2]) * scale, __uint_as_float(o[4 * e + 3]) * scale);
    } else if (dst) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float f[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) f[x] = __uint_as_float(o[8 * e + x]) * scale;
        *reinterpret_cast<uint4*>(dst + i * 16 + e * 8) = pack8(f);
      }
    }
  }
}

// two pairs of floats from shared memory
__device__ __forceinline__ void lds_pairs(uint32_t addr, f2& a, f2& b) {
  asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(a), "=l"(b) : "r"(addr));
}
__device__ __forceinline__ f2 pair_of(const uint32_t (&v)[32], int e) { return f2_make(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])); }
// Pair e of a run of exponentials: some on either unit, so that neither waits for the other.
__device__ __forceinline__ f2 exp2_mixed(f2 x, int e) { return (e & 3) < kPoly ? exp2_poly(x) : exp2_pair(x); }

// ------------------------------------------------------------------------------------------------ keys: dK, dV
template <int D>
__global__ void __launch_bounds__(kThreads, 1)
attention_bwd_keys_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                          const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                          const __grid_constant__ BwdParams p) {
  using C = BwdCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const Layout<D> m{smem_u32(smem)};
  volatile int& abort_flag = *reinterpret_cast<volatile int*>(smem + (m.bar(10) - m.base));
  uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(smem + (m.bar(11) - m.base));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  setup<D>(m, &abort_flag, &tmem_slot, warp);
  constexpr uint32_t tmem = 0;             // the address of an allocation of all 512 columns

  const Sizes& z = p.z;
  const int off = z.lk - z.lq, q_tiles = (z.lq + kTile - 1) / kTile;
  struct Walk {
    Item it;
    int k0, n, first, per_head, begin, count;
  };
  auto walk_of = [&](int id) {
    Walk w;
    w.it = item_of(p, id, z.kv_heads);
    w.k0 = w.it.tile * kTile;
    w.n = keys_of(z, w.it.b);
    w.first = z.causal ? min(q_tiles, max(0, w.k0 - off) / kTile) : 0;         // the first query tile with a row that sees a key here
    w.per_head = w.k0 < w.n ? q_tiles - w.first : 0;
    w.begin = w.it.split * p.per_split;
    w.count = max(0, min(z.group * w.per_head, w.begin + p.per_split) - w.begin);
    return w;
  };
  // pass i of a walk: query tile `tile_at` of head `head_at`
  auto head_at = [&](const Walk& w, int i) { return w.it.head * z.group + (w.begin + i) / w.per_head; };
  auto tile_at = [&](const Walk& w, int i) { return w.first + (w.begin + i) % w.per_head; };
  auto g_at = [](int i) { return i % C::kG; };
  auto q_at = [](int i) { return C::kG + i % C::kQ; };
  // r counts the CTA's passes, x its items with any, bits holds the phases of the stages; each role for itself
  int r = 0, x = 0;
  uint32_t bits = 0;

  if (warp == kTmaWarp) {
    // ------------------------------------------------------------ TMA producer: K, V, then q0, dout0 (with lse2, delta), q1, ...
    bool ok = lane == 0;
    bits = ~0u;                            // of the stages' release: all are free at first
    for (int id = blockIdx.x; id < p.items && ok; id += gridDim.x) {
      const Walk w = walk_of(id);
      if (w.count == 0) continue;
      ok = x == 0 || mbar_wait(m.bar(kFixedFree), (x - 1) & 1, &abort_flag);
      if (!ok) break;
      mbar_expect_tx(m.bar(kFixedFull), 2 * C::kBytes);
      load_rows<D, kTile>(m.fixed(0), &map_k, m.bar(kFixedFull), w.k0, w.it.head, w.it.b);
      load_rows<D, kTile>(m.fixed(1), &map_v, m.bar(kFixedFull), w.k0, w.it.head, w.it.b);
      for (int i = 0; i < w.count && ok; ++i) {
        const int s = q_at(i), g = g_at(i), h = head_at(w, i), q0 = tile_at(w, i) * kTile;
        ok = mbar_wait(m.empty(s), phase_of(bits, s), &abort_flag);
        if (!ok) break;
        mbar_expect_tx(m.full(s), C::kBytes);
        load_rows<D, kTile>(m.stage(s), &map_q, m.full(s), q0, h, w.it.b);
        ok = mbar_wait(m.empty(g), phase_of(bits, g), &abort_flag);
        if (!ok) break;
        mbar_expect_tx(m.full(g), C::kBytes + C::kRowBytes);
        const int64_t at = (static_cast<int64_t>(w.it.b) * z.heads + h) * p.lq_pad + q0;
        bulk_load(m.row_data(g), p.lse2 + at, kTile * 4, m.full(g));
        bulk_load(m.row_data(g) + kTile * 4, p.delta + at, kTile * 4, m.full(g));
        load_rows<D, kTile>(m.stage(g), &map_do, m.full(g), q0, h, w.it.b);
      }
      ++x;
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMA issuer
    bool ok = true;
    for (int id = blockIdx.x; id < p.items && ok; id += gridDim.x) {
      const Walk w = walk_of(id);
      if (w.count == 0) continue;
      // Causal, more queries than keys: the first -off queries see nothing. Whole tiles of them are not walked; in the tile they
      // share with others their rows of q and dout are cleared (by a whole warp), so that whatever they hold meets a probability
      // of 0 as 0.
      auto clear_blind = [&](int i, uint32_t at) {
        const int blind = -off - tile_at(w, i) * kTile;
        if (z.causal && blind > 0) zero_rows<D>(at, kTile * 128, 0, min(kTile, blind));
      };
      auto scores = [&](int i) {           // S^T(i) = K Q^T
        const int s = q_at(i);
        if (!warp_wait(m.full(s), phase_of(bits, s), &abort_flag)) return false;
        clear_blind(i, m.stage(s));
        tc_fence_after();
        product_ss<D>(tmem + C::kS, m.fixed(0), m.stage(s));
        tc_commit_warp(m.bar(kSFull));
        return true;
      };
      auto gradients = [&](int i) {        // dP^T(i) = V dO^T
        const int g = g_at(i);
        if (!warp_wait(m.full(g), phase_of(bits, g), &abort_flag)) return false;
        clear_blind(i, m.stage(g));
        tc_fence_after();
        product_ss<D>(tmem + C::kDp, m.fixed(1), m.stage(g));
        tc_commit_warp(m.bar(kDpFull));
        if (i + 1 == w.count) tc_commit_warp(m.bar(kFixedFree));
        return true;
      };
      ok = warp_wait(m.bar(kFixedFull), x & 1, &abort_flag) && scores(0) && gradients(0);
      for (int i = 0; i < w.count && ok; ++i) {
        const bool more = i + 1 < w.count;
        ok = warp_wait(m.bar(kPReady), (r + i) & 1, &abort_flag) &&
             (i > 0 || x == 0 || warp_wait(m.bar(kAccFree), (x - 1) & 1, &abort_flag));
        if (!ok) break;
        tc_fence_after();
        product_ts<D>(tmem + C::kAcc0, tmem + C::kS, m.stage(g_at(i)), kTile / 16, i > 0);
        ok = (!more || scores(i + 1)) && warp_wait(m.bar(kDsReady), (r + i) & 1, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        tc_commit_warp(m.empty(g_at(i)));      // dV(i) and dP(i) are through with it, and delta has been read
        product_ts<D>(tmem + C::kAcc1, tmem + C::kDp, m.stage(q_at(i)), kTile / 16, i > 0);
        tc_commit_warp(m.empty(q_at(i)));
        if (!more) tc_commit_warp(m.bar(kDone));
        ok = !more || gradients(i + 1);
      }
      r += w.count;
      ++x;
    }
  } else {
    // ------------------------------------------------------------ probabilities: thread = key, warpgroup wg has 32 queries
    const int wg = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + C::kS + wg * 32, dp_at = tmem + lanes + C::kDp + wg * 32;
    const f2 c2 = f2_dup(p.c);
    const uint32_t ds_step = static_cast<uint32_t>(p.k_tiles) * (kDsTile / 16);        // to the next query tile's
    bool ok = true;
    for (int id = blockIdx.x; id < p.items && ok; id += gridDim.x) {
      const Walk w = walk_of(id);
      const int row = w.k0 + (threadIdx.x & 127);
      const bool row_ok = row < w.n;
      // the pass's query tile and the thread's place in the tiles of dS, which the walk goes through in order
      int qt = 0;
      uint32_t ds = 0;                   // in 16 bytes
      if (w.count > 0) {
        qt = tile_at(w, 0);
        ds = ds_index(p, w.it.b * z.heads + head_at(w, 0), qt, w.it.tile) * (kDsTile / 16) +
             (((threadIdx.x >> 6) & 1) * kDsHalf + wg * 4 * kDsGroup) / 16 + (threadIdx.x & 63);
      }
      for (int i = 0; i < w.count; ++i, ++r) {
        const uint32_t rows = m.row_data(g_at(i)) + wg * 128;
        // queries of these 32 before `from` do not see this key
        int from = row_ok ? 0 : 32;
        if (z.causal && row_ok) from = row - off - qt * kTile - wg * 32;
        const bool edge = __any_sync(0xffffffffu, from > 0);
        ok = warp_wait(m.full(g_at(i)), phase_of(bits, g_at(i)), &abort_flag);
        if (!ok) break;
        f2 pr[16], rd[16];               // the log-sums are read while the scores are waited for (after it: 1310 instead of 950 cycles to P)
#pragma unroll
        for (int e = 0; e < 16; e += 2) lds_pairs(rows + e * 8, rd[e], rd[e + 1]);
        ok = warp_wait(m.bar(kSFull), r & 1, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[32], word[16];
        tc_ld32(s_at, s);
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) pr[e] = exp2_mixed(f2_fma(pair_of(s, e), c2, rd[e]), e);
        if (edge) {
#pragma unroll
          for (int e = 0; e < 16; ++e) pr[e] = f2_make(2 * e >= from ? f2_lo(pr[e]) : 0.f, 2 * e + 1 >= from ? f2_hi(pr[e]) : 0.f);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) word[e] = bf16_of_f2(pr[e]);
        tc_st16(s_at, word);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(m.bar(kPReady));

        ok = warp_wait(m.bar(kDpFull), r & 1, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        tc_ld32(dp_at, s);
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          f2 d0, d1;
          lds_pairs(rows + kTile * 4 + e * 8, d0, d1);
          word[e] = bf16_of_f2(f2_mul(pr[e], f2_add(pair_of(s, e), d0)));
          word[e + 1] = bf16_of_f2(f2_mul(pr[e + 1], f2_add(pair_of(s, e + 1), d1)));
        }
        if (!row_ok) {                   // what lies behind the sample's keys may be NaN
#pragma unroll
          for (int e = 0; e < 16; ++e) word[e] = 0u;
        }
        tc_st16(dp_at, word);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(m.bar(kDsReady));
        // 512 contiguous bytes a warp and store (through shared memory and copies: the same time, D = 64 5 % more)
        if (p.ds != nullptr) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            reinterpret_cast<uint4*>(p.ds)[static_cast<uint64_t>(ds) + e * (kDsGroup / 16)] = make_uint4(word[4 * e], word[4 * e + 1], word[4 * e + 2], word[4 * e + 3]);
        }
        if (++qt == q_tiles) {
          qt = w.first;
          ds += w.first * ds_step;
        }
        ds += ds_step;
      }
      if (ok && w.count > 0) {
        ok = warp_wait(m.bar(kDone), x & 1, &abort_flag);
        tc_fence_after();
      }
      // warpgroups 0 and 1: the halves of dV; 2 and 3: of dK
      const int64_t at = ((static_cast<int64_t>(w.it.b) * z.lk + row) * z.kv_heads + w.it.head) * D + (wg & 1) * (D / 2);
      __nv_bfloat16* dst = wg < 2 ? p.dv : p.dk;
      float* part = wg < 2 ? p.part0 : p.part1;
      store_row<D / 2>(tmem + lanes + (wg < 2 ? C::kAcc0 : C::kAcc1) + (wg & 1) * (D / 2), w.count > 0, wg < 2 ? 1.f : p.scale,
                       ok && row < z.lk, dst ? dst + at : nullptr, dst && part ? part + w.it.split * p.elements + at : nullptr);
      if (w.count > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(m.bar(kAccFree));
        ++x;
      }
    }
  }
  teardown(&abort_flag, p.status, tmem, warp);
}

// ------------------------------------------------------------------------------------------------ queries: dQ
// P stays in registers here, so the scores have two buffers and S(j + 1) is ready
// when the warpgroups come to it.
template <int D>
__global__ void __launch_bounds__(kThreads, 1)
attention_bwd_queries_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                             const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                             const __grid_constant__ BwdParams p) {
  using C = BwdCfg<D>;
  constexpr uint32_t kS1 = C::kAcc1;       // second buffer of the scores
  extern __shared__ __align__(1024) uint8_t smem[];
  const Layout<D> m{smem_u32(smem)};
  volatile int& abort_flag = *reinterpret_cast<volatile int*>(smem + (m.bar(10) - m.base));
  uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(smem + (m.bar(11) - m.base));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  setup<D>(m, &abort_flag, &tmem_slot, warp);
  constexpr uint32_t tmem = 0;             // the address of an allocation of all 512 columns

  const Sizes& z = p.z;
  struct Walk {
    Item it;
    int q0, n, j0, count;
  };
  auto walk_of = [&](int id) {
    Walk w;
    w.it = item_of(p, id, z.heads);
    w.q0 = w.it.tile * kTile;
    w.n = keys_of(z, w.it.b);
    w.j0 = w.it.split * p.per_split;
    const int lim = key_limit(z, w.n, min(z.lq, w.q0 + kTile) - 1);
    w.count = max(0, min((lim + kTile - 1) / kTile, w.j0 + p.per_split) - w.j0);
    return w;
  };
  // r counts the CTA's passes, x its items with any, bits holds the phases of the stages (of the score buffers); each role for itself
  int r = 0, x = 0;
  uint32_t bits = 0;

  if (warp == kTmaWarp) {
    // ------------------------------------------------------------ TMA producer: q, dout, then K0, V0, K1, V1, ...
    bool ok = lane == 0;
    bits = ~0u;                            // of the stages' release: all are free at first
    for (int id = blockIdx.x; id < p.items && ok; id += gridDim.x) {
      const Walk w = walk_of(id);
      if (w.count == 0) continue;
      ok = x == 0 || mbar_wait(m.bar(kFixedFree), (x - 1) & 1, &abort_flag);
      if (!ok) break;
      mbar_expect_tx(m.bar(kFixedFull), 2 * C::kBytes);
      load_rows<D, kTile>(m.fixed(0), &map_q, m.bar(kFixedFull), w.q0, w.it.head, w.it.b);
      load_rows<D, kTile>(m.fixed(1), &map_do, m.bar(kFixedFull), w.q0, w.it.head, w.it.b);
      for (int i = 0; i < 2 * w.count; ++i) {
        const int s = i % C::kStages;
        ok = mbar_wait(m.empty(s), phase_of(bits, s), &abort_flag);
        if (!ok) break;
        mbar_expect_tx(m.full(s), C::kBytes);
        load_rows<D, kTile>(m.stage(s), (i & 1) ? &map_v : &map_k, m.full(s), (w.j0 + (i >> 1)) * kTile, w.it.head / z.group, w.it.b);
      }
      ++x;
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMA issuer
    bool ok = true;
    for (int id = blockIdx.x; id < p.items && ok; id += gridDim.x) {
      const Walk w = walk_of(id);
      if (w.count == 0) continue;
      auto k_stage = [&](int j) { return 2 * j % C::kStages; };
      auto v_stage = [&](int j) { return (2 * j + 1) % C::kStages; };
      auto keys_in = [&](int j) { return min(kTile, w.n - (w.j0 + j) * kTile); };
      auto scores = [&](int j) {           // S(j) = Q K_j^T; the keys' rows behind the sample's length are cleared for dS K
        const int s = k_stage(j), keys = keys_in(j);
        if (!warp_wait(m.full(s), phase_of(bits, s), &abort_flag)) return false;
        if (keys & 15) zero_rows<D>(m.stage(s), kTile * 128, keys, (keys + 15) & ~15);
        tc_fence_after();
        product_ss<D>(tmem + ((j & 1) ? kS1 : C::kS), m.fixed(0), m.stage(s));
        tc_commit_warp(m.bar(kSFull + (j & 1)));
        return true;
      };
      auto gradients = [&](int j) {        // dP(j) = dO V_j^T
        const int s = v_stage(j);
        if (!warp_wait(m.full(s), phase_of(bits, s), &abort_flag)) return false;
        tc_fence_after();
        product_ss<D>(tmem + C::kDp, m.fixed(1), m.stage(s));
        tc_commit_warp(m.bar(kDpFull));
        tc_commit_warp(m.empty(s));
        if (j + 1 == w.count) tc_commit_warp(m.bar(kFixedFree));      // S(j) came before
        return true;
      };
      ok = warp_wait(m.bar(kFixedFull), x & 1, &abort_flag) && scores(0) && (w.count == 1 || scores(1)) && gradients(0);
      for (int j = 0; j < w.count && ok; ++j) {      // dS(j) is ready: dQ += dS K, the next dP, the scores after the next
        ok = warp_wait(m.bar(kDsReady), (r + j) & 1, &abort_flag) &&
             (j > 0 || x == 0 || warp_wait(m.bar(kAccFree), (x - 1) & 1, &abort_flag));
        if (!ok) break;
        tc_fence_after();
        product_ts<D>(tmem + C::kAcc0, tmem + C::kDp, m.stage(k_stage(j)), (keys_in(j) + 15) / 16, j > 0);
        tc_commit_warp(m.empty(k_stage(j)));
        if (j + 1 == w.count) tc_commit_warp(m.bar(kDone));
        ok = (j + 1 >= w.count || gradients(j + 1)) && (j + 2 >= w.count || scores(j + 2));
      }
      r += w.count;
      ++x;
    }
  } else {
    // ------------------------------------------------------------ probabilities: thread = query, warpgroup wg has 32 keys
    const int wg = warp >> 2, col = wg * 32;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t dp_at = tmem + lanes + C::kDp + col;
    const f2 c2 = f2_dup(p.c);
    bool ok = true;
    for (int id = blockIdx.x; id < p.items && ok; id += gridDim.x) {
      const Walk w = walk_of(id);
      const int row = w.q0 + (threadIdx.x & 127), h = w.it.head, b = w.it.b;
      const int lim = key_limit(z, w.n, row);
      const int lim_all = __shfl_sync(0xffffffffu, lim, 0);
      const int64_t at = (static_cast<int64_t>(b) * z.heads + h) * p.lq_pad + row;
      const f2 lse = f2_dup(p.lse2[at]), delta = f2_dup(p.delta[at]);
      for (int j = 0; j < w.count; ++j, ++r) {
        ok = warp_wait(m.bar(kSFull + (j & 1)), phase_of(bits, j & 1), &abort_flag);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[32], word[16];
        tc_ld32(tmem + lanes + ((j & 1) ? kS1 : C::kS) + col, s);
        tc_wait_ld();
        f2 pr[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) pr[e] = exp2_mixed(f2_fma(pair_of(s, e), c2, lse), e);
        ok = warp_wait(m.bar(kDpFull), r & 1, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        tc_ld32(dp_at, s);
        tc_wait_ld();
        const int key = (w.j0 + j) * kTile + col, from = lim - key;      // keys from here on are not seen
#pragma unroll
        for (int e = 0; e < 16; ++e) pr[e] = f2_mul(pr[e], f2_add(pair_of(s, e), delta));
        if (key + 32 > lim_all) {        // what lies behind the sample's keys may be NaN
#pragma unroll
          for (int e = 0; e < 16; ++e) pr[e] = f2_make(2 * e < from ? f2_lo(pr[e]) : 0.f, 2 * e + 1 < from ? f2_hi(pr[e]) : 0.f);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) word[e] = bf16_of_f2(pr[e]);
        tc_st16(dp_at, word);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(m.bar(kDsReady));
      }
      if (ok && w.count > 0) {
        ok = warp_wait(m.bar(kDone), x & 1, &abort_flag);
        tc_fence_after();
      }
      const int64_t dense = ((static_cast<int64_t>(b) * z.heads + h) * z.lq + row) * D + wg * (D / 4);
      store_row<D / 4>(tmem + lanes + C::kAcc0 + wg * (D / 4), w.count > 0, p.scale, ok && row < z.lq,
                       p.dq + b * p.sdq.b + row * p.sdq.l + h * p.sdq.h + wg * (D / 4),
                       p.part0 ? p.part0 + w.it.split * p.elements + dense : nullptr);
      if (w.count > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(m.bar(kAccFree));
        ++x;
      }
    }
  }
  teardown(&abort_flag, p.status, tmem, warp);
}

// ------------------------------------------------------------------------------------------------ queries, dS stored: dQ
// dQ = dS K with the dS that the keys kernel left in memory, which bounds it: [8, 4096, 16, 128] reads 1 GiB in 178 us, 6.0 TB/s.
// 64 keys a stage; a CTA takes a query tile, or a range of its keys where there are few query tiles; two share an SM, so that one
// loads while the other stores.
template <int D>
struct DqCfg {
  static constexpr uint32_t kKeyBytes = tile_bytes<D>() / 2, kStageBytes = kDsHalf + kKeyBytes;
  static constexpr int kStages = D == 128 ? 3 : 4, kBars = 2 * kStages + 1;
  static constexpr int kSmem = kStages * static_cast<int>(kStageBytes) + kBars * 8 + 24, kThreads = 192;
  static_assert(2 * (kSmem + 1024) <= 228 * 1024 && kStageBytes >= tile_bytes<D>() / 2, "shared memory of two CTAs");
};
template <int D>
__global__ void __launch_bounds__(DqCfg<D>::kThreads, 2)
attention_bwd_dq_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_dq,
                        const __grid_constant__ BwdParams p) {
  using C = DqCfg<D>;
  constexpr int kStep = kTile / 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem), bars = base + C::kStages * C::kStageBytes, done = bars + 16 * C::kStages;
  auto stage = [&](int i) { return base + i % C::kStages * C::kStageBytes; };      // K, then dS
  auto full = [&](int i) { return bars + 8 * (i % C::kStages); };
  auto empty = [&](int i) { return bars + 8 * (C::kStages + i % C::kStages); };
  volatile int& abort_flag = *reinterpret_cast<volatile int*>(smem + (bars - base) + C::kBars * 8 + 8);
  uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(smem + (bars - base) + C::kBars * 8 + 16);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < C::kBars; ++i) mbar_init(bars + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4) tc_alloc(smem_u32(&tmem_slot), 128);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  after_previous();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);

  const Sizes& z = p.z;
  const Item it = item_of(p, p.items - 1 - static_cast<int>(blockIdx.x), z.heads);       // what was stored last may still be in L2
  const int q0 = it.tile * kTile, n = keys_of(z, it.b), step0 = it.split * p.per_split * 2;      // in steps of 64 keys
  const int count = min((key_limit(z, n, min(z.lq, q0 + kTile) - 1) + kStep - 1) / kStep - step0, p.per_split * 2);
  if (warp == 5) {
    if (lane == 0 && count > 0) {
      asm volatile("fence.proxy.async.global;" ::: "memory");      // dS was written by ordinary stores
      const uint8_t* ds = p.ds + static_cast<int64_t>(ds_index(p, it.b * z.heads + it.head, it.tile, 0)) * kDsTile + static_cast<int64_t>(step0) * kDsHalf;
      for (int i = 0; i < count; ++i) {
        if (!mbar_wait(empty(i), ((i / C::kStages) & 1) ^ 1, &abort_flag)) break;
        mbar_expect_tx(full(i), C::kStageBytes);
        bulk_load(stage(i) + C::kKeyBytes, ds + static_cast<int64_t>(i) * kDsHalf, kDsHalf, full(i));
        load_rows<D, kStep>(stage(i), &map_k, full(i), (step0 + i) * kStep, it.head / z.group, it.b);
      }
    }
  } else if (warp == 4) {
    bool ok = true;
    for (int i = 0; i < count && ok; ++i) {
      ok = warp_wait(full(i), (i / C::kStages) & 1, &abort_flag);
      if (!ok) break;
      // keys that exist; their rows up to the next multiple of 16 are cleared, the product over the others is left out
      const int keys = min(kStep, n - (step0 + i) * kStep), steps = (keys + 15) / 16;
      if (keys & 15) zero_rows<D>(stage(i), kStep * 128, keys, steps * 16);
      tc_fence_after();
      const uint64_t k = tc_desc_sw128(stage(i), kStep * 128), ds = tc_desc_plain_mn(stage(i) + C::kKeyBytes, kDsGroup, 128);
#pragma unroll
      for (int x = 0; x < kStep / 16; ++x)
        if (x < steps) tc_mma_ss(tmem, ds + x * (16 * 16 / 16), k + x * (16 * 128 / 16), tc_idesc_bf16(kTile, D, true, true), i > 0 || x > 0);
      tc_commit_warp(empty(i));
    }
    if (ok && count > 0) tc_commit_warp(done);
  } else {
    bool ok = true;
    if (count > 0) {
      ok = warp_wait(done, 0, &abort_flag);
      tc_fence_after();
    }
    // out through the first stages, which no product reads any more
    const int r = threadIdx.x, first = q0 + r - lane;
    const uint32_t to = base + r * 128, from = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    if (p.part0) {
      const int64_t row = (static_cast<int64_t>(it.b) * z.heads + it.head) * z.lq + q0 + r;
      store_row<D>(from, count > 0, p.scale, ok && q0 + r < z.lq, nullptr, p.part0 + it.split * p.elements + row * D);
      ok = false;
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      if (p.part0) break;
      uint32_t o[32];
      __syncwarp();
      if (count > 0) {
        tc_ld32(from + i * 32, o);
        tc_wait_ld();
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0u;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) f[x] = __uint_as_float(o[8 * e + x]) * p.scale;
        const uint4 v = pack8(f);
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                     ::"r"(to + (i >> 1) * (kTile * 128) + ((((i & 1) * 4 + e) ^ (r & 7)) << 4)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                     : "memory");
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0 && ok && first < z.lq) {
#pragma unroll
      for (int c = 0; c < D / 64; ++c) tma_store_4d(&map_dq, to + c * (kTile * 128), c * 64, first, it.head, it.b);
      asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
    }
    __syncwarp();
  }
  __syncwarp();
  if (abort_flag) {
    // Copies still in flight land before shared memory is released.
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tc_dealloc(tmem, 128);
  }
}

// ------------------------------------------------------------------------------------------------ joining the ranges
// dst[row] = sum over splits of part[split][row] in ascending order; rows of D, one of (batch, head, token) order for dq. Four
// elements a thread.
struct SumParams {
  const float* part;
  __nv_bfloat16* dst;
  int splits;
  int64_t elements;
  int d, lq, heads;                      // lq > 0: rows are (batch, head, token), dst has strides
  Strided s;
};
__global__ void __launch_bounds__(256) attention_sum_kernel(const __grid_constant__ SumParams p) {
  after_previous();
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= p.elements) return;
  const float* src = after_previous(p.part) + i;
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float4 v = *reinterpret_cast<const float4*>(src + s * p.elements);
    t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
  }
  __nv_bfloat16* dst = p.dst + i;
  if (p.lq) {
    const int64_t row = i / p.d, bh = row / p.lq, l = row - bh * p.lq, b = bh / p.heads, h = bh - b * p.heads;
    dst = p.dst + b * p.s.b + l * p.s.l + h * p.s.h + (i - row * p.d);
  }
  __nv_bfloat162 o[2] = {__floats2bfloat162_rn(t.x, t.y), __floats2bfloat162_rn(t.z, t.w)};
  *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
}

// Ranges the work of `ctas` CTAs, `items` passes each, is cut into: two CTAs a SM, none with fewer than `least` passes; one where
// there are CTAs enough.
int split_count(int64_t ctas, int64_t items, int64_t least) {
  if (ctas == 0 || ctas >= sm_count()) return 1;
  return static_cast<int>(std::max<int64_t>(1, std::min(ceil_div(2LL * sm_count(), ctas), items / least)));
}
constexpr int64_t kDsBytes = 1ll << 30;
struct Plan {
  int64_t lq_pad, row_floats;            // lse2 and delta
  int key_splits, key_per, query_splits, query_per;
  int64_t key_elements, query_elements, key_items, query_items;
  int64_t units, unit_bytes, at_once;    // key heads of all samples; dS of one; those whose dS is stored at a time, 0: it is not
  explicit Plan(const Shape& s) {
    const int64_t q_tiles = ceil_div(s.lq, kTile), k_tiles = ceil_div(s.lk, kTile), group = s.heads / s.kv_heads;
    lq_pad = q_tiles * kTile;
    row_floats = 2 * s.batch * s.heads * lq_pad;
    key_splits = split_count(k_tiles * s.kv_heads * s.batch, group * q_tiles, 4);
    key_per = static_cast<int>(std::max<int64_t>(1, ceil_div(group * q_tiles, key_splits)));
    key_elements = s.batch * s.lk * s.kv_heads * s.d;
    query_elements = s.batch * s.lq * s.heads * s.d;
    key_items = k_tiles * key_splits * s.kv_heads * s.batch;
    // Above kDsBytes dS is stored and read in parts of the key heads, up to four times as large where fewer parts leave fewer
    // rounds of CTAs half empty ([1, 16384, 16, 128], 2 parts of 8 heads: 6.9 -> 5.6 ms); where the rounds that all parts
    // together take exceed the undivided ones' by a tenth, making dS again is as fast ([1, 32768, 16, 128], 25.5 ms both) or
    // faster (causal, tiles of unequal length, [1, 16384, 16 / 4, 64]: 2.3 instead of 3.5 ms in 2 parts, hence a round more).
    units = s.batch * s.kv_heads;
    unit_bytes = group * q_tiles * k_tiles * kDsTile;
    at_once = unit_bytes && unit_bytes <= 4 * kDsBytes ? units : 0;
    if (at_once && units > kDsBytes / unit_bytes) {
      auto rounds = [&](int64_t heads) { return ceil_div(heads * k_tiles * key_splits, sm_count()) + (s.causal ? 1 : 0); };
      const int64_t least = ceil_div(units, 4 * kDsBytes / unit_bytes);
      int64_t best = rounds(units) + rounds(units) / 10;
      at_once = 0;
      for (int64_t parts = least; parts <= std::min(units, 4 * least); ++parts) {
        const int64_t each = ceil_div(units, parts), full = units / each, cost = full * rounds(each) + rounds(units - full * each);
        if (cost <= best) best = cost, at_once = each;
      }
    }
    query_splits = at_once ? split_count(at_once * group * q_tiles, k_tiles, 8) : split_count(q_tiles * s.heads * s.batch, k_tiles, 4);
    query_per = static_cast<int>(std::max<int64_t>(1, ceil_div(k_tiles, query_splits)));
    query_items = q_tiles * query_splits * s.heads * s.batch;
  }
  int64_t key_part() const { return key_splits > 1 ? key_splits * key_elements : 0; }
  int64_t query_part() const { return query_splits > 1 ? query_splits * query_elements : 0; }
  int64_t floats() const { return (row_floats + 2 * key_part() + query_part() + 63) / 64 * 64; }
  int64_t bytes() const { return floats() * 4 + at_once * unit_bytes; }
};

template <int D>
int launch(const char* who, const CUtensorMap* maps, const Plan& plan, const Shape& s, const RowsParams& rows, BwdParams p, cudaStream_t st) {
  using C = BwdCfg<D>;
  static PerDeviceOnce once;
  const cudaError_t rc = per_device_once(once, [] {
    cudaError_t e = cudaFuncSetAttribute(attention_bwd_keys_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(attention_bwd_dq_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, DqCfg<D>::kSmem);
    return e ? e : cudaFuncSetAttribute(attention_bwd_queries_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  ANIMA_REQUIRE(rc == cudaSuccess, ANIMA_E_CUDA, "%s: cannot reserve %d bytes of shared memory: %s", who, C::kSmem,
                cudaGetErrorString(rc));
  float *ws = const_cast<float*>(p.lse2), *part = p.part0;
  // One CTA a SM goes through all its items; causal, whose items differ in length, four rounds of CTAs, which the GPU hands out
  // as SMs get free ([4, 2047, 16 / 4 heads, 64] 293 -> 270 us; not causal, four rounds cost [8, 4096 x 512] 597 -> 614).
  const int64_t most = (p.z.causal ? 4LL : 1LL) * sm_count();
  auto grid = [&](int64_t items) { return dim3(static_cast<unsigned>(std::min(items, most))); };
  if (plan.row_floats) {
    const dim3 over(static_cast<unsigned>(ceil_div(plan.lq_pad * s.heads, rows_per_cta<D>())), static_cast<unsigned>(s.batch));
    launch_after(attention_rows_kernel<D>, over, dim3(256), 0, st, rows);
    ANIMA_CHECK_LAUNCH(who);
  }
  auto join = [&](const float* from, __nv_bfloat16* to, int splits, int64_t elements, int lq) {
    const SumParams sp = {from, to, splits, elements, D, lq, p.z.heads, p.sdq};
    launch_after(attention_sum_kernel, dim3(static_cast<unsigned>(ceil_div(elements, 1024))), dim3(256), 0, st, sp);
    ANIMA_CHECK_LAUNCH(who);
    return ANIMA_OK;
  };
  p.q_tiles = static_cast<int>(ceil_div(s.lq, kTile));
  p.k_tiles = static_cast<int>(ceil_div(s.lk, kTile));
  BwdParams keys = p, queries = p;
    keys.tiles = p.k_tiles;
  keys.splits = plan.key_splits;
  keys.per_split = plan.key_per;
  keys.elements = plan.key_elements;
  keys.part0 = plan.key_part() ? part : nullptr;
  keys.part1 = plan.key_part() ? part + plan.key_part() : nullptr;
  queries.tiles = p.q_tiles;
  queries.splits = plan.query_splits;
  queries.per_split = plan.query_per;
  queries.elements = plan.query_elements;
  queries.part0 = plan.query_part() ? part + 2 * plan.key_part() : nullptr;
  const bool want_queries = p.dq && plan.query_elements, store = want_queries && plan.at_once;
  const bool want_keys = ((p.dk || p.dv) && plan.key_elements) || store;
  if (store) keys.ds = queries.ds = reinterpret_cast<uint8_t*>(ws + plan.floats());
  const int64_t step = store ? plan.at_once : plan.units, group = s.heads / s.kv_heads;
  auto heads_of = [&](BwdParams& q, int64_t head0, int64_t heads) {
    q.head0 = static_cast<int>(head0);
    q.heads_now = static_cast<int>(heads);
    q.items = static_cast<int>(heads * q.tiles * q.splits);
    q.block = p.z.causal ? static_cast<int>(ceil_div(4LL * sm_count(), q.tiles)) : 1;
  };
  for (int64_t u = 0; want_keys && u < plan.units; u += step) {
    const int64_t now = std::min(step, plan.units - u);
    heads_of(keys, u, now);
    keys.ds_head = queries.ds_head = static_cast<int>(u * group);
    launch_after(attention_bwd_keys_kernel<D>, grid(keys.items), dim3(kThreads), C::kSmem, st, maps[0], maps[1], maps[2], maps[3], keys);
    ANIMA_CHECK_LAUNCH(who);
    if (!store) continue;
    heads_of(queries, u * group, now * group);
    launch_after(attention_bwd_dq_kernel<D>, dim3(static_cast<unsigned>(queries.items)), dim3(DqCfg<D>::kThreads), DqCfg<D>::kSmem, st,
                 maps[4], maps[5], queries);
    ANIMA_CHECK_LAUNCH(who);
  }
  if (want_queries && !plan.at_once) {
    heads_of(queries, 0, plan.units * group);
    queries.last_first = p.z.causal;
    launch_after(attention_bwd_queries_kernel<D>, grid(queries.items), dim3(kThreads), C::kSmem, st, maps[0], maps[1], maps[2], maps[3], queries);
    ANIMA_CHECK_LAUNCH(who);
  }
  if (keys.part0 && want_keys) {
    if (p.dv)
      if (int e = join(keys.part0, p.dv, keys.splits, keys.elements, 0)) return e;
    if (p.dk)
      if (int e = join(keys.part1, p.dk, keys.splits, keys.elements, 0)) return e;
  }
  if (queries.part0 && want_queries) return join(queries.part0, p.dq, queries.splits, queries.elements, p.z.lq);
  return ANIMA_OK;
}

}  // namespace
}  // namespace attn
}  // namespace anima

using namespace anima;

extern "C" int64_t anima_attention_bwd_workspace_bytes(int64_t batch, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads,
                                                       int64_t head_dim, int causal) {
  if (int rc = attn::check_sizes("attention_bwd", batch, lq, lk, heads, kv_heads, head_dim)) return rc;
  const attn::Shape s(batch, lq, lk, heads, kv_heads, head_dim, causal);
  const attn::Plan plan(s);
  ANIMA_REQUIRE(plan.key_items < (1ll << 30) && plan.query_items < (1ll << 30), ANIMA_E_TOO_LARGE, "attention_bwd: too many tiles");
  return plan.bytes();
}

extern "C" int anima_attention_bwd(const void* dout, const int64_t* dout_strides, const void* q, const int64_t* q_strides,
                                   const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                   const void* out, const float* lse, const int32_t* kv_lengths, int64_t batch, int64_t lq,
                                   int64_t lk, int64_t heads, int64_t kv_heads, int64_t head_dim, float scale, int causal,
                                   void* dq, void* dk, void* dv, void* workspace, int64_t workspace_bytes, int32_t* status,
                                   void* stream) {
  const char* who = "attention_bwd";
  const int64_t need = anima_attention_bwd_workspace_bytes(batch, lq, lk, heads, kv_heads, head_dim, causal);
  if (need < 0) return static_cast<int>(need);
  ANIMA_REQUIRE(scale > 0.f && scale < INFINITY, ANIMA_E_ARG, "%s: scale must be positive and finite", who);
  const bool no_q = batch * lq == 0, no_k = batch * lk == 0;
  if (int rc = attn::check_tensor(who, "dout", dout, dout_strides, no_q)) return rc;
  if (int rc = attn::check_tensor(who, "q", q, q_strides, no_q)) return rc;
  if (int rc = attn::check_tensor(who, "k", k, k_strides, no_k)) return rc;
  if (int rc = attn::check_tensor(who, "v", v, v_strides, no_k)) return rc;
  ANIMA_REQUIRE(no_q || (out && lse), ANIMA_E_ARG, "%s: null pointer", who);
  ANIMA_REQUIRE(aligned16(out) && aligned16(dq) && aligned16(dk) && aligned16(dv) && aligned16(workspace), ANIMA_E_ALIGN,
                "%s: tensors must be 16-byte aligned", who);
  ANIMA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), ANIMA_E_WORKSPACE, "%s: workspace of %lld bytes, %lld needed",
                who, (long long)workspace_bytes, (long long)need);
  if (no_q && no_k) return ANIMA_OK;
  const attn::Shape s(batch, lq, lk, heads, kv_heads, head_dim, causal);
  const attn::Plan plan(s);
  attn::Strided sq = attn::strided(q_strides), sdo = attn::strided(dout_strides);
  attn::Strided dense = {lq * heads * head_dim, heads * head_dim, head_dim};
  s.regroup(sq);
  s.regroup(sdo);
  s.regroup(dense);
  float* ws = static_cast<float*>(workspace);
  attn::BwdParams p = {};
  p.z = s.sizes(kv_lengths);
  p.c = scale * attn::kLog2e;
  p.scale = scale;
  p.lse2 = ws;
  p.delta = ws + plan.row_floats / 2;
  p.lq_pad = static_cast<int>(plan.lq_pad);
  p.dq = static_cast<__nv_bfloat16*>(dq);
  p.dk = static_cast<__nv_bfloat16*>(dk);
  p.dv = static_cast<__nv_bfloat16*>(dv);
  p.sdq = dense;
  p.part0 = ws + plan.row_floats;
  p.status = status;
  attn::RowsParams rows = {};
  rows.out = static_cast<const __nv_bfloat16*>(out);
  rows.dout = static_cast<const __nv_bfloat16*>(dout);
  rows.so = dense;
  rows.sdo = sdo;
  rows.lse = lse;
  rows.lse2 = ws;
  rows.delta = ws + plan.row_floats / 2;
  rows.lq = p.z.lq;
  rows.lq_pad = p.lq_pad;
  rows.heads = p.z.heads;
  rows.by_heads = attn::Divisor(s.heads);
  const void* stand_in = no_q ? k : q;
  CUtensorMap maps[6];                   // q, dout, k, v in whole tiles; K by 64 keys, dq by 32 queries
  ANIMA_REQUIRE(attn::bind_context() && attn::encode_heads(&maps[0], q, sq, s.batch, s.lq, s.heads, s.d, stand_in) &&
                    attn::encode_heads(&maps[1], dout, sdo, s.batch, s.lq, s.heads, s.d, stand_in) &&
                    attn::encode_heads(&maps[2], k, attn::strided(k_strides), s.batch, s.lk, s.kv_heads, s.d, stand_in) &&
                    attn::encode_heads(&maps[4], k, attn::strided(k_strides), s.batch, s.lk, s.kv_heads, s.d, stand_in, 64) &&
                    attn::encode_heads(&maps[5], dq ? dq : stand_in, dense, s.batch, s.lq, s.heads, s.d, stand_in, 32) &&
                    attn::encode_heads(&maps[3], v, attn::strided(v_strides), s.batch, s.lk, s.kv_heads, s.d, stand_in),
                ANIMA_E_CUDA, "%s: cuTensorMapEncodeTiled failed (driver entry point missing or bad operand)", who);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return head_dim == 64 ? attn::launch<64>(who, maps, plan, s, rows, p, st) : attn::launch<128>(who, maps, plan, s, rows, p, st);
}
