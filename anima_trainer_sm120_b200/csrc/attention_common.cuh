// What the attention kernels share: sizes, key ranges, tensor maps, checks of arguments.
//
//   s[i, j] = scale * q[i] . k[j],  p[i, j] = exp(s[i, j]) / sum over seen j' of exp(s[i, j']),  out[i] = sum_j p[i, j] v[j]
//   lse[i]  = ln(sum_j exp(s[i, j]))
//   delta[i] = out[i] . dout[i],    ds[i, j] = p[i, j] (dout[i] . v[j] - delta[i])
//   dq[i] = scale * sum_j ds[i, j] k[j],  dk[j] = scale * sum_i ds[i, j] q[i],  dv[j] = sum_i p[i, j] dout[i]
//
// A key is seen by a query if it lies before the sample's length and, causal, at most lk - lq places after the query. A
// query that sees no key has output 0 and lse -inf and takes no part in the gradients. kv_heads may divide heads.
#pragma once

#include <cmath>

#include "f32x2.cuh"
#include "tc_util.cuh"

namespace anima {
namespace attn {

constexpr int kTile = 128;               // rows of a tile, queries or keys
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Sizes {
  int lq, lk, heads, kv_heads, group;    // group: query heads a key head serves
  int causal;
  const int32_t* lengths;
};

__device__ __forceinline__ int keys_of(const Sizes& z, int b) { return z.lengths ? max(0, min(z.lk, z.lengths[b])) : z.lk; }
// keys that query i of a sample with n keys sees are 0 .. limit - 1
__device__ __forceinline__ int key_limit(const Sizes& z, int n, int i) { return z.causal ? max(0, min(n, i + z.lk - z.lq + 1)) : n; }

// 2^x on the special-function unit, of which an SM finishes 16 a cycle
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^x on the multiply-add pipes, two values at once: x = n + f, n the nearest integer, |f| <= 1/2; 2^f by a polynomial of degree
// 4 with value 1 at 0, fitted to the least relative error (Lawson's weighted least squares; 2.9e-6 in fp32 arithmetic,
// which the rounding of the result to bf16 exceeds a thousand times). Adding 1.5 2^23 + 127 rounds to n and leaves n + 127 in
// the low bits, the exponent of 2^n. Below -126.5 that is 0 and so is the result; NaN stays NaN. x at most 127.
__device__ __forceinline__ f2 exp2_poly(f2 x) {
  float lo, hi;
  asm("max.NaN.f32 %0, %1, 0fC2FE0000;" : "=f"(lo) : "f"(f2_lo(x)));     // -127
  asm("max.NaN.f32 %0, %1, 0fC2FE0000;" : "=f"(hi) : "f"(f2_hi(x)));
  x = f2_make(lo, hi);
  const f2 t = f2_add(x, f2_dup(12583039.f));
  const f2 f = f2_fma(f2_add(t, f2_dup(-12583039.f)), f2_dup(-1.f), x);
  f2 p = f2_fma(f, f2_dup(0.009582852944731712f), f2_dup(0.055906426161527634f));
  p = f2_fma(p, f, f2_dup(0.24024099111557007f));
  p = f2_fma(p, f, f2_dup(0.6931241750717163f));
  p = f2_fma(p, f, f2_dup(1.f));
  const uint32_t a = static_cast<uint32_t>(t), b = static_cast<uint32_t>(t >> 32);
  return f2_mul(p, f2_make(__uint_as_float(a << 23), __uint_as_float(b << 23)));
}
__device__ __forceinline__ f2 exp2_pair(f2 x) { return f2_make(exp2_approx(f2_lo(x)), exp2_approx(f2_hi(x))); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A wait of a whole warp with one answer for all its lanes.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}
// Every item takes the stages of a ring from the first on, so that where a pass finds its operands follows from its number in
// the item alone, which the compiler keeps in uniform registers (with stages counted through all items the products' descriptors
// went through ordinary ones: 72 instead of 20 cycles an instruction). What carries over from item to item, the phases of the
// barriers, is one bit each.
__device__ __forceinline__ uint32_t phase_of(uint32_t& bits, int s) {      // of the next completion of barrier s
  const uint32_t now = (bits >> s) & 1u;
  bits ^= 1u << s;
  return now;
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
               ::"l"(map), "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
// n / d for n < 2^31 with one multiplication, rounded up as by Granlund and Montgomery: the hardware has no division of integers,
// and the four of an item's place made a short call 0.3 us longer.
struct Divisor {
  uint32_t mul = 0, shift = 0;
  Divisor() = default;
  explicit Divisor(int64_t d) {
    while ((1ll << shift) < d) ++shift;
    mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ int of(int n) const { return static_cast<int>((__umulhi(n, mul) + n) >> shift); }
};

// ROWS tokens of one head: D / 64 chunks of ROWS x 128 bytes (swizzled), one behind the other. Tokens behind the last one arrive
// as zeros.
template <int D, int ROWS>
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap* map, uint32_t bar, int token, int head, int b) {
#pragma unroll
  for (int c = 0; c < D / 64; ++c) tma_load_4d(dst + c * (ROWS * 128), map, bar, c * 64, token, head, b);
}
template <int D>
constexpr uint32_t tile_bytes() { return kTile * D * 2; }

// Rows first .. last - 1 of a tile in shared memory (chunks `chunk` bytes apart) become zero (a whole warp): what TMA brought from
// behind a sample's length may be NaN, which a product with a probability of 0 would spread.
template <int D>
__device__ __forceinline__ void zero_rows(uint32_t tile, uint32_t chunk, int first, int last) {
  const int lane = threadIdx.x & 31;
  for (int i = first * 8 + lane; i < last * 8; i += 32) {
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(tile + c * chunk + i * 16), "r"(0) : "memory");
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

// ------------------------------------------------------------------------------------------------ host side
struct Strided {                         // element strides of (batch, token, head); the head vector is dense
  int64_t b, l, h;
};

inline int check_sizes(const char* who, int64_t batch, int64_t lq, int64_t lk, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  ANIMA_REQUIRE(batch >= 0 && lq >= 0 && lk >= 0 && heads > 0 && kv_heads > 0, ANIMA_E_ARG, "%s: bad sizes", who);
  ANIMA_REQUIRE(head_dim == 64 || head_dim == 128, ANIMA_E_UNSUPPORTED, "%s: head_dim=%lld is not supported (64 or 128)", who,
                (long long)head_dim);
  ANIMA_REQUIRE(heads % kv_heads == 0, ANIMA_E_SHAPE, "%s: heads=%lld is not a multiple of kv_heads=%lld", who,
                (long long)heads, (long long)kv_heads);
  ANIMA_REQUIRE(batch < 65536 && heads < 65536 && lq < (1ll << 30) && lk < (1ll << 30) && heads * lq < (1ll << 30) && batch * heads * lq < (1ll << 40),
                ANIMA_E_TOO_LARGE, "%s: too large", who);
  return ANIMA_OK;
}
inline int check_tensor(const char* who, const char* name, const void* p, const int64_t* s, bool empty) {
  ANIMA_REQUIRE(s, ANIMA_E_ARG, "%s: strides of %s are missing", who, name);
  ANIMA_REQUIRE(p || empty, ANIMA_E_ARG, "%s: null pointer (%s)", who, name);
  ANIMA_REQUIRE(s[0] >= 0 && s[1] >= 0 && s[2] >= 0, ANIMA_E_ARG, "%s: negative stride of %s", who, name);
  ANIMA_REQUIRE(aligned16(p) && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0, ANIMA_E_ALIGN,
                "%s: %s must be 16-byte aligned, its strides multiples of 8 elements", who, name);
  ANIMA_REQUIRE(s[0] < (1ll << 38) && s[1] < (1ll << 38) && s[2] < (1ll << 38), ANIMA_E_TOO_LARGE, "%s: strides of %s are too large",
                who, name);
  return ANIMA_OK;
}
inline Strided strided(const int64_t* s) { return {s[0], s[1], s[2]}; }

// Sizes of a call as the kernels see it. One query token a sample: the heads that share a key head become its tokens (all
// keys of the sample are seen, so nothing depends on a query's place), and each key is read once for all of them.
struct Shape {
  int64_t batch, lq, lk, heads, kv_heads, d;
  int causal;
  bool regrouped;
  Shape(int64_t batch, int64_t lq_, int64_t lk, int64_t heads_, int64_t kv_heads, int64_t d, int causal_)
      : batch(batch), lq(lq_ == 1 ? heads_ / kv_heads : lq_), lk(lk), heads(lq_ == 1 ? kv_heads : heads_), kv_heads(kv_heads), d(d),
        causal(lq_ == 1 ? 0 : causal_ != 0), regrouped(lq_ == 1) {}
  void regroup(Strided& s) const {       // of a tensor with the queries' heads
    if (!regrouped) return;
    s.l = s.h;
    s.h = s.l * lq;
  }
  Sizes sizes(const int32_t* lengths) const {
    return {static_cast<int>(lq), static_cast<int>(lk), static_cast<int>(heads), static_cast<int>(kv_heads),
            static_cast<int>(heads / kv_heads), causal, lengths};
  }
};

// A thread that has made no runtime call yet (autograd's worker, say) has no current context, without which the driver
// refuses to encode a tensor map; making its device current again binds one.
inline bool bind_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}

// Tensor map of a (batch, token, head, D) bf16 tensor, boxes of `rows` tokens x 64 elements. A tensor without elements gets the
// map of one that is never read (`stand_in`: any valid address).
inline bool encode_heads(CUtensorMap* map, const void* p, const Strided& s, int64_t batch, int64_t len, int64_t heads, int64_t d,
                         const void* stand_in, uint32_t rows = kTile) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const bool none = batch * len == 0;
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)std::max<int64_t>(1, len), (cuuint64_t)heads, (cuuint64_t)std::max<int64_t>(1, batch)};
  // the stride of a dimension of one element is not used; any valid one will do
  auto bytes = [&](int64_t n, int64_t stride) { return (cuuint64_t)(n > 1 && !none ? stride * 2 : 2 * d); };
  const cuuint64_t strides[3] = {bytes(len, s.l), bytes(heads, s.h), bytes(batch, s.b)};
  const cuuint32_t box[4] = {64, rows, 1, 1}, step[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(none ? stand_in : p), dims, strides, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace attn
}  // namespace anima
