// Head vectors of q / k kept in lanes: the norm weight folded into a token's rotation, and the copy ring that feeds the lanes.
#pragma once

#include "f32x2.cuh"

namespace anima {
namespace headvec {

// Eight lanes own one token and walk its heads. Lane l holds elements 8l..8l+7 and 64+8l..64+8l+7 (two 16-byte
// accesses), so an element and its rotate-half partner are in the same lane: a vector costs three shuffles (its sum)
// instead of four plus one per element, which bound the half-warp form that held 8 consecutive elements per lane.
// With the norm weight folded into the token's rotation, held in registers and reused by every head,
//   a1 = w1 c1, b1 = w2 s1, a2 = w2 c2, b2 = w1 s2   (1 / 2: the halves; s, c: the tables)
//   out1 = rstd (x1 a1 - x2 b1),  out2 = rstd (x2 a2 + x1 b2)
//   gw1  = g1 a1 + g2 b2,         gw2  = g2 a2 - g1 b1                (the gradient of x / rms, backward)
// fp32 in pairs. [8, 4096, 16, 128]: forward 57.6 -> 46.2 us (5810 GB/s), backward 80.6 -> 64.4 (6250 GB/s).
struct Rotation {
  f2 a1[4], b1[4], a2[4], b2[4];   // without rotary: a1 = w1, a2 = w2
};

template <bool WBF16>
__device__ __forceinline__ void load8(const void* p, int at, f2 (&v)[4]) {
  if (WBF16) {
    const uint4 r = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + at);
    v[0] = f2_of_bf16(r.x); v[1] = f2_of_bf16(r.y); v[2] = f2_of_bf16(r.z); v[3] = f2_of_bf16(r.w);
  } else {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 lo = q[0], hi = q[1];
    v[0] = f2_make(lo.x, lo.y); v[1] = f2_make(lo.z, lo.w); v[2] = f2_make(hi.x, hi.y); v[3] = f2_make(hi.z, hi.w);
  }
}

template <int D, bool ROPE, bool WBF16>
__device__ __forceinline__ void load_rotation(Rotation& r, const void* w, const float* cos_tab, const float* sin_tab,
                                              int64_t pos, int l) {
  f2 w1[4], w2[4];
  load8<WBF16>(w, l * 8, w1);
  load8<WBF16>(w, D / 2 + l * 8, w2);
  if (ROPE) {
    load8<false>(cos_tab + pos * D, l * 8, r.a1);
    load8<false>(cos_tab + pos * D, D / 2 + l * 8, r.a2);
    load8<false>(sin_tab + pos * D, l * 8, r.b1);
    load8<false>(sin_tab + pos * D, D / 2 + l * 8, r.b2);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (ROPE) {
      r.a1[e] = f2_mul(w1[e], r.a1[e]);
      r.a2[e] = f2_mul(w2[e], r.a2[e]);
      r.b1[e] = f2_mul(w2[e], f2_mul(r.b1[e], f2_dup(-1.f)));   // enters with its sign
      r.b2[e] = f2_mul(w1[e], r.b2[e]);
    } else {
      r.a1[e] = w1[e];
      r.a2[e] = w2[e];
    }
  }
}

// The loads run ahead of the arithmetic through a ring in shared memory filled with cp.async: each thread copies
// exactly the 16-byte chunks it reads itself (no barrier, no registers), kAhead heads ahead. With loads unrolled into
// registers the 128 registers a thread leave 16 warps and about 32 KB in flight a SM: 5.0 TB/s.
template <int CHUNKS, int STAGES, int THREADS>   // 16-byte chunks of one head, ring slots, threads a CTA
struct Ring {
  uint32_t base;
  __device__ __forceinline__ Ring(void* smem) : base(static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + threadIdx.x * 16) {}
  __device__ __forceinline__ uint32_t at(int slot, int c) const { return base + (slot * CHUNKS + c) * THREADS * 16; }
  __device__ __forceinline__ void copy(int slot, int c, const void* src) const {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at(slot, c)), "l"(src) : "memory");
  }
  __device__ __forceinline__ static void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  __device__ __forceinline__ static void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory"); }
  __device__ __forceinline__ uint4 read(int slot, int c) const {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at(slot, c)));
    return v;
  }
};
__device__ __forceinline__ void widen(const uint4& v, f2 (&f)[4]) {
  f[0] = f2_of_bf16(v.x); f[1] = f2_of_bf16(v.y); f[2] = f2_of_bf16(v.z); f[3] = f2_of_bf16(v.w);
}
__device__ __forceinline__ uint4 narrow(const f2 (&f)[4]) {
  return make_uint4(bf16_of_f2(f[0]), bf16_of_f2(f[1]), bf16_of_f2(f[2]), bf16_of_f2(f[3]));
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v, unsigned mask) {   // over the token's lanes
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
  return v;
}

}  // namespace headvec
}  // namespace anima
