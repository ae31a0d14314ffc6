// What the attention kernels over the 8-bit cache share: codes and weights as f16, and how partial results are joined.
#pragma once

#include "pi_kv8.cuh"
#include "pi_mma.cuh"

namespace pi_kv8 {

// Weights are stored times 2^12 relative to a running maximum that may lag 2^3 behind: at most 2^15, below the largest f16, and
// precise down to 2^-26 of the largest (both planes: 2^-14), which the many tokens beside one of nearly all the weight need where that
// one adds little to the result.  The maximum is only taken across lanes when a score exceeds it by more.  (A lag of 2^8 with 2^7: 0.2 % faster; of
// 2^2 with 2^13: 0.7 % slower.)
constexpr float kTopWeight = 12.f, kLag = 3.f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two codes as f16: bytes 0 and 1, or 2 and 3, of a word.  int8 (its sign bit flipped): 1024 + (code + 128) in the mantissa, less 1152.
template <int KIND>
__device__ __forceinline__ uint32_t widen(uint32_t w, bool high) {
  if (KIND == PI_INT8) {
    const uint32_t h = __byte_perm(w, 0x64646464u, high ? 0x4342 : 0x4140);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)(high ? w >> 16 : w)));
  return h;
}
template <int KIND>
__device__ __forceinline__ uint32_t unsign(uint32_t w) {
  return KIND == PI_INT8 ? w ^ 0x80808080u : w;
}
// f16 pair of two values and the pair of what is left.
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return pack_f16(a - f.x, b - f.y);
}

// How much a partial result (maximum, sum) counts beside the maximum of all: one that saw nothing does not, one that is not a
// number makes the whole one.
__device__ __forceinline__ float join_factor(float top, float sum, float all) {
  if (sum != sum) return sum;
  return top == -INFINITY ? 0.f : exp2_fast(top - all);
}
__device__ __forceinline__ uint32_t peer_addr(const void* mine, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(pi_mma::smem_addr(mine)), "r"(rank));
  return a;
}
__device__ __forceinline__ float2 peer2(const float2* mine, uint32_t rank) {   // the same variable of another CTA of the cluster
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(peer_addr(mine, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 peer4(const float* mine, uint32_t rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer_addr(mine, rank)) : "memory");
  return v;
}

}  // namespace pi_kv8
