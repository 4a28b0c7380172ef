// What the append and the attention over the 8-bit cache share: rotation, rounding, codes.
#pragma once
#include "kv_cache8.h"
#include "ptx.cuh"

namespace ccl {
namespace kv8 {

constexpr float kLeastScale = 9.094947017729282e-13f;  // 2^-40: a block of zeros divides by something

__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Products and their sum are rounded one by one, as separate fp32 operations would (a contracted multiply-add differs in the last
// bit, which a rounding to bf16 and then to 8 bits can turn into a whole step).
__device__ __forceinline__ void rotate(float a, float b, float c, float s, float& x, float& y) {
  x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  y = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
}

template <bool INT8>
__device__ __forceinline__ float scale_of(float amax) {
  const float s = __fdiv_rn(amax, INT8 ? 127.f : 448.f);
  return s < kLeastScale ? kLeastScale : s;  // (a NaN stays)
}
// A scale that many values are divided by. With the correctly rounded reciprocal r, q = x r is corrected by its residual to the correctly
// rounded quotient, q + (x - q s) r (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990):
// three operations a value where a division is a dozen. (A quotient so small that the residual is not exact has the code zero anyhow.)
struct Divisor {
  float s, r;  // r 0: s is not finite, and is divided by
};
__device__ __forceinline__ Divisor divisor(float s) { return {s, s < INFINITY ? __frcp_rn(s) : 0.f}; }
__device__ __forceinline__ float over(float x, const Divisor& d) {
  const float q = x * d.r;
  return d.r == 0.f ? __fdiv_rn(x, d.s) : fmaf(fmaf(-q, d.s, x), d.r, q);
}
// Four values over one scale -> four codes.
template <bool INT8>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, const Divisor& scale) {
  a = over(a, scale);
  b = over(b, scale);
  c = over(c, scale);
  d = over(d, scale);
  if constexpr (INT8) {
    auto q = [](float x) { return (uint32_t)(max(-127, min(127, __float2int_rn(x))) & 0xff); };
    return q(a) | (q(b) << 8) | (q(c) << 16) | (q(d) << 24);
  } else {
    uint16_t l, h;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(l) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(d), "f"(c));
    return (uint32_t)l | ((uint32_t)h << 16);
  }
}
// The largest magnitude of two packed bf16 values and what was seen before, as bf16 bits (a NaN is larger than everything).
__device__ __forceinline__ uint32_t amax_bits(uint32_t seen, uint32_t w) {
  w &= 0x7fff7fffu;
  return max(seen, max(w & 0xffffu, w >> 16));
}
__device__ __forceinline__ float bits_f(uint32_t b) { return __uint_as_float(b << 16); }

}  // namespace kv8
}  // namespace ccl
