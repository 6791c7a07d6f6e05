// fp32 arithmetic of the operators that are bound by issue: approximate exp2 and reciprocal, and two values in a 64-bit register,
// for which sm_100a's packed instructions do in one issue what two would, with the same rounding.
#pragma once

#include "common.cuh"

namespace qg {

// 2^t to 2^-22, 1 / d to 2^-23; subnormal results are 0.
__device__ __forceinline__ float ex2_approx(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}
__device__ __forceinline__ float rcp_approx(float d) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}

using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 f2_make(float lo, float hi) {
  f32x2 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void f2_get(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 f2_mul(f32x2 a, f32x2 b) {
  f32x2 v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ f32x2 f2_add(f32x2 a, f32x2 b) {
  f32x2 v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ f32x2 f2_sub(f32x2 a, f32x2 b) {
  f32x2 v;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ f32x2 f2_fma(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
// The largest of three absolute values; NaN if one is.
__device__ __forceinline__ float f3_max_abs(float a, float b, float c) {
  float v;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
  return v;
}
template <bool BF16>
__device__ __forceinline__ f32x2 f2_of_half2(uint32_t w) {
  if constexpr (BF16) return f2_make(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return f2_make(f.x, f.y);
}

}  // namespace qg
