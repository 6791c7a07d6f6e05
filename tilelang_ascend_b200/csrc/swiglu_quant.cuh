// SiLU-gated product and per-token quantiser in one pass, for sm_100a: bf16 / f16 [M, 2 F] (gate | up) -> int8 [M, F] + fp32 scale [M].
//
//   a = g / (1 + exp(-g)) * u          s = RN32(max(max|a|, 1e-4) / 127)  (round_scale: the power of two not below it)
//   y = the integer nearest to a / s
//
// y and s are those of the exact a, so that they depend on no implementation's rounding of exp: fp32 values decide all but
// the elements next to a border, which are taken again in fp64 - the candidates for the row's largest value, a few per row, and the
// quotients within SQ_NEAR of a half, about one in 3000.  (For |u| < 1e26 where g < -80: below that exp leaves fp32's normal range.)
//
// 4 F bytes in and F out per row.
#pragma once

#include "act_quant.cuh"
#include "common.cuh"

namespace qg {

struct SwigluQuantParams {
  const uint4* X;   // [M, 2 F]
  int8_t* Y;        // [M, F]
  float* S;         // [M]
  long long M;
  int F;            // multiple of 8
  int round_scale;
};

// What fp32 makes of a: exp to 2 ulp, the quotient to 2, and three roundings, 6.6e-7 in all; times 127 with the two roundings of the
// quotient by s, 9.8e-5 of a step.
constexpr float SQ_NEAR = 1.5e-4f;
constexpr float SQ_TOP = 1.0f - 0x1p-18f;  // whoever is this near to the fp32 maximum may be the largest

__device__ __forceinline__ float sq_gate(float g, float u) {
  const float e = expf(-fabsf(g));  // at most 1, so that nothing overflows
  return __fdividef(g < 0.0f ? g * e : g, 1.0f + e) * u;
}
__device__ __forceinline__ double sq_gate64(float g, float u) { return (double)g / (1.0 + exp(-(double)g)) * (double)u; }

template <bool BF16>
__device__ __forceinline__ float sq_element(const void* p, long long i) {
  uint16_t h;
  asm volatile("ld.global.u16 %0, [%1];" : "=h"(h) : "l"(static_cast<const uint16_t*>(p) + i));
  if constexpr (BF16) return __uint_as_float((uint32_t)h << 16);
  return __half2float(__ushort_as_half(h));
}

// |a| of the elements of chunk c that may be the row's largest, in fp64.
template <bool BF16>
__device__ __noinline__ double sq_largest64(const uint4* x, int chunks, int c, float from) {
  double best = 0.0;
  for (int i = 0; i < 8; ++i) {
    const float g = sq_element<BF16>(x, 8ll * c + i), u = sq_element<BF16>(x, 8ll * (chunks + c) + i);
    if (fabsf(sq_gate(g, u)) >= from) best = fmax(best, fabs(sq_gate64(g, u)));
  }
  return best;
}
// The codes of the marked elements of chunk c in fp64.
template <bool BF16>
__device__ __noinline__ uint2 sq_codes64(const uint4* x, int chunks, int c, float scale, uint32_t marked, uint2 codes) {
  for (int i = 0; i < 8; ++i) {
    if (!((marked >> i) & 1u)) continue;
    const float g = sq_element<BF16>(x, 8ll * c + i), u = sq_element<BF16>(x, 8ll * (chunks + c) + i);
    const double q = fmin(fmax(rint(sq_gate64(g, u) / (double)scale), -127.0), 127.0);
    const uint32_t code = (uint32_t)(int)q & 0xffu, at = 8u * (i & 3);
    uint32_t& w = i < 4 ? codes.x : codes.y;
    w = (w & ~(0xffu << at)) | (code << at);
  }
  return codes;
}

template <bool BF16>
__device__ __forceinline__ void sq_gate8(const uint4& g, const uint4& u, float (&a)[8]) {
  float gf[8], uf[8];
  aq_unpack8(g, BF16, gf);
  aq_unpack8(u, BF16, uf);
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = sq_gate(gf[i], uf[i]);
}

template <int TPR, int KEEP, bool BF16>
__global__ void __launch_bounds__(aq_block(TPR)) swiglu_quant_kernel(const SwigluQuantParams p) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int ROWS = aq_block(TPR) / TPR;
  constexpr int WPR = TPR / 32;  // warps per row
  __shared__ uint32_t red[aq_block(TPR) / 32];
  __shared__ unsigned long long largest[ROWS];
  const int t = threadIdx.x % TPR;
  const int r = threadIdx.x / TPR;
  const int warp = threadIdx.x >> 5;
  const long long row = (long long)blockIdx.x * ROWS + r;
  const bool live = row < p.M;
  const int chunks = p.F >> 3;
  const uint4* x = p.X + (live ? row : 0) * 2 * chunks;
  if (t == 0) largest[r] = 0ull;

  float a[KEEP][8];
  uint32_t m = 0;  // |a| as an integer: the same order, with inf and NaN on top
  auto take = [&](int c, float (&v)[8]) {
    sq_gate8<BF16>(ld_written(x + c), ld_written(x + chunks + c), v);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  };
  if (live) {
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (t + i * TPR < chunks) take(t + i * TPR, a[i]);
    for (int c = t + KEEP * TPR; c < chunks; c += TPR) {
      float v[8];
      take(c, v);
    }
  }
  const uint32_t own = m;
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) red[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WPR; ++w) m = max(m, red[r * WPR + w]);
  const bool finite = m < 0x7f800000u;
  const float from = __uint_as_float(m) * SQ_TOP;
  if (live && finite && m != 0 && __uint_as_float(own) >= from) {
    double best = 0.0;
    for (int c = t; c < chunks; c += TPR) best = fmax(best, sq_largest64<BF16>(x, chunks, c, from));
    atomicMax(&largest[r], (unsigned long long)__double_as_longlong(best));
  }
  __syncthreads();
  float scale = (float)(fmax(__longlong_as_double((long long)largest[r]), 1e-4) / 127.0);
  if (p.round_scale) scale = aq_pow2_ceil(scale);
  if (!finite) scale = __uint_as_float(m);  // inf or NaN: it stays one
  if (!live) return;
  if (t == 0) p.S[row] = scale;
  const float rcp = __frcp_rn(scale);
  uint2* y = reinterpret_cast<uint2*>(p.Y) + row * chunks;
  auto store = [&](int c, const float (&v)[8]) {
    const float MAGIC = 12582912.0f;  // 1.5 * 2^23: the sum's low bits are the nearest integer
    float f[8];
    uint32_t marked = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = v[i] * rcp;
      f[i] = q + MAGIC;
      if (fabsf(q - (f[i] - MAGIC)) > 0.5f - SQ_NEAR) marked |= 1u << i;
    }
    uint2 codes = make_uint2(aq_pack4(f), aq_pack4(f + 4));
    if (marked) codes = sq_codes64<BF16>(x, chunks, c, scale, marked, codes);
    y[c] = codes;
  };
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (t + i * TPR < chunks) store(t + i * TPR, a[i]);
  for (int c = t + KEEP * TPR; c < chunks; c += TPR) {
    float v[8];
    sq_gate8<BF16>(ld_written(x + c), ld_written(x + chunks + c), v);
    store(c, v);
  }
}

}  // namespace qg
