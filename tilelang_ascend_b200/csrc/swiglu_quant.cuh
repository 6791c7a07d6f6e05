// SiLU-gated product and per-token quantiser in one pass, for sm_100a: bf16 / f16 [M, 2 F] (gate | up) -> int8 [M, F] + fp32 scale [M].
//
//   a = g / (1 + exp(-g)) * u          s = RN32(max(max|a|, 1e-4) / 127)  (round_scale: the power of two not below it)
//   y = the integer nearest to a / s
//
// y and s are those of the exact a, so that they depend on no implementation's rounding of exp.  fp32 values decide all but
// the elements next to a border, which are taken again in fp64: the candidates for the row's largest value, one or two per row, and the
// quotients that lie as near to n + 1/2 as fp32 may be wrong, one in 1000 or so.
//
// What fp32 makes of a, relative: 2^-22 by ex2.approx, |g| 7.5e-8 by the rounding of its argument where g < 0 (where g > 0 the factor
// e / (1 + e) takes it down to 2e-8), 2^-24 by the sum, 2^-23 by rcp.approx, 2^-23 by two products: 5.4e-7 + 7.5e-8 max(0, -g).  The
// quotient by s adds 2.4e-7.
//
// bf16 has products that fp32 has not: below g = -87 its sigmoid is 0, which |u| of 2^96 and more brings back into the range of codes, and
// |g u| goes up to 1e77, whose 127th part may still be an fp32 number.  Both show in what a row's reductions give anyway (the lowest gate, a
// maximum that is no number); such a row is looked through again and, where it has to be, done in fp64 as a whole.
//
// 4 F bytes in and F out per row.  A row is held in registers as fp32 between its maximum and its codes.  Pairs of values go through
// the packed fp32 instructions; two MUFU operations per element are the next bound behind memory.
#pragma once

#include <type_traits>

#include "act_quant.cuh"
#include "common.cuh"
#include "packed_float.cuh"

namespace qg {

struct SwigluQuantParams {
  const uint4* X;   // [M, 2 F]
  int8_t* Y;        // [M, F]
  float* S;         // [M]
  long long M;
  int F;            // multiple of 8
  int round_scale;
};

// --------------------------------------------------------------------------------------------------- a in fp32 and fp64
__device__ __forceinline__ f32x2 sq_gate(f32x2 g, f32x2 u) {
  const float L = -1.4426950408889634f;  // -log2(e)
  float t0, t1, d0, d1;
  f2_get(f2_mul(g, f2_make(L, L)), t0, t1);
  f2_get(f2_add(f2_make(ex2_approx(t0), ex2_approx(t1)), f2_make(1.0f, 1.0f)), d0, d1);
  return f2_mul(f2_mul(g, f2_make(rcp_approx(d0), rcp_approx(d1))), u);
}
template <bool BF16>
__device__ __forceinline__ float sq_float(uint32_t bits) {
  if constexpr (BF16) return __uint_as_float(bits << 16);
  return __half2float(__ushort_as_half((unsigned short)bits));
}
template <bool BF16>
__device__ __forceinline__ float sq_element(const uint4* p, int i) {
  return sq_float<BF16>(*(reinterpret_cast<const volatile uint16_t*>(p) + i));
}
// In fp64, to 2 or 3 of its ulps (for g > -100): exp(-g) = 2^k exp(r), |r| <= ln 2 / 2, by its Taylor series (the first term left out is
// below 5e-18), then g u times a reciprocal refined by Newton's steps.  45 instructions in a chain, without a branch or a call, because a
// whole row waits for them; exp() and a division are three times as many.
__device__ __forceinline__ double sq_gate64(float g, float u) {
  constexpr double LN2_HI = 0x1.62e42ffp-1, LN2_LO = -0x1.718432a1b0e26p-35;  // ln 2 to 30 bits, and the rest: k LN2_HI is exact
  const double x = fmin(fmax(-(double)g, -700.0), 700.0);
  const double shifted = fma(x, 1.4426950408889634, 0x1.8p52);  // the low bits are the nearest integer k
  const double k = shifted - 0x1.8p52;
  const double r = fma(k, -LN2_LO, fma(k, -LN2_HI, x));
  double e = 1.0 / 6227020800.0;
  e = fma(e, r, 1.0 / 479001600.0);
  e = fma(e, r, 1.0 / 39916800.0);
  e = fma(e, r, 1.0 / 3628800.0);
  e = fma(e, r, 1.0 / 362880.0);
  e = fma(e, r, 1.0 / 40320.0);
  e = fma(e, r, 1.0 / 5040.0);
  e = fma(e, r, 1.0 / 720.0);
  e = fma(e, r, 1.0 / 120.0);
  e = fma(e, r, 1.0 / 24.0);
  e = fma(e, r, 1.0 / 6.0);
  e = fma(e, r, 0.5);
  e = fma(e, r, 1.0);
  e = fma(e, r, 1.0);
  e = __hiloint2double(__double2hiint(e) + (__double2loint(shifted) << 20), __double2loint(e));
  const double d = 1.0 + e, n = (double)g * (double)u;  // (the product of two 16-bit values is exact)
  double y;
  asm("rcp.approx.ftz.f64 %0, %1;" : "=d"(y) : "d"(d));
  y = fma(fma(-d, y, 1.0), y, y);
  y = fma(fma(-d, y, 1.0), y, y);
  y = fma(fma(-d, y, 1.0), y, y);
  const double q = n * y;
  return fma(fma(-d, q, n), y, q);
}

template <bool BF16>
__device__ __forceinline__ void sq_gate8(const uint4& g, const uint4& u, f32x2 (&a)[4]) {
  const uint32_t gw[4] = {g.x, g.y, g.z, g.w}, uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = sq_gate(f2_of_half2<BF16>(gw[i]), f2_of_half2<BF16>(uw[i]));
}

// The elements of a chunk that are marked, in fp64: the largest |a| of them ...
template <bool BF16>
__device__ __noinline__ double sq_largest64(const uint4* gp, const uint4* up, uint32_t marked) {
  double best = 0.0;
  for (; marked != 0; marked &= marked - 1) {
    const int i = __ffs(marked) - 1;
    best = fmax(best, fabs(sq_gate64(sq_element<BF16>(gp, i), sq_element<BF16>(up, i))));
  }
  return best;
}
// ... and their codes, which take the place of those that fp32 gave.
template <bool BF16>
__device__ __noinline__ uint2 sq_codes64(const uint4* gp, const uint4* up, float scale, uint32_t marked, uint2 codes) {
  for (; marked != 0; marked &= marked - 1) {
    const int i = __ffs(marked) - 1;
    const double q = sq_gate64(sq_element<BF16>(gp, i), sq_element<BF16>(up, i)) / (double)scale;
    const uint32_t code = (uint32_t)__double2int_rn(fmin(fmax(q, -127.0), 127.0)) & 0xffu, at = 8u * (i & 3);
    uint32_t& w = i < 4 ? codes.x : codes.y;
    w = (w & ~(0xffu << at)) | (code << at);
  }
  return codes;
}

// A row whose lowest gate or largest product says that fp32 may not hold its products: where its inputs are numbers, and one of them is
// large enough for that, every element again in fp64.  An infinite scale (max|a| / 127 beyond fp32) gives codes of 0.
template <int TPR>
__device__ __noinline__ void sq_far_row(const uint4* x, int chunks, int t, int round_scale, uint32_t* largest, uint2* y, float* s) {
  uint32_t m2 = 0;  // largest magnitude, as bits of bf16
  for (int c = t; c < chunks; c += TPR) {
    const uint4 g = ld_written(x + c), u = ld_written(x + chunks + c);
    const uint32_t M = 0x7fff7fffu;
    m2 = __vimax3_u16x2(__vimax3_u16x2(m2, g.x & M, g.y & M), g.z & M, g.w & M);
    m2 = __vimax3_u16x2(__vimax3_u16x2(m2, u.x & M, u.y & M), u.z & M, u.w & M);
  }
  const uint32_t most = max(m2 & 0xffffu, m2 >> 16);
  int no_number = most >= 0x7f80u, far = most >= 0x5f80u;  // 0x5f80: 2^64
  if constexpr (TPR > 32) {
    no_number = __syncthreads_or(no_number);
    far = __syncthreads_or(far);
  } else {
    no_number = __any_sync(0xffffffffu, no_number);
    far = __any_sync(0xffffffffu, far);
  }
  if (no_number || !far) return;
  double best = 1e-4;
  for (int c = t; c < chunks; c += TPR) best = fmax(best, sq_largest64<true>(x + c, x + chunks + c, 0xffu));
  uint32_t bits = __float_as_uint((float)(best * (1.0 / 127.0)));
  if constexpr (TPR > 32) {
    atomicMax(largest, bits);
    __syncthreads();
    bits = *largest;
  } else {
    bits = __reduce_max_sync(0xffffffffu, bits);
  }
  float scale = __uint_as_float(bits);
  if (round_scale) scale = aq_pow2_ceil(scale);
  if (t == 0) *s = scale;
  for (int c = t; c < chunks; c += TPR) y[c] = sq_codes64<true>(x + c, x + chunks + c, scale, 0xffu, make_uint2(0u, 0u));
}

// TPR threads share a row, KEEP chunks of eight elements of it in each one's registers; longer rows are computed again for their codes.
// The blocks are persistent: the next row's loads are issued when this one's values are in fp32, and are in flight while its
// maximum is settled and its codes are stored.
__host__ __device__ constexpr int sq_block(int tpr) { return tpr == 32 ? 128 : tpr; }
// Blocks per SM that the registers have to allow: 384 threads where a warp has a row to itself, otherwise 512 at five chunks and more,
// so that another row goes on while one waits for its two barriers.  us, 128 registers / the compiler's 168 - 180: 5000 x 7168
// 43.5 / 46.5, 4000 x 14336 81 / 100, but 32768 x 2048 64.5 / 62.9.
__host__ __device__ constexpr int sq_min_blocks(int tpr, int keep) {
  const int threads = keep > 4 ? (tpr == 32 ? 384 : 512) : keep > 2 ? 640 : keep == 2 ? 768 : 1024;
  return threads / sq_block(tpr) > 0 ? threads / sq_block(tpr) : 1;
}
__host__ __device__ constexpr int sq_smem_bytes(int tpr, int keep) { return keep * 32 * sq_block(tpr); }
template <int TPR, int KEEP, bool BF16>
__global__ void __launch_bounds__(sq_block(TPR), sq_min_blocks(TPR, KEEP)) swiglu_quant_kernel(const SwigluQuantParams p) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int ROWS = sq_block(TPR) / TPR;
  constexpr int WPR = TPR / 32;  // warps per row
  static_assert(WPR == 1 || ROWS == 1, "barriers are of the whole block");
  // Eight chunks in 128 registers: a row's number is 32 bits wide (2^31 rows of 3592 elements and more are beyond any memory), the
  // addresses are not kept.  8000 x 4096 34.0 us, otherwise 35.8.
  constexpr bool TIGHT = KEEP == 8 && TPR > 32;
  using Row = std::conditional_t<TIGHT, int, long long>;
  __shared__ uint32_t red[2][WPR];
  __shared__ uint32_t largest[2];  // scales as bits, of this row and the next one
  const int t = threadIdx.x % TPR;
  const int warp = threadIdx.x >> 5;
  const int chunks = p.F >> 3;
  const Row step = (Row)gridDim.x * ROWS;
  Row row = (Row)blockIdx.x * ROWS + threadIdx.x / TPR;
  if (WPR > 1 && t == 0) largest[0] = 0u;
  // a thread copies its own chunks into its own slots, so that no barrier is needed to read them
  extern __shared__ uint4 sq_slots[];
  uint4* slot = sq_slots + threadIdx.x;  // gate chunk i: slot[2 i block], up chunk i: slot[(2 i + 1) block]
  constexpr int BLOCK = sq_block(TPR);
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (t + i * TPR >= chunks) slot[2 * i * BLOCK] = slot[(2 * i + 1) * BLOCK] = make_uint4(0u, 0u, 0u, 0u);
  auto load = [&](Row of) {
    const uint4* x = p.X + (long long)of * 2 * chunks;
    if (of < p.M) {
#pragma unroll
      for (int i = 0; i < KEEP; ++i) {
        const int c = t + i * TPR;
        if (c < chunks) {
          cp_async16(smem_u32(slot + 2 * i * BLOCK), x + c);
          cp_async16(smem_u32(slot + (2 * i + 1) * BLOCK), x + chunks + c);
        }
      }
    }
  };
  load(row);
  const f32x2 magic = f2_make(12582912.0f, 12582912.0f);
  for (int turn = 0; row < p.M; row += step, turn ^= 1) {
    const uint4* x = p.X + (long long)row * 2 * chunks;
    f32x2 a[KEEP][4];
    float most[KEEP], top = 0.0f;  // |a|: of a chunk, of this thread
    uint32_t low2 = 0;             // the lowest gates of this thread, as bits: negative numbers are the larger the lower they are
    auto take = [&](const uint4& gc, const uint4& uc, f32x2 (&v)[4]) {
      low2 = __vimax3_u16x2(__vimax3_u16x2(low2, gc.x, gc.y), gc.z, gc.w);
      sq_gate8<BF16>(gc, uc, v);
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) f2_get(v[i], f[2 * i], f[2 * i + 1]);
      return f3_max_abs(f3_max_abs(f[0], f[1], f[2]), f3_max_abs(f[3], f[4], f[5]), f3_max_abs(f[6], f[7], 0.0f));
    };
    cp_async_wait();
#pragma unroll
    for (int i = 0; i < KEEP; ++i) most[i] = take(slot[2 * i * BLOCK], slot[(2 * i + 1) * BLOCK], a[i]);
#pragma unroll
    for (int i = 0; i < KEEP; i += 2) top = f3_max_abs(top, most[i], most[i + 1 < KEEP ? i + 1 : i]);
    for (int c = t + KEEP * TPR; c < chunks; c += TPR) {
      f32x2 v[4];
      top = f3_max_abs(top, take(ld_written(x + c), ld_written(x + chunks + c), v), 0.0f);
    }
    uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7fffffffu);  // as integers NaN and inf are on top
    uint32_t low = __reduce_max_sync(0xffffffffu, max(low2 & 0xffffu, low2 >> 16));
    if (WPR > 1) {
      if ((threadIdx.x & 31) == 0) {
        red[0][warp] = m;
        red[1][warp] = low;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WPR; ++w) {
        m = max(m, red[0][w]);
        low = max(low, red[1][w]);
      }
      if (t == 0) largest[turn ^ 1] = 0u;  // everybody is through with the last row's
    }
    const bool finite = m < 0x7f800000u;
    const bool odd = BF16 && (!finite || low > 0xc2aeu);  // 0xc2ae: -87
    float lowest = 0.0f;  // max(0, -g) over the row; beyond 88 fp32 gives 0 for a
    if (low & 0x8000u) lowest = fminf(BF16 ? __uint_as_float((low & 0x7fffu) << 16) : __half2float(__ushort_as_half((unsigned short)(low & 0x7fffu))), 88.0f);
    const float off = 5.5e-7f + 7.5e-8f * lowest;
    const float from = __uint_as_float(m) * (1.0f - (2.0f * off + 2e-7f));
    double best = 0.0;
    // Whoever may be the largest: nearly always one element of one thread, whose gate and up are kept over the next row's loads.
    uint32_t only = 0;  // (gate, up): not both zero
    const bool may = finite && m != 0 && top >= from;
    if (may) {
      auto consider = [&](const uint4* gp, const uint4* up, const f32x2 (&v)[4]) {
        uint32_t marked = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float lo, hi;
          f2_get(v[i], lo, hi);
          marked |= (fabsf(lo) >= from ? 1u << (2 * i) : 0u) | (fabsf(hi) >= from ? 2u << (2 * i) : 0u);
        }
        if (only == 0 && (marked & (marked - 1)) == 0) {
          const int i = __ffs(marked) - 1;
          only = reinterpret_cast<const volatile uint16_t*>(gp)[i] | (uint32_t)reinterpret_cast<const volatile uint16_t*>(up)[i] << 16;
        } else {
          best = fmax(best, sq_largest64<BF16>(gp, up, marked));
        }
      };
#pragma unroll
      for (int i = 0; i < KEEP; ++i)
        if (most[i] >= from) consider(slot + 2 * i * BLOCK, slot + (2 * i + 1) * BLOCK, a[i]);
      for (int c = t + KEEP * TPR; c < chunks; c += TPR) {
        f32x2 v[4];
        const float most_here = take(ld_written(x + c), ld_written(x + chunks + c), v);
        if (most_here >= from) consider(x + c, x + chunks + c, v);
      }
    }
    load(row + step);  // every slot has been read
    if (only != 0) best = fmax(best, fabs(sq_gate64(sq_float<BF16>(only & 0xffffu), sq_float<BF16>(only >> 16))));
    // The scale of each candidate, as bits; rounding keeps the order, so that the largest is the row's.
    uint32_t bits = __float_as_uint((float)(fmax(best, 1e-4) * (1.0 / 127.0)));
    if (WPR > 1) {
      if (may) atomicMax(&largest[turn], bits);
      __syncthreads();
      bits = max(bits, largest[turn]);
    } else {
      bits = __reduce_max_sync(0xffffffffu, bits);
    }
    float scale = __uint_as_float(bits);
    if (p.round_scale) scale = aq_pow2_ceil(scale);
    if (!finite) scale = __uint_as_float(m);  // inf or NaN: it stays one
    if (t == 0) p.S[row] = scale;
    const float rcp = rcp_approx(scale);
    const float share = finite ? rcp * (off + 2.5e-7f) : 0.0f;  // what a quotient may be off by, per |a|
    uint2* y = reinterpret_cast<uint2*>(p.Y) + (long long)row * chunks;
    const f32x2 rcp2 = f2_make(rcp, rcp);
    auto store = [&](int c, const f32x2 (&v)[4], float m) {
      float f[8], d[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2 s = f2_fma(v[i], rcp2, magic);  // 1.5 * 2^23 + a / s: the low bits are the nearest integer
        f2_get(s, f[2 * i], f[2 * i + 1]);
        f2_get(f2_fma(v[i], rcp2, f2_sub(magic, s)), d[2 * i], d[2 * i + 1]);  // how far it is
      }
      uint2 codes = make_uint2(aq_pack4(f), aq_pack4(f + 4));
      const float sure = 0.5f - m * share;
      if (f3_max_abs(f3_max_abs(d[0], d[1], d[2]), f3_max_abs(d[3], d[4], d[5]), f3_max_abs(d[6], d[7], 0.0f)) > sure) {
        uint32_t marked = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float lo, hi;
          f2_get(v[i], lo, hi);
          // by each one's own size, or, where the registers are full (32768 x 2048 64 -> 71 us with it), by the chunk's largest
          const float lo_sure = KEEP < 8 ? 0.5f - fabsf(lo) * share : sure, hi_sure = KEEP < 8 ? 0.5f - fabsf(hi) * share : sure;
          marked |= (fabsf(d[2 * i]) > lo_sure ? 1u << (2 * i) : 0u) | (fabsf(d[2 * i + 1]) > hi_sure ? 2u << (2 * i) : 0u);
        }
        if (marked) codes = sq_codes64<BF16>(x + c, x + chunks + c, scale, marked, codes);
      }
      y[c] = codes;
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (t + i * TPR < chunks) store(t + i * TPR, a[i], most[i]);
    for (int c = t + KEEP * TPR; c < chunks; c += TPR) {
      f32x2 v[4];
      sq_gate8<BF16>(ld_written(x + c), ld_written(x + chunks + c), v);
      store(c, v, __uint_as_float(m));
    }
    if (odd) {
      Row again = row;
      if constexpr (TIGHT) asm volatile("" : "+r"(again));  // the addresses are computed once more, not kept until here
      const long long r = again;
      sq_far_row<TPR>(p.X + r * 2 * chunks, chunks, t, p.round_scale, &largest[turn], reinterpret_cast<uint2*>(p.Y) + r * chunks, p.S + r);
    }
  }
}

}  // namespace qg
