// Rows into the experts' order and back, for sm_100a.
//
// moe_act_quant_kernel: the per-token quantiser's arithmetic (act_quant.cuh, bit for bit), each row written to all the
// places of its token.  A row is read once, 2 N bytes, and written top_k times, N bytes each.
//
// moe_combine_kernel: out[t] = cast(base[t] + sum_j weights[t, j] * y[rows[t, j]]), fp32, j in order.  A thread has 16 bytes of a row.
// 2 top_k N bytes in and 2 N out per token, which is what bounds it once up to eight entries are in flight per thread: 4096 tokens of 7168, eight
// entries each, 6.7 TB/s (79 us; 92 with one entry after another, and 16 tokens 1.8 us instead of 3.0).
#pragma once

#include "act_quant.cuh"
#include "common.cuh"
#include "packed_float.cuh"

namespace qg {

struct MoeActQuantParams {
  const uint4* X;   // [T, N] bf16 or f16
  const int* rows;  // [T, k]: places in Y; negative: dropped, -2 - r: row r of Y is cleared
  int8_t* Y;        // [T * k, N]
  float* S;         // [T * k]
  long long T;
  int N;            // multiple of 8
  int k;
  int round_scale;
};

// aq_quant8 with the fp32 steps in pairs: the same roundings, the same bits.
template <bool BF16>
__device__ __forceinline__ uint2 mq_quant8(const uint4& v, f32x2 less_scale, f32x2 rcp) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  const f32x2 magic = f2_make(12582912.0f, 12582912.0f);
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 x = f2_of_half2<BF16>(w[i]);
    const f32x2 q0 = f2_mul(x, rcp);
    const f32x2 q1 = f2_fma(f2_fma(q0, less_scale, x), rcp, q0);
    const f32x2 q2 = f2_fma(f2_fma(q1, less_scale, x), rcp, q1);
    f2_get(f2_add(q2, magic), f[2 * i], f[2 * i + 1]);
  }
  return make_uint2(aq_pack4(f), aq_pack4(f + 4));
}

// TPR threads share a row, KEEP chunks of eight elements of it in each one's registers; longer rows are read a second time.  The
// blocks are persistent: the next row's chunks and places are fetched while this one's codes are stored.
__host__ __device__ constexpr int mq_block(int tpr) { return tpr == 32 ? 128 : tpr; }
__host__ __device__ constexpr int mq_smem_bytes(int tpr, int keep) { return keep * 16 * mq_block(tpr); }
template <int TPR, int KEEP, bool BF16>
__global__ void __launch_bounds__(mq_block(TPR), KEEP > 4 ? (512 + mq_block(TPR) - 1) / mq_block(TPR) : 1) moe_act_quant_kernel(const MoeActQuantParams p) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int BLOCK = mq_block(TPR), ROWS = BLOCK / TPR, WPR = TPR / 32;
  static_assert(WPR == 1 || ROWS == 1, "barriers are of the whole block");
  __shared__ float red[2][WPR];
  extern __shared__ uint4 mq_slots[];  // a thread's own chunks: no barrier is needed to read them
  uint4* slot = mq_slots + threadIdx.x;
  const int t = threadIdx.x % TPR, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunks = p.N >> 3;
  const long long R = p.T * p.k;
  const int step = gridDim.x * ROWS;
  int row = blockIdx.x * ROWS + threadIdx.x / TPR;
  int places = -1;  // lane j: place j of the next row (up to 32 of them)
  auto fetch = [&](int of) {
    if (of >= p.T) return;
    const uint4* x = p.X + (long long)of * chunks;
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (t + i * TPR < chunks) cp_async16(smem_u32(slot + i * BLOCK), x + t + i * TPR);
    if (lane < p.k) places = ld_written(p.rows + (long long)of * p.k + lane);
  };
  fetch(row);
  for (int turn = 0; row < p.T; row += step, turn ^= 1) {
    const uint4* x = p.X + (long long)row * chunks;
    uint4 keep[KEEP];
    uint32_t m2 = 0u;
    cp_async_wait();
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      if (t + i * TPR < chunks) {
        keep[i] = slot[i * BLOCK];
        m2 = aq_absmax8(keep[i], BF16, m2);
      }
    }
    for (int c = t + KEEP * TPR; c < chunks; c += TPR) m2 = aq_absmax8(ld_written(x + c), BF16, m2);
    float m = aq_pair_max(m2, BF16);
    m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
    const int at_lane = places;
    fetch(row + step);  // every slot has been read
    if (WPR > 1) {
      if (lane == 0) red[turn][warp] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WPR; ++w) m = fmaxf(m, red[turn][w]);
    }
    const float amax = fmaxf(m, 1e-4f);
    float scale = __fdiv_rn(amax, 127.0f);
    if (p.round_scale) scale = aq_pow2_ceil(scale);
    const float rcp = __frcp_rn(scale);
    const f32x2 less_scale = f2_make(-scale, -scale), rcp2 = f2_make(rcp, rcp);
    uint2 code[KEEP];
#pragma unroll
    for (int i = 0; i < KEEP; ++i) code[i] = mq_quant8<BF16>(keep[i], less_scale, rcp2);
    for (int j = 0; j < p.k; ++j) {
      const int at = j < 32 ? __shfl_sync(0xffffffffu, at_lane, j) : ld_written(p.rows + (long long)row * p.k + j);
      const long long to = at >= 0 ? at : -2ll - at;
      if (to < 0 || to >= R) continue;
      uint2* y = reinterpret_cast<uint2*>(p.Y) + to * chunks;
      const uint32_t mask = at >= 0 ? 0xffffffffu : 0u;
#pragma unroll
      for (int i = 0; i < KEEP; ++i)
        if (t + i * TPR < chunks) __stcs(y + t + i * TPR, make_uint2(code[i].x & mask, code[i].y & mask));
      for (int c = t + KEEP * TPR; c < chunks; c += TPR) {
        const uint2 v = mq_quant8<BF16>(ld_written(x + c), less_scale, rcp2);
        __stcs(y + c, make_uint2(v.x & mask, v.y & mask));
      }
      if (t == 0) p.S[to] = at >= 0 ? scale : 0.0f;
    }
  }
}

struct MoeCombineParams {
  const uint4* Y;        // [R, N] bf16 or f16
  const int* rows;       // [T, k]: rows of Y; outside 0 .. R - 1: dropped
  const float* weights;  // [T, k]
  const uint4* base;     // [T, N] or null
  uint4* out;            // [T, N]
  long long R, T;
  int N;                 // multiple of 8
  int k;
  int parts;             // blocks per token
};

constexpr int MC_THREADS = 128;  // (256: 4096 tokens of 7168, eight entries each 81.5 us instead of 79.1)

// AHEAD entries of a token are in flight at a time: their places and weights, then their 16 bytes.
template <bool BF16, int AHEAD>
__global__ void __launch_bounds__(MC_THREADS) moe_combine_kernel(const MoeCombineParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const long long t = blockIdx.x / p.parts;
  const int chunks = p.N >> 3, c = (int)(blockIdx.x - t * p.parts) * MC_THREADS + threadIdx.x;
  if (c >= chunks) return;
  float acc[8], f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  if (p.base != nullptr) aq_unpack8(ld_written(p.base + t * chunks + c), BF16, acc);
  const int* rows = p.rows + t * p.k;
  const float* weights = p.weights + t * p.k;
  for (int j0 = 0; j0 < p.k; j0 += AHEAD) {
    int row[AHEAD];
    float w[AHEAD];
    uint4 v[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      row[j] = j0 + j < p.k ? ld_written(rows + j0 + j) : -1;
      w[j] = j0 + j < p.k ? ld_written(weights + j0 + j) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (row[j] >= 0 && row[j] < p.R) v[j] = ld_written(p.Y + (long long)row[j] * chunks + c);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (row[j] < 0 || row[j] >= p.R) continue;
      aq_unpack8(v[j], BF16, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = fmaf(w[j], f[i], acc[i]);
    }
  }
  p.out[t * chunks + c] = make_uint4(pack_out2<BF16>(acc[0], acc[1]), pack_out2<BF16>(acc[2], acc[3]), pack_out2<BF16>(acc[4], acc[5]),
                                     pack_out2<BF16>(acc[6], acc[7]));
}

}  // namespace qg
