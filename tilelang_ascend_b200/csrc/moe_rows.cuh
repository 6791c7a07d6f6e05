// Rows into the experts' order and back, for sm_100a.
//
// moe_act_quant_kernel: the per-token quantiser's arithmetic (act_quant.cuh, bit for bit), each row written to all the
// places of its token.  A row is read once, 2 N bytes, and written top_k times, N bytes each.
//
// moe_combine_kernel: out[t] = cast(base[t] + sum_j weights[t, j] * y[rows[t, j]]), fp32, j in order.  A thread has 16 bytes of a row.
// 2 top_k N bytes in and 2 N out per token.
#pragma once

#include "act_quant.cuh"
#include "common.cuh"

namespace qg {

struct MoeActQuantParams {
  const uint4* X;   // [T, N] bf16 or f16
  const int* rows;  // [T, k]: places in Y; negative: dropped, -2 - r: row r of Y is cleared
  int8_t* Y;        // [T * k, N]
  float* S;         // [T * k]
  long long T;
  int N;            // multiple of 8
  int k;
  int is_bf16;
  int round_scale;
};

template <int TPR, int KEEP>
__global__ void __launch_bounds__(aq_block(TPR)) moe_act_quant_kernel(const MoeActQuantParams p) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int ROWS = aq_block(TPR) / TPR;
  constexpr int WPR = TPR / 32;  // warps per row
  __shared__ float red[aq_block(TPR) / 32];
  const int t = threadIdx.x % TPR;
  const int r = threadIdx.x / TPR;
  const int warp = threadIdx.x >> 5;
  const long long row = (long long)blockIdx.x * ROWS + r;
  const bool live = row < p.T;
  const int chunks = p.N >> 3;
  const bool bf16 = p.is_bf16 != 0;
  const uint4* x = p.X + (live ? row : 0) * chunks;

  uint4 keep[KEEP];
  uint32_t m2 = 0u;
  if (live) {
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      const int c = t + i * TPR;
      if (c < chunks) {
        keep[i] = ld_written(x + c);
        m2 = aq_absmax8(keep[i], bf16, m2);
      }
    }
    for (int c = t + KEEP * TPR; c < chunks; c += TPR) m2 = aq_absmax8(ld_written(x + c), bf16, m2);
  }
  float m = aq_pair_max(m2, bf16);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (WPR > 1) {
    if ((threadIdx.x & 31) == 0) red[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WPR; ++w) m = fmaxf(m, red[r * WPR + w]);
  }
  if (!live) return;

  const float amax = fmaxf(m, 1e-4f);
  float scale = __fdiv_rn(amax, 127.0f);
  if (p.round_scale) scale = aq_pow2_ceil(scale);
  const float rcp = __frcp_rn(scale);
  const long long R = p.T * p.k;
  auto store = [&](int c, const uint2& v) {
    for (int j = 0; j < p.k; ++j) {
      const int at = ld_written(p.rows + row * p.k + j);
      const long long to = at >= 0 ? at : -2ll - at;
      if (to < 0 || to >= R) continue;
      reinterpret_cast<uint2*>(p.Y)[to * chunks + c] = at >= 0 ? v : make_uint2(0u, 0u);
      if (c == 0) p.S[to] = at >= 0 ? scale : 0.0f;
    }
  };
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int c = t + i * TPR;
    if (c < chunks) store(c, aq_quant8(keep[i], bf16, scale, rcp));
  }
  for (int c = t + KEEP * TPR; c < chunks; c += TPR) store(c, aq_quant8(ld_written(x + c), bf16, scale, rcp));
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

constexpr int MC_THREADS = 256;

template <bool BF16>
__global__ void __launch_bounds__(MC_THREADS) moe_combine_kernel(const MoeCombineParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const long long t = blockIdx.x / p.parts;
  const int chunks = p.N >> 3, c = (int)(blockIdx.x - t * p.parts) * MC_THREADS + threadIdx.x;
  if (c >= chunks) return;
  float acc[8], v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  if (p.base != nullptr) aq_unpack8(ld_written(p.base + t * chunks + c), BF16, acc);
  for (int j = 0; j < p.k; ++j) {
    const int row = ld_written(p.rows + t * p.k + j);
    if (row < 0 || row >= p.R) continue;
    const float w = ld_written(p.weights + t * p.k + j);
    aq_unpack8(ld_written(p.Y + (long long)row * chunks + c), BF16, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, v[i], acc[i]);
  }
  p.out[t * chunks + c] = make_uint4(pack_out2<BF16>(acc[0], acc[1]), pack_out2<BF16>(acc[2], acc[3]), pack_out2<BF16>(acc[4], acc[5]),
                                     pack_out2<BF16>(acc[6], acc[7]));
}

}  // namespace qg
