// Expert routing for sm_100a: logits [T, E] -> the top_k experts of every token and their weights.
//
//   s = softmax(l) or sigmoid(l)          c = s + bias (bias optional)          an expert is offered if l > -inf and c > -inf
//   groups: the value of a group is the sum of its one or two largest offered c; the top_groups best groups stay
//   experts = the top_k largest c that are offered and in a group that stays, ties to the lowest index, -1 where there are none
//   w = s[experts], divided by their sum if asked for, times a factor
//
// The picks are those of the real numbers: two scores that fp32 cannot tell apart must not depend on how a kernel adds.  Without
// a bias the logits themselves are compared (both score functions are increasing).  With one, or with sums of two scores, fp32
// values are compared and a token whose decision is nearer than the error of the fp32 scores is decided again in fp64.
//
// One warp per token, experts dealt to the lanes (lane + 32 i), in registers.
#pragma once

#include "common.cuh"

namespace qg {

constexpr int RT_WARPS = 4;       // warps of a block, a token each
constexpr int RT_MAX_E = 1024;    // experts: 32 per lane
constexpr int RT_MAX_K = 32;      // picks: one per lane
constexpr int RT_MAX_GROUPS = 32; // groups: one per lane

enum : int { RT_F16 = 0, RT_BF16 = 1, RT_F32 = 2 };

struct MoeRouteParams {
  const void* logits;  // [T, E]
  const float* bias;   // [E] or null
  float* weights;      // [T, k]
  int* experts;        // [T, k]
  long long T;
  int E, k, groups, group_n, top_groups, group_top;
  int softmax, renormalize;
  float scale;
};

template <int DT>
__device__ __forceinline__ float rt_load(const void* p, long long i) {
  if constexpr (DT == RT_F32) {
    return ld_written(static_cast<const float*>(p) + i);
  } else {
    uint16_t h;
    asm volatile("ld.global.u16 %0, [%1];" : "=h"(h) : "l"(static_cast<const uint16_t*>(p) + i));
    if constexpr (DT == RT_BF16) return __uint_as_float((uint32_t)h << 16);
    return __half2float(__ushort_as_half(h));
  }
}

// The larger value, or NaN if either is one.
__device__ __forceinline__ float rt_max(float a, float b) {
  float v;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(a), "f"(b));
  return v;
}

// Values as unsigned numbers of the same order; NaN above everything, both zeros alike, -inf (not offered) at RT_NONE.
template <typename K> struct RtKey;
template <> struct RtKey<uint32_t> {
  using F = float;
  static constexpr uint32_t NONE = 0x007fffffu;
  static __device__ __forceinline__ uint32_t of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v != v ? 0xffffffffu : b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
  }
  static __device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
};
template <> struct RtKey<unsigned long long> {
  using F = double;
  static constexpr unsigned long long NONE = 0x000fffffffffffffull;
  static __device__ __forceinline__ unsigned long long of(double v) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
    return v != v ? ~0ull : b ^ ((unsigned long long)((long long)b >> 63) | 0x8000000000000000ull);
  }
  static __device__ __forceinline__ double value(unsigned long long k) {
    return __longlong_as_double((long long)(k & 0x8000000000000000ull ? k ^ 0x8000000000000000ull : ~k));
  }
  static __device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return ((unsigned long long)hi << 32) | lo;
  }
};

// The groups that stay, as a bit mask.  `keys`: this warp's c in shared memory.  P lanes share a group and keep its two largest
// keys.  `eps` >= 0: `near` is set where the border between the groups that stay and the others is no wider than the error of c.
template <typename K>
__device__ __forceinline__ uint32_t rt_groups(const MoeRouteParams& p, const K* keys, int lane, typename RtKey<K>::F eps, bool& near) {
  using F = typename RtKey<K>::F;
  int share = 1;
  while (share * 2 * p.groups <= 32) share *= 2;
  const int g = lane / share, part = lane - g * share;
  K a = 0, b = 0;  // largest, second largest
  if (g < p.groups) {
    for (int i = part; i < p.group_n; i += share) {
      const K v = keys[g * p.group_n + i];
      if (v > a) { b = a; a = v; }
      else if (v > b) b = v;
    }
  }
  for (int o = 1; o < share; o *= 2) {
    const K a2 = __shfl_xor_sync(0xffffffffu, a, o), b2 = __shfl_xor_sync(0xffffffffu, b, o);
    const K lo = a < a2 ? a : a2, hi2 = b > b2 ? b : b2;
    a = a > a2 ? a : a2;
    b = lo > hi2 ? lo : hi2;
  }
  F v = RtKey<K>::value(a > RtKey<K>::NONE ? a : RtKey<K>::NONE);
  if (p.group_top == 2 && b > RtKey<K>::NONE) v += RtKey<K>::value(b);
  const K mine = g < p.groups ? RtKey<K>::of(v) : 0;
  int rank = 0;
  for (int j = 0; j < p.groups; ++j) {
    const K other = __shfl_sync(0xffffffffu, mine, j * share);
    rank += (other > mine || (other == mine && j < g)) ? 1 : 0;
  }
  const bool leads = part == 0 && g < p.groups;
  if (eps >= 0 && p.top_groups < p.groups) {
    const uint32_t last = __ballot_sync(0xffffffffu, leads && rank == p.top_groups - 1);
    const uint32_t next = __ballot_sync(0xffffffffu, leads && rank == p.top_groups);
    const F x = __shfl_sync(0xffffffffu, v, __ffs(last) - 1), y = __shfl_sync(0xffffffffu, v, __ffs(next) - 1);
    if (x - y <= 2 * eps + (F)0x1p-21 * (fabs(x) + fabs(y))) near = true;
  }
  uint32_t stays = 0;
  const uint32_t kept = __ballot_sync(0xffffffffu, leads && rank < p.top_groups);
  for (int j = 0; j < p.groups; ++j) stays |= ((kept >> (j * share)) & 1u) << j;
  return stays;
}

// One token again in fp64; lane j < k returns pick j or -1.
__device__ __noinline__ int rt_decide_in_64(const MoeRouteParams& p, const void* row, int dt, unsigned long long* keys, bool by_logits,
                                            float top, int lane) {
  using K = RtKey<unsigned long long>;
  auto logit = [&](int e) { return dt == RT_F32 ? rt_load<RT_F32>(row, e) : dt == RT_BF16 ? rt_load<RT_BF16>(row, e) : rt_load<RT_F16>(row, e); };
  double sum = 0;
  if (p.softmax) {
    for (int e = lane; e < p.E; e += 32) sum += exp((double)logit(e) - (double)top);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  auto fill = [&](bool logits) {
    __syncwarp();
    for (int e = lane; e < p.E; e += 32) {
      const float l = logit(e);
      double c = (double)l;
      if (!logits) {
        c = p.softmax ? exp((double)l - (double)top) / sum : 1.0 / (1.0 + exp(-(double)l));
        if (p.bias != nullptr) c += (double)ld_written(p.bias + e);
        if (l == -INFINITY) c = -INFINITY;
      }
      keys[e] = K::of(c);
    }
    __syncwarp();
  };
  fill(false);
  bool near = false;
  uint32_t stays = 0xffffffffu;
  if (p.groups > 1) stays = rt_groups<unsigned long long>(p, keys, lane, -1.0, near);
  if (by_logits) fill(true);
  int pick = -1;
  for (int r = 0; r < p.k; ++r) {
    unsigned long long best = 0;
    int at = 0x7fffffff;
    for (int e = lane; e < p.E; e += 32)
      if (((stays >> (e / p.group_n)) & 1u) && keys[e] > best) { best = keys[e]; at = e; }
    const unsigned long long m = K::warp_max(best);
    if (m <= K::NONE) break;
    const int e = __reduce_min_sync(0xffffffffu, best == m ? at : 0x7fffffff);
    if (lane == r) pick = e;
    __syncwarp();
    if (lane == 0) keys[e] = 0;
    __syncwarp();
  }
  return pick;
}

template <int DT, int V>
__global__ void __launch_bounds__(RT_WARPS * 32) moe_route_kernel(const MoeRouteParams p) {
  using K = RtKey<uint32_t>;
  extern __shared__ unsigned long long rt_smem[];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long* keys64 = rt_smem + (size_t)warp * p.E;
  uint32_t* keys32 = reinterpret_cast<uint32_t*>(keys64);
  const bool by_logits = p.bias == nullptr;                                      // the picks' order
  const bool groups_by_logits = by_logits && p.group_top == 1;                   // the groups' order
  const bool need_scores = !by_logits || (p.groups > 1 && !groups_by_logits);
  const bool need_sum = p.softmax && (need_scores || !p.renormalize);
  for (long long t = (long long)blockIdx.x * RT_WARPS + warp; t < p.T; t += (long long)gridDim.x * RT_WARPS) {
    const void* row = static_cast<const char*>(p.logits) + t * p.E * (DT == RT_F32 ? 4 : 2);
    float l[V];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane + 32 * i;
      l[i] = e < p.E ? rt_load<DT>(row, e) : -INFINITY;
      top = rt_max(top, l[i]);
    }
    float sum = 1.0f;
    if (p.softmax) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = rt_max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    uint32_t key[V];
    if (need_sum) {
      sum = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) sum += lane + 32 * i < p.E ? expf(l[i] - top) : 0.0f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    const float inv_sum = 1.0f / sum;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane + 32 * i;
      float c = l[i];
      if (need_scores && e < p.E) {
        c = p.softmax ? expf(l[i] - top) * inv_sum : 1.0f / (1.0f + expf(-l[i]));
        if (p.bias != nullptr) c += ld_written(p.bias + e);
        if (l[i] == -INFINITY) c = -INFINITY;
      }
      key[i] = e < p.E ? K::of(c) : 0u;
    }
    // fp32 scores are off by less than 2^-20 of the largest score that there can be
    const float eps = 0x1p-20f * (p.softmax ? inv_sum : 1.0f);
    bool near = false;
    if (p.groups > 1) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (lane + 32 * i < p.E) keys32[lane + 32 * i] = key[i];
      __syncwarp();
      const uint32_t stays = rt_groups<uint32_t>(p, keys32, lane, groups_by_logits ? -1.0f : eps, near);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = lane + 32 * i;
        if (by_logits) key[i] = e < p.E ? K::of(l[i]) : 0u;
        if (e >= p.E || !((stays >> (e / p.group_n)) & 1u)) key[i] = 0u;
      }
    }
    int pick = -1;
    float prev = INFINITY;
    for (int r = 0; r < (by_logits ? p.k : p.k + 1); ++r) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) best = max(best, key[i]);
      const uint32_t m = K::warp_max(best);
      if (m <= K::NONE) break;
      if (!by_logits) {
        const float v = K::value(m);
        if (r > 0 && prev - v <= 2 * eps + 0x1p-21f * (fabsf(prev) + fabsf(v))) near = true;
        prev = v;
      }
      if (r == p.k) break;
      int at = 0x7fffffff;
#pragma unroll
      for (int i = V - 1; i >= 0; --i)
        if (key[i] == m) at = lane + 32 * i;
      const int e = __reduce_min_sync(0xffffffffu, at);
      if (lane == r) pick = e;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (lane + 32 * i == e) key[i] = 0u;
    }
    if (near) pick = rt_decide_in_64(p, row, DT, keys64, by_logits, top, lane);
    // weights: lane j has pick j.  Divided by their sum they depend on differences of the logits only, which keeps them
    // exact where all the picked scores are tiny.
    const bool there = pick >= 0;
    const float lp = there ? rt_load<DT>(row, pick) : -INFINITY;
    float s;
    if (p.renormalize) {
      float lm = lp;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) lm = fmaxf(lm, __shfl_xor_sync(0xffffffffu, lm, o));
      s = p.softmax || lm < -30.0f ? expf(lp - lm) : 1.0f / (1.0f + expf(-lp));
      if (p.softmax) s += top - top;  // the sum of all scores is NaN where a logit is NaN or +inf
      if (!there) s = 0.0f;
      float all = s;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      s = s / all;
    } else {
      s = p.softmax ? expf(lp - top) * inv_sum : 1.0f / (1.0f + expf(-lp));
    }
    if (lane < p.k) {
      p.experts[t * p.k + lane] = pick;
      p.weights[t * p.k + lane] = there ? s * p.scale : 0.0f;
    }
  }
}

}  // namespace qg
