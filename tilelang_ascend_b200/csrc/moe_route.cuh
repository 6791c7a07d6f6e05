// Expert routing for sm_100a: logits [T, E] -> the top_k experts of every token and their weights.
//
//   s = softmax(l) or sigmoid(l)          c = s + bias (bias optional)          an expert is offered if l > -inf and c > -inf
//   groups: the value of a group is the sum of its one or two largest offered c; the top_groups best groups stay
//   experts = the top_k largest c that are offered and in a group that stays, ties to the lowest index, -1 where there are none
//   w = s[experts], divided by their sum if asked for, times a factor
//
// The picks are those of the real numbers: two scores that fp32 cannot tell apart must not depend on how a kernel adds.  Without
// a bias the logits themselves are compared (both score functions are increasing).  With one, or with sums of two scores, fp32
// values are compared and a token whose decision is nearer than the error of the fp32 scores is decided again in fp64 (random
// scores: one token in some hundreds; what fp64 gives the same number is a tie).  That error goes by the largest finite bias: one of -1e9 among
// others of 0.1 sends every token there, 16384 x 256 with groups 75 us instead of 25 (-inf, which takes an expert out, 26).
//
// One warp per token.  The experts of a group are dealt to a power of two of lanes, so that shuffles settle it whatever its size
// (through shared memory 8000 x 160 in 8 groups was 17.3 us instead of 10.9).  A lane has up to V consecutive experts as 32-bit keys
// in the order of the values, whose lowest bits are the place within the lane, and sorts them (in lists of eight) in registers.  The
// value that top_k lanes' heads reach bounds the picks from below: a maximum over the heads, one redux instruction, top_k times.  The
// keys from there on, a dozen or so, are gathered by votes and each lane counts how many come before its own.  (A maximum over the
// heads per pick, with a step of the winner's list, was 32 instructions a pick; this is 130 for all.)  What bounds it is issue:
// 16384 x 256 in bf16 with bias and groups is 1.5 us of memory and 792 instructions of a warp per token, 11 us at one a cycle;
// measured 21.6.
#pragma once

#include "common.cuh"
#include "packed_float.cuh"

namespace qg {

constexpr int RT_WARPS = 4;       // warps of a block, a token each
constexpr int RT_MAX_E = 1024;    // experts: 32 per lane, up to 60 where groups leave lanes idle
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
  int log_share, per_lane;  // a group's experts are dealt to 2^log_share lanes, per_lane to each
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

// Two experts whose scores are the same number.
template <int DT>
__device__ __forceinline__ bool rt_equal(const MoeRouteParams& p, const void* row, int e, int f, bool by_logits) {
  return rt_load<DT>(row, e) == rt_load<DT>(row, f) && (by_logits || ld_written(p.bias + e) == ld_written(p.bias + f));
}

// Values as unsigned numbers of the same order; NaN above everything, both zeros alike, -inf (not offered) at RT_NONE.
constexpr int RT_LIST = 72;  // two lists of 36 entries of a warp, on a 16-byte boundary
__host__ __device__ constexpr int rt_smem_bytes(int E) { return 8 * (RT_WARPS * E + RT_WARPS * RT_LIST); }
static_assert(RT_WARPS % 2 == 0, "the lists, behind the warps' keys, start on a 16-byte boundary");

template <typename K> struct RtKey;
template <> struct RtKey<uint32_t> {
  using F = float;
  static constexpr uint32_t NONE = 0x007fffffu;
  static __device__ __forceinline__ uint32_t of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);  // (a NaN comes out of an addition as 0x7fffffff)
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
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

// What a group with the largest keys a and b is worth.  Keys of logits stand for their scores, for softmax times a common factor.
template <typename F, typename K>
__device__ __forceinline__ F rt_group_value(const MoeRouteParams& p, K a, K b, bool by_logits, float top) {
  F v = RtKey<K>::value(a > RtKey<K>::NONE ? a : RtKey<K>::NONE);
  if (p.group_top == 1) return v;
  F w = RtKey<K>::value(b > RtKey<K>::NONE ? b : RtKey<K>::NONE);
  if (by_logits && a > RtKey<K>::NONE) {
    auto score = [&](F l) -> F {
      if constexpr (sizeof(F) == 8) return p.softmax ? exp(l - (F)top) : 1.0 / (1.0 + exp(-l));
      else return p.softmax ? expf(l - top) : __fdividef(1.0f, 1.0f + expf(-l));
    };
    v = score(v);
    w = b > RtKey<K>::NONE ? score(w) : w;
  }
  return b > RtKey<K>::NONE ? v + w : v;
}

// The groups that stay, as a bit mask, from the keys of all experts in shared memory.
__device__ __forceinline__ uint32_t rt_groups_in_64(const MoeRouteParams& p, const unsigned long long* keys, int lane, bool by_logits, float top) {
  using K = RtKey<unsigned long long>;
  const int share = 1 << p.log_share, g = lane >> p.log_share, part = lane & (share - 1);
  unsigned long long a = 0, b = 0;  // largest, second largest of this lane's part of group g
  if (g < p.groups) {
    for (int i = part; i < p.group_n; i += share) {
      const unsigned long long v = keys[g * p.group_n + i];
      if (v > a) { b = a; a = v; }
      else if (v > b) b = v;
    }
  }
  for (int o = 1; o < share; o *= 2) {
    const unsigned long long a2 = __shfl_xor_sync(0xffffffffu, a, o), b2 = __shfl_xor_sync(0xffffffffu, b, o);
    b = max(max(b, b2), min(a, a2));
    a = max(a, a2);
  }
  const unsigned long long mine = g < p.groups ? K::of(rt_group_value<double>(p, a, b, by_logits, top)) : 0;
  int rank = 0;
  for (int j = 0; j < p.groups; ++j) {
    const unsigned long long other = __shfl_sync(0xffffffffu, mine, j << p.log_share);
    rank += (other > mine || (other == mine && j < g)) ? 1 : 0;
  }
  const uint32_t kept = __ballot_sync(0xffffffffu, part == 0 && g < p.groups && rank < p.top_groups);
  uint32_t stays = 0;
  for (int j = 0; j < p.groups; ++j) stays |= ((kept >> (j << p.log_share)) & 1u) << j;
  return stays;
}

// What is compared, in fp64: without a bias the exact logits.
struct RtScore64 {
  const MoeRouteParams& p;
  const void* row;
  int dt;
  bool by_logits;
  float top = 0.0f;
  double sum = 1.0;
  __device__ __forceinline__ float logit(int e) const {
    return dt == RT_F32 ? rt_load<RT_F32>(row, e) : dt == RT_BF16 ? rt_load<RT_BF16>(row, e) : rt_load<RT_F16>(row, e);
  }
  __device__ __forceinline__ void prepare(int lane) {
    uint32_t most = 0;
    for (int e = lane; e < p.E; e += 32) most = max(most, RtKey<uint32_t>::of(logit(e)));
    top = RtKey<uint32_t>::value(RtKey<uint32_t>::warp_max(most));
    if (!p.softmax || by_logits) return;
    sum = 0.0;
    for (int e = lane; e < p.E; e += 32) sum += exp((double)logit(e) - (double)top);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  __device__ __forceinline__ unsigned long long key(int e) const {
    const float l = logit(e);
    double c = (double)l;
    if (!by_logits) {
      c = (p.softmax ? exp((double)l - (double)top) / sum : 1.0 / (1.0 + exp(-(double)l))) + (double)ld_written(p.bias + e);
      if (l == -INFINITY) c = -INFINITY;
    }
    return RtKey<unsigned long long>::of(c);
  }
};

// One token again in fp64; lane j < k returns pick j or -1.
__device__ __noinline__ int rt_decide_in_64(const MoeRouteParams& p, const void* row, int dt, unsigned long long* keys, bool by_logits, int lane) {
  using K = RtKey<unsigned long long>;
  RtScore64 score{p, row, dt, by_logits};
  score.prepare(lane);
  __syncwarp();
  for (int e = lane; e < p.E; e += 32) keys[e] = score.key(e);
  __syncwarp();
  if (p.groups > 1) {
    const uint32_t stays = rt_groups_in_64(p, keys, lane, by_logits, score.top);
    __syncwarp();
    for (int e = lane; e < p.E; e += 32)
      if (!((stays >> (e / p.group_n)) & 1u)) keys[e] = 0;
  }
  int pick = -1;
  for (int r = 0; r < p.k; ++r) {
    __syncwarp();
    unsigned long long best = 0;
    int at = 0x7fffffff;
    for (int e = lane; e < p.E; e += 32) {
      const unsigned long long k = keys[e];
      if (k > best) { best = k; at = e; }
    }
    const unsigned long long m = K::warp_max(best);
    if (m <= K::NONE) break;
    const int e = __reduce_min_sync(0xffffffffu, best == m ? at : 0x7fffffff);
    if (lane == r) pick = e;
    if (lane == (e & 31)) keys[e] = 0;
  }
  return pick;
}

// The order of n candidates, expert `e` of lane < n, in fp64.
__device__ __noinline__ int rt_rank_in_64(const MoeRouteParams& p, const void* row, int dt, bool by_logits, int e, int n, int lane) {
  RtScore64 score{p, row, dt, by_logits};
  if (p.softmax && !by_logits) score.prepare(lane);
  const unsigned long long mine = lane < n ? score.key(e) : 0ull;
  int rank = 0;
  for (int i = 0; i < n; ++i) {
    const unsigned long long other = __shfl_sync(0xffffffffu, mine, i);
    const int f = __shfl_sync(0xffffffffu, e, i);
    rank += other > mine || (other == mine && f < e) ? 1 : 0;
  }
  return lane < n ? rank : lane;
}

constexpr float RT_LOG2E = 1.4426950408889634f;
// Off by less than 2^-21: the error of exp, 2^-22 + |l| 7.5e-8, enters times s (1 - s), and sum and reciprocal add 1.5 * 2^-23.
__device__ __forceinline__ float rt_sigmoid(float l) { return rcp_approx(1.0f + ex2_approx(-RT_LOG2E * l)); }
// exp(l - top) to 2^-22 + |l - top| 7.5e-8, relative: the argument's rounding is put right behind the approximation.
__device__ __forceinline__ float rt_exp_below(float l, float top) {
  const float x = l - top, t = x * RT_LOG2E, e = ex2_approx(t);
  return x < -100.0f ? 0.0f : fmaf(e, fmaf(x, RT_LOG2E, -t) * 0.6931471806f, e);
}

// Largest first.
template <int L>
__device__ __forceinline__ void rt_sort(uint32_t (&k)[L]) {
  auto order = [&](int i, int j) {
    const uint32_t hi = max(k[i], k[j]), lo = min(k[i], k[j]);
    k[i] = hi;
    k[j] = lo;
  };
  if constexpr (L == 2) {
    order(0, 1);
  } else if constexpr (L == 4) {
    order(0, 1), order(2, 3), order(0, 2), order(1, 3), order(1, 2);
  } else if constexpr (L == 8) {
    order(0, 2), order(1, 3), order(4, 6), order(5, 7), order(0, 4), order(1, 5), order(2, 6), order(3, 7), order(0, 1), order(2, 3);
    order(4, 5), order(6, 7), order(2, 4), order(3, 5), order(1, 4), order(3, 6), order(1, 2), order(3, 4), order(5, 6);
  }
}

// A lane's V logits, by loads of up to 16 bytes (VEC: every lane has all V or none, and rows keep the alignment) or one by one.
template <int DT, int V, bool VEC>
struct RtRow {
  static constexpr int BYTES = V * (DT == RT_F32 ? 4 : 2);
  static constexpr int WORDS = VEC ? (BYTES + 3) / 4 : V;
  uint32_t w[WORDS];
  __device__ __forceinline__ RtRow() {  // -inf, which a lane without experts keeps
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = !VEC || DT == RT_F32 ? 0xff800000u : (DT == RT_BF16 ? 0xff80ff80u : 0xfc00fc00u);
  }
  __device__ __forceinline__ void load(const void* row, int first, int count) {
    const char* p = static_cast<const char*>(row) + (long long)first * (DT == RT_F32 ? 4 : 2);
    if constexpr (!VEC) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = i < count ? __float_as_uint(rt_load<DT>(row, first + i)) : 0xff800000u;
    } else {
      if (count == 0) return;
      if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
          const uint4 v = ld_written(reinterpret_cast<const uint4*>(p) + i);
          w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
      } else if constexpr (BYTES == 8) {
        const uint2 v = ld_written(reinterpret_cast<const uint2*>(p));
        w[0] = v.x, w[1] = v.y;
      } else if constexpr (BYTES == 4) {
        w[0] = (uint32_t)ld_written(reinterpret_cast<const int*>(p));
      } else {
        uint16_t h;
        asm volatile("ld.global.u16 %0, [%1];" : "=h"(h) : "l"(p));
        w[0] = h;
      }
    }
  }
  __device__ __forceinline__ void values(float (&l)[V]) const {
    if constexpr (!VEC) {
#pragma unroll
      for (int i = 0; i < V; ++i) l[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (DT == RT_F32) l[i] = __uint_as_float(w[i]);
        else if constexpr (DT == RT_BF16) l[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        else l[i] = __half2float(__ushort_as_half((unsigned short)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu)));
      }
    }
  }
};

// Blocks per SM that the registers have to allow.  us, 16384 x 256 with groups: 108 registers 30, 80 25.6, 72 23.7, 64 25.5, 48 27.0.
__host__ __device__ constexpr int rt_min_blocks(int V) { return V <= 8 ? 7 : V == 16 ? 4 : 2; }
template <int DT, int V, bool VEC>
__global__ void __launch_bounds__(RT_WARPS * 32, rt_min_blocks(V)) moe_route_kernel(const MoeRouteParams p) {
  using K = RtKey<uint32_t>;
  constexpr int L = V < 8 ? V : 8, S = V / L;  // sorted lists of a lane
  constexpr uint32_t PLACE = V - 1;            // the lowest bits of a key: V - 1 - place within the lane
  extern __shared__ __align__(16) unsigned long long rt_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long* keys64 = rt_smem + (size_t)warp * p.E;
  // candidates, and what is in each place of the order: (expert backwards, value)
  uint2* list = reinterpret_cast<uint2*>(rt_smem + (size_t)RT_WARPS * p.E) + warp * RT_LIST;
  uint2* place = list + RT_LIST / 2;
  // Lanes of a power of two to a group, so that it is settled by shuffles; in the order of the experts.
  const int share = 1 << p.log_share, part = lane & (share - 1), my_group = lane >> p.log_share;
  const int first = my_group * p.group_n + part * p.per_lane;
  const int count = my_group < p.groups ? max(0, min(p.per_lane, p.group_n - part * p.per_lane)) : 0;
  const bool by_logits = p.bias == nullptr;  // the picks' order
  const bool need_sum = p.softmax && (!by_logits || !p.renormalize);
  const bool need_top = p.softmax && (need_sum || (p.groups > 1 && p.group_top == 2));
  const uint32_t below = (1u << lane) - 1u;
  const uint32_t backwards = (uint32_t)(31 - lane) * V;
  auto expert_of = [&](uint32_t lane_and_place) {  // both backwards
    const int l = 31 - (int)(lane_and_place / V);
    return (l >> p.log_share) * p.group_n + (l & (share - 1)) * p.per_lane + (int)(PLACE - (lane_and_place & PLACE));
  };
  pdl_wait();
  pdl_launch_dependents();
  float bias[V];
  float most_bias = 0.0f;
  if (!by_logits) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      bias[i] = i < count ? ld_written(p.bias + first + i) : -INFINITY;
      if (fabsf(bias[i]) < INFINITY) most_bias = fmaxf(most_bias, fabsf(bias[i]));
    }
    most_bias = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most_bias)));
  }
  const long long row_bytes = (long long)p.E * (DT == RT_F32 ? 4 : 2);
  const int step = gridDim.x * RT_WARPS;
  int t = blockIdx.x * RT_WARPS + warp;
  const char* row = static_cast<const char*>(p.logits) + t * row_bytes;
  RtRow<DT, V, VEC> next;
  if (t < p.T) next.load(row, first, count);
  for (; t < p.T; t += step, row += step * row_bytes) {
    float l[V];
    next.values(l);
    if (t + step < p.T) next.load(row + step * row_bytes, first, count);
    float top = 0.0f, inv_sum = 1.0f;
    float c[V];
    if (need_top) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) m = max(m, K::of(l[i]));
      top = K::value(K::warp_max(m));
    }
    if (need_sum) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        c[i] = rt_exp_below(l[i], top);
        sum += c[i];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      inv_sum = 1.0f / sum;
    }
    // Keys.  What is not offered is -inf.
    uint32_t key[S][L];
    bool exact = true;  // the place takes no bits from a value
    if (by_logits) {
#pragma unroll
      for (int i = 0; i < V; ++i) c[i] = l[i];
      if constexpr (DT == RT_F32) {  // (16-bit logits end in zeros)
        uint32_t lost = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) lost |= __float_as_uint(l[i]) & PLACE;
        exact = !__any_sync(0xffffffffu, lost != 0);
      }
    } else {
      float least = l[0];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        c[i] = (p.softmax ? c[i] * inv_sum : rt_sigmoid(l[i])) + bias[i];
        least = fminf(least, l[i]);
      }
      if (least == -INFINITY) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (l[i] == -INFINITY) c[i] = -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) key[i / L][i % L] = (K::of(c[i]) & ~PLACE) | (PLACE - i);
    // How near two c may come before fp32 cannot tell them apart, in units of 2^-24 of the largest score that there can be.  sigmoid: 8 each
    // (rt_sigmoid), 16.  softmax: the exponentials 4 each (what smaller ones are off by is less), their products with 1 / sum 1 each, and
    // the sum, whose V + 4 additions, exponentials and division move all scores alike, V + 9: V + 19.  Then, of the largest score
    // and bias, the sum with the bias 1 each and the bits that the place takes 2 (V - 1) of either.  3 V + 19 in all, of the 20 + 4 V here.
    const float score = p.softmax && !by_logits ? inv_sum : 1.0f;
    const float tol = 0x1p-20f * score + (0x1p-22f + V * 0x1p-22f) * (most_bias + score);
    bool near = false, kept = true;
#pragma unroll
    for (int s = 0; s < S; ++s) rt_sort<L>(key[s]);
    if (p.groups > 1) {
      // The two largest of the group, by the exact logits where those are what is compared.
      uint32_t a = 0, b = 0;
      if (by_logits) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const uint32_t k = K::of(l[i]);
          b = max(b, min(a, k));
          a = max(a, k);
        }
      } else {
        a = key[0][0];
        b = L > 1 ? key[0][1 % L] : 0u;
#pragma unroll
        for (int s = 1; s < S; ++s) {
          b = max(max(b, key[s][1 % L]), min(a, key[s][0]));
          a = max(a, key[s][0]);
        }
      }
      for (int o = 1; o < share; o *= 2) {
        const uint32_t a2 = __shfl_xor_sync(0xffffffffu, a, o), b2 = __shfl_xor_sync(0xffffffffu, b, o);
        b = max(max(b, b2), min(a, a2));
        a = max(a, a2);
      }
      if (!by_logits) a = a < K::NONE ? a : a & ~PLACE, b = b < K::NONE ? b : b & ~PLACE;
      const float v = rt_group_value<float>(p, a, b, by_logits, top);
      const bool inside = my_group < p.groups;
      const uint32_t mine = inside ? K::of(v) : 0u;
      int rank = 0;  // groups in front of mine: each of its lanes asks some of the others
      for (int j0 = 0; j0 < p.groups; j0 += share) {
        const int j = j0 + part;
        const uint32_t other = __shfl_sync(0xffffffffu, mine, (j << p.log_share) & 31);
        rank += j < p.groups && (other > mine || (other == mine && j < my_group)) ? 1 : 0;
      }
      for (int o = 1; o < share; o *= 2) rank += __shfl_xor_sync(0xffffffffu, rank, o);
      if (!(by_logits && p.group_top == 1)) {
        const uint32_t last = __ballot_sync(0xffffffffu, inside && rank == p.top_groups - 1);
        const uint32_t behind = __ballot_sync(0xffffffffu, inside && rank == p.top_groups);
        const float x = __shfl_sync(0xffffffffu, v, __ffs(last) - 1), y = __shfl_sync(0xffffffffu, v, __ffs(behind) - 1);
        const float off = 2 * (by_logits ? 0x1.4p-20f : tol);  // (the logits' scores are of whole logits)
        near = most_bias < 0x1p126f ? x - y <= off : !(x - y > off);  // two sums may both be beyond fp32
      }
      kept = rank < p.top_groups;
    }
    // Candidates: whatever is not below the value that top_k lanes' heads, and one more where it has to be looked at how near it comes,
    // reach; less what fp32 may be off by, so that fp64 finds among them whatever it may prefer.
    const bool check = !by_logits || !exact;
    const int rounds = check ? p.k + 1 : p.k;
    uint32_t from = 0, rest = 0;
    if (kept) {
      rest = key[0][0];
#pragma unroll
      for (int s = 1; s < S; ++s) rest = max(rest, key[s][0]);
      rest &= ~PLACE;
    }
#pragma unroll 1
    for (int r = 0; r < rounds; r += 3) {  // (one or two too many make candidates more, no fewer)
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        from = K::warp_max(rest);
        if (rest == from) rest = 0;
      }
    }
    if (!by_logits && from > K::NONE) from = K::of(K::value(from) - tol) & ~PLACE;
    from = max(from, (K::NONE + 1u) & ~PLACE);
    int n = 0;
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int d = 0; d < L; ++d) {
        const bool in = kept && key[s][d] >= from;
        const uint32_t who = __ballot_sync(0xffffffffu, in);
        if (who == 0) break;
        const int at = n + __popc(who & below);
        if (in && at < 32) list[at] = make_uint2((key[s][d] & PLACE) | backwards, key[s][d] & ~PLACE);
        n += __popc(who);
      }
    }
    int pick = -1, rank = lane;
    if (n <= 32 && !near) {
      // The order of the candidates: value, then expert.
      if (lane < 4) list[n + lane] = make_uint2(0u, 0u);
      __syncwarp();
      const uint2 mine = lane < n ? list[lane] : make_uint2(0u, 0u);
      const unsigned long long mine64 = ((unsigned long long)mine.y << 32) | mine.x;
      int in_front = 0;
      for (int i = 0; i < n; i += 4) {
        const uint4 two = *reinterpret_cast<const uint4*>(list + i), more = *reinterpret_cast<const uint4*>(list + i + 2);
        in_front += (((unsigned long long)two.y << 32) | two.x) > mine64;
        in_front += (((unsigned long long)two.w << 32) | two.z) > mine64;
        in_front += (((unsigned long long)more.y << 32) | more.x) > mine64;
        in_front += (((unsigned long long)more.w << 32) | more.z) > mine64;
      }
      if (lane < n) {
        pick = expert_of(mine.x);
        rank = in_front;
      }
      if (check) {
        // Each candidate against the one in front of it, those behind the last pick against that pick: a run of equal ones across the
        // last place may hide one that is larger.
        if (rank < p.k) place[rank] = mine;
        __syncwarp();
        bool close = false;
        if (lane < n && rank > 0) {
          const uint2 front = place[min(rank, p.k) - 1];
          close = by_logits ? mine.y == front.y : K::value(front.y) - K::value(mine.y) <= tol;
          if (close) close = !rt_equal<DT>(p, row, expert_of(front.x), pick, by_logits);  // a tie is in the right order
        }
        if (__any_sync(0xffffffffu, close)) rank = rt_rank_in_64(p, row, DT, by_logits, pick, n, lane);
      }
    } else {
      // Many equal values, or more picks than heads: a maximum at a time.
      if (!kept) {
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int i = 0; i < L; ++i) key[s][i] = 0u;
      }
      uint32_t last = 0;
#pragma unroll 1
      for (int r = 0; r < rounds && !near; ++r) {
        uint32_t head = key[0][0];
#pragma unroll
        for (int s = 1; s < S; ++s) head = max(head, key[s][0]);
        const uint32_t value = head & ~PLACE, m = K::warp_max(value);
        const bool owner = value == m;
        const uint32_t owners = __ballot_sync(0xffffffffu, owner);
        if (m <= K::NONE) break;
        const int first_owner = __ffs(owners) - 1;  // equal values: the lowest lane, and within a lane the lowest place
        const int e = __shfl_sync(0xffffffffu, first + (int)(PLACE - (head & PLACE)), first_owner);
        if (check && r > 0 && (by_logits ? m == last : K::value(last) - K::value(m) <= tol)) {
          const int f = __shfl_sync(0xffffffffu, pick, r - 1);
          if (r < p.k) {
            near = !rt_equal<DT>(p, row, e, f, by_logits);
          } else {  // behind the last pick: all that are left
            constexpr int HALF = V > 32 ? V / 2 : V;  // places to a mask
#pragma unroll
            for (int h = 0; h < V; h += HALF) {
              uint32_t left = 0;  // those of this lane that come as near
#pragma unroll
              for (int s = 0; s < HALF / L; ++s)
#pragma unroll
                for (int i = 0; i < L; ++i) {
                  const uint32_t of = key[h / L + s][i], v = of & ~PLACE;
                  if (by_logits ? v == last : K::value(last) - K::value(v) <= tol) left |= 1u << (PLACE - (of & PLACE) - h);
                }
              for (; left != 0 && !near; left &= left - 1) near = !rt_equal<DT>(p, row, first + h + __ffs(left) - 1, f, by_logits);
            }
            near = __any_sync(0xffffffffu, near);
          }
        }
        last = m;
        if (r == p.k) break;
        if (lane == r) pick = e;
        if (lane == first_owner) {
#pragma unroll
          for (int s = 0; s < S; ++s) {
            if (S == 1 || key[s][0] == head) {
#pragma unroll
              for (int i = 0; i + 1 < L; ++i) key[s][i] = key[s][i + 1];
              key[s][L - 1] = 0u;
            }
          }
        }
      }
      if (near) pick = rt_decide_in_64(p, row, DT, keys64, by_logits, lane);
    }
    const bool there = rank < p.k && pick >= 0;
    const float lp = there ? rt_load<DT>(row, pick) : -INFINITY;
    __syncwarp();  // the lists have been read
    // weights: a lane has the pick of place `rank`.  Divided by their sum they depend on differences of the logits only, which keeps them
    // exact where all the picked scores are tiny.
    float s;
    if (p.renormalize) {
      if (p.softmax || __all_sync(0xffffffffu, lp < -30.0f)) {
        const float most = K::value(K::warp_max(K::of(lp)));  // a NaN among the picks is on top
        s = there ? expf(lp - most) : 0.0f;
        if (need_top) s += top - top;  // the sum of all scores is NaN where a logit is NaN or +inf
      } else {
        // times 2^46, so that scores below fp32's range, as exp(l) in two factors, are in it
        const float e = expf(lp < -30.0f ? 0.5f * lp : -lp);
        s = lp < -30.0f ? e * (e * 0x1p46f) : __fdividef(0x1p46f, 1.0f + e);
        if (!there) s = 0.0f;
      }
      float all = s;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      s = __fdividef(s, all);
    } else {
      s = p.softmax ? expf(lp - top) * inv_sum : __fdividef(1.0f, 1.0f + expf(-lp));
    }
    if (rank < p.k) {
      const long long at = (long long)t * p.k + rank;
      p.experts[at] = pick;
      p.weights[at] = there ? s * p.scale : 0.0f;
    }
  }
}

}  // namespace qg
