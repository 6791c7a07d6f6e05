// From routed experts to the tables of the grouped product, for sm_100a: a stable counting sort of the T * top_k picks by expert.
//
//   sizes[e]   = picks of expert e
//   rows[i]    = place of pick i when the picks are stacked expert by expert, in their own order within one
//   block table: one entry (expert, first row, valid rows) per block_M rows of an expert, as the grouped product takes it
//
// A few hundred thousand 4-byte values: what costs is latency, and issue on the few SMs that take part.  Everything is one
// launch, of one cluster of up to 16 CTAs.  A warp walks its stretch of the picks once, 32 at a time: the lanes leave their bits in a word per
// expert in shared memory, which gives each the lanes with the same expert, and the warp's own counter gives the rank among the warp's
// picks, which stays in a register with the pick.  (__match_any_sync gives the lanes in one instruction, which takes 70 cycles of
// the SM; a vote for each bit of the index takes 45 instructions.)  The counters are then summed over the warps, the CTAs (through
// distributed shared memory) and the experts, two threads to an expert, and a pick's place is three sums.
#pragma once

#include "common.cuh"

namespace qg {

constexpr int MB_MAX_E = 1024;
constexpr int MB_MAX_CLUSTER = 16;

struct MoeBlocksParams {
  const int* experts;  // [R]
  int* meta;           // [blocks, 3]
  int* rows;           // [R]
  int* sizes;          // [E]
  int R, E, block_m, blocks;
};

constexpr int MB_ITEMS = 8;  // picks of a lane that stay in registers
constexpr int MB_SHARE = 2;  // threads to an expert

__host__ __device__ constexpr int mb_smem_bytes(int warps, int E) { return ((2 * warps + 4) * (E + 1) + 64) * 4; }

__device__ __forceinline__ int ld_cluster(const int* p, uint32_t rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_u32(smem_u32(p), rank)) : "memory");
  return v;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Sum over the warp's lanes below this one.
__device__ __forceinline__ int warp_sum_below(int v, int lane, int& all) {
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  all = __shfl_sync(0xffffffffu, x, 31);
  return x - v;
}

// Few picks: a pick's place is the number of picks that come before it, and an expert's first row the number of picks of
// lower experts, counted by comparing with all of them; one CTA, one thread per pick and one per expert.
constexpr int MB_FEW = 128;
__global__ void __launch_bounds__(1024) moe_blocks_few_kernel(const MoeBlocksParams p) {
  __shared__ __align__(16) uint32_t keys[MB_FEW + 4];  // expert * MB_FEW + place in the input; dropped picks as expert E
  __shared__ int warp_blocks[32], warp_end[32];
  const int threads = blockDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, i = threadIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  uint32_t key = 0xffffffffu;
  if (i < p.R) {
    const int v = ld_written(p.experts + i);
    key = (uint32_t)(v >= 0 && v < p.E ? v : p.E) * MB_FEW + i;
  }
  if (i < (p.R + 3) / 4 * 4) keys[i] = key;
  __syncthreads();
  const int quads = (p.R + 3) / 4;
  const uint32_t hi = (uint32_t)(i + 1) * MB_FEW;  // behind this thread's expert
  int place = 0, up_to = 0;
  for (int q = 0; q < quads; ++q) {
    const uint4 k = reinterpret_cast<const uint4*>(keys)[q];
    if (warp * 32 < p.R) place += (k.x < key) + (k.y < key) + (k.z < key) + (k.w < key);
    up_to += (k.x < hi) + (k.y < hi) + (k.z < hi) + (k.w < hi);
  }
  if (i < p.R) p.rows[i] = key < (uint32_t)p.E * MB_FEW ? place : -2 - place;
  if (lane == 31) warp_end[warp] = up_to;
  __syncthreads();
  int before = __shfl_up_sync(0xffffffffu, up_to, 1);
  if (lane == 0) before = warp > 0 ? warp_end[warp - 1] : 0;
  const int rows = i < p.E ? up_to - before : 0, mine = (rows + p.block_m - 1) / p.block_m;
  if (i < p.E) p.sizes[i] = rows;
  int all;
  int at = warp_sum_below(mine, lane, all);
  if (lane == 0) warp_blocks[warp] = all;
  __syncthreads();
  int total = 0;
  for (int w = 0; w < threads / 32; ++w) {
    const int n = warp_blocks[w];
    if (w < warp) at += n;
    total += n;
  }
  for (int b = 0; b < mine; ++b) {
    int* m = p.meta + 3 * (at + b);
    m[0] = i;
    m[1] = before + b * p.block_m;
    m[2] = min(p.block_m, rows - b * p.block_m);
  }
  for (int b = total + i; b < p.blocks; b += threads) {
    int* m = p.meta + 3 * b;
    m[0] = -1;
    m[1] = p.R;
    m[2] = 0;
  }
}

template <int WARPS>
__global__ void __launch_bounds__(WARPS * 32) moe_blocks_kernel(const MoeBlocksParams p) {
  extern __shared__ __align__(16) int mb_smem[];
  constexpr int threads = WARPS * 32, warps = WARPS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int B = p.E + 1;  // buckets: the experts, and the dropped picks
  int* count = mb_smem;              // [warps][B] picks of a warp, then those of the warps in front of it
  uint32_t* lanes = reinterpret_cast<uint32_t*>(count + warps * B);  // [warps][B] lanes of the 32 picks in hand; zero in between
  int* mine = count + 2 * warps * B; // [B] picks of this CTA
  int* first = mine + B;             // [B] first row of a bucket
  int* next = first + B;             // [B] first row of this CTA's picks of a bucket
  int* block_end = next + B;         // [B] blocks of the buckets up to and with this one
  int* warp_rows = block_end + B;    // [32]
  int* warp_blocks = warp_rows + 32; // [32]
  const uint32_t ctas = cluster_nctarank(), cta = cluster_ctarank();
  for (int i = threadIdx.x; i < 2 * warps * B / 4; i += threads) reinterpret_cast<int4*>(count)[i] = make_int4(0, 0, 0, 0);
  pdl_wait();
  pdl_launch_dependents();
  const long long walkers = (long long)ctas * warps;
  const long long stretch = ((p.R + walkers - 1) / walkers + 31) / 32 * 32;
  const int begin = (int)min((long long)p.R, (cta * (long long)warps + warp) * stretch), end = (int)min((long long)p.R, begin + stretch);
  int* my_count = count + warp * B;
  const uint32_t below = (1u << lane) - 1u;
  int e[MB_ITEMS], rank[MB_ITEMS];  // of the first MB_ITEMS * 32 picks; -1 beyond the end
  auto load = [&](int from, int (&b)[MB_ITEMS]) {
#pragma unroll
    for (int j = 0; j < MB_ITEMS; ++j) {
      const int i = from + 32 * j + lane;
      b[j] = -1;
      if (i < end) {
        const int v = ld_written(p.experts + i);
        b[j] = v >= 0 && v < p.E ? v : p.E;
      }
    }
  };
  uint32_t* my_lanes = lanes + warp * B;
  auto ranks = [&](int from, const int (&b)[MB_ITEMS], int (&r)[MB_ITEMS]) {
#pragma unroll
    for (int j = 0; j < MB_ITEMS; ++j) {
      if (from + 32 * j >= end) break;
      if (b[j] >= 0) atomicOr(my_lanes + b[j], 1u << lane);
      __syncwarp();
      uint32_t same = 0;
      if (b[j] >= 0) {
        same = my_lanes[b[j]];
        r[j] = my_count[b[j]] + __popc(same & below);
      }
      __syncwarp();
      if (same >> lane == 1u) {  // the last of them
        my_count[b[j]] = r[j] + 1;
        my_lanes[b[j]] = 0u;
      }
      __syncwarp();
    }
  };
  load(begin, e);
  __syncthreads();  // the counters are zero
  ranks(begin, e, rank);
  for (int from = begin + 32 * MB_ITEMS; from < end; from += 32 * MB_ITEMS) {  // longer stretches: the ranks wait in `rows`
    int b[MB_ITEMS], r[MB_ITEMS];
    load(from, b);
    ranks(from, b, r);
#pragma unroll
    for (int j = 0; j < MB_ITEMS; ++j)
      if (b[j] >= 0) p.rows[from + 32 * j + lane] = r[j];
  }
  __syncthreads();
  // Sums over the warps in front, and the CTA's picks.  MB_SHARE neighbouring lanes have a bucket, each a run of warps (or of CTAs).
  const int part = threadIdx.x & (MB_SHARE - 1);
  auto sum_below = [&](int v, int& all) {  // over the lanes of a bucket
    int x = v;
#pragma unroll
    for (int o = 1; o < MB_SHARE; o *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, x, o, MB_SHARE);
      if (part >= o) x += y;
    }
    all = __shfl_sync(0xffffffffu, x, MB_SHARE - 1, MB_SHARE);
    return x - v;
  };
  constexpr int RUN = WARPS / MB_SHARE;
  for (int b0 = 0; b0 < B; b0 += threads / MB_SHARE) {
    const int b = b0 + threadIdx.x / MB_SHARE;
    int* of = count + part * RUN * B + min(b, B - 1);
    int c[RUN], sum = 0, all;
#pragma unroll
    for (int w = 0; w < RUN; ++w) {
      c[w] = of[w * B];
      sum += c[w];
    }
    int at = sum_below(sum, all);
    if (b < B) {
#pragma unroll
      for (int w = 0; w < RUN; ++w) {
        of[w * B] = at;
        at += c[w];
      }
      if (part == 0) mine[b] = all;
    }
  }
  if (ctas > 1) cluster_sync_all();
  else __syncthreads();
  for (int b0 = 0; b0 < B; b0 += threads / MB_SHARE) {
    const int b = b0 + threadIdx.x / MB_SHARE;
    int before = 0, sum = 0, all_before, all;
    if (ctas > 1) {
      int c[MB_MAX_CLUSTER / MB_SHARE];
#pragma unroll
      for (int j = 0; j < MB_MAX_CLUSTER / MB_SHARE; ++j) {
        const uint32_t other = part + j * MB_SHARE;
        c[j] = b < B && other < ctas ? ld_cluster(mine + b, other) : 0;
      }
#pragma unroll
      for (int j = 0; j < MB_MAX_CLUSTER / MB_SHARE; ++j) {
        sum += c[j];
        if (part + j * MB_SHARE < cta) before += c[j];
      }
      sum_below(sum, all);
      sum_below(before, all_before);
    } else {
      all = b < B ? mine[b] : 0;
      all_before = 0;
    }
    if (b < B && part == 0) {
      first[b] = all;  // for now: rows of the bucket
      next[b] = all_before;
      if (cta == 0 && b < p.E) p.sizes[b] = all;
    }
  }
  if (ctas > 1) cluster_arrive();  // this CTA reads no other's shared memory from here on
  __syncthreads();
  // First rows: buckets dealt to the threads in runs.
  const int per = (B + threads - 1) / threads, e0 = min(B, (int)threadIdx.x * per), e1 = min(B, e0 + per);
  auto blocks_of = [&](int b, int rows) { return b < p.E ? (rows + p.block_m - 1) / p.block_m : 0; };
  int run_rows = 0, run_blocks = 0;
  for (int b = e0; b < e1; ++b) {
    run_rows += first[b];
    run_blocks += blocks_of(b, first[b]);
  }
  int all_rows, all_blocks;
  int below_rows = warp_sum_below(run_rows, lane, all_rows), below_blocks = warp_sum_below(run_blocks, lane, all_blocks);
  if (lane == 0) { warp_rows[warp] = all_rows; warp_blocks[warp] = all_blocks; }
  __syncthreads();
  if (e0 < e1) {
    for (int w = 0; w < warp; ++w) { below_rows += warp_rows[w]; below_blocks += warp_blocks[w]; }
    for (int b = e0; b < e1; ++b) {
      const int rows = first[b];
      first[b] = below_rows;
      next[b] += below_rows;
      below_rows += rows;
      below_blocks += blocks_of(b, rows);
      block_end[b] = below_blocks;
    }
  }
  __syncthreads();
  auto store = [&](int i, int b, int r) {
    const int place = r + my_count[b] + next[b];
    p.rows[i] = b < p.E ? place : -2 - place;
  };
#pragma unroll
  for (int j = 0; j < MB_ITEMS; ++j)
    if (e[j] >= 0) store(begin + 32 * j + lane, e[j], rank[j]);
  for (int from = begin + 32 * MB_ITEMS; from < end; from += 32 * MB_ITEMS) {
    int b[MB_ITEMS], r[MB_ITEMS];
    load(from, b);
#pragma unroll
    for (int j = 0; j < MB_ITEMS; ++j) r[j] = b[j] >= 0 ? ld_written(p.rows + from + 32 * j + lane) : 0;
#pragma unroll
    for (int j = 0; j < MB_ITEMS; ++j)
      if (b[j] >= 0) store(from + 32 * j + lane, b[j], r[j]);
  }
  // block table
  for (int b = (int)cta * threads + threadIdx.x; b < p.blocks; b += (int)ctas * threads) {
    int lo = 0, hi = p.E;  // the first expert whose blocks end behind b
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (block_end[mid] > b) hi = mid;
      else lo = mid + 1;
    }
    int g = -1, row = p.R, n = 0;
    if (lo < p.E) {
      const int done = (b - (lo > 0 ? block_end[lo - 1] : 0)) * p.block_m;
      g = lo;
      row = first[lo] + done;
      n = min(p.block_m, first[lo + 1] - row);
    }
    p.meta[3 * b] = g;
    p.meta[3 * b + 1] = row;
    p.meta[3 * b + 2] = n;
  }
  if (ctas > 1) cluster_wait();  // no CTA's shared memory goes while another may still read it
}

}  // namespace qg
