// From routed experts to the tables of the grouped product, for sm_100a: a stable counting sort of the T * top_k picks by expert.
//
//   sizes[e]   = picks of expert e
//   rows[i]    = place of pick i when the picks are stacked expert by expert, in their own order within one
//   block table: one entry (expert, first row, valid rows) per block_M rows of an expert, as the grouped product takes it
//
// A few hundred thousand 4-byte values: what costs is latency, so everything is one launch, of one cluster of up to 16 CTAs.
// Each warp counts its own stretch of the picks in shared memory, the counts are summed over warps and, through distributed
// shared memory, over CTAs, and a second walk over the same stretch hands out the places: a vote of the lanes with the
// same expert gives the place within 32 picks, the warp's own counter that of the 32.
#pragma once

#include "common.cuh"

namespace qg {

constexpr int MB_MAX_E = 1024;
constexpr int MB_MAX_THREADS = 1024;
constexpr int MB_MAX_CLUSTER = 16;

struct MoeBlocksParams {
  const int* experts;  // [R]
  int* meta;           // [blocks, 3]
  int* rows;           // [R]
  int* sizes;          // [E]
  int R, E, block_m, blocks;
};

__host__ __device__ constexpr int mb_smem_bytes(int threads, int E) { return ((threads / 32 + 3) * (E + 1) + 64) * 4; }

__device__ __forceinline__ int ld_cluster(const int* p, uint32_t rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_u32(smem_u32(p), rank)) : "memory");
  return v;
}

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

__global__ void __launch_bounds__(MB_MAX_THREADS) moe_blocks_kernel(const MoeBlocksParams p) {
  extern __shared__ int mb_smem[];
  const int threads = blockDim.x, warps = threads >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int B = p.E + 1;  // buckets: the experts, and the dropped picks
  int* count = mb_smem;              // [warps][B]: this warp's picks, then its next place
  int* mine = count + warps * B;     // [B] this CTA's picks
  int* first = mine + B;             // [B] first row of a bucket
  int* block_end = first + B;        // [B] blocks of the buckets up to and with this one
  int* warp_rows = block_end + B;    // [32]
  int* warp_blocks = warp_rows + 32; // [32]
  const uint32_t ctas = cluster_nctarank(), cta = cluster_ctarank();
  for (int i = threadIdx.x; i < warps * B; i += threads) count[i] = 0;
  pdl_wait();
  pdl_launch_dependents();
  __syncthreads();
  const long long walkers = (long long)ctas * warps;
  const long long stretch = ((p.R + walkers - 1) / walkers + 31) / 32 * 32;
  const int begin = (int)min((long long)p.R, (cta * (long long)warps + warp) * stretch), end = (int)min((long long)p.R, begin + stretch);
  int* my_count = count + warp * B;
  auto bucket = [&](int i) {
    const int e = ld_written(p.experts + i);
    return e >= 0 && e < p.E ? e : p.E;
  };
  for (int i = begin + lane; i < end; i += 32) atomicAdd(my_count + bucket(i), 1);
  __syncthreads();
  for (int e = threadIdx.x; e < B; e += threads) {
    int sum = 0;
    for (int w = 0; w < warps; ++w) {
      const int c = count[w * B + e];
      count[w * B + e] = sum;
      sum += c;
    }
    mine[e] = sum;
  }
  cluster_sync_all();
  // Buckets dealt to the threads in runs, so that sums over a thread's run and over the threads below it give first rows.
  const int per = (B + threads - 1) / threads, e0 = min(B, (int)threadIdx.x * per), e1 = min(B, e0 + per);
  int run_rows = 0, run_blocks = 0;
  for (int e = e0; e < e1; ++e) {
    int all = 0, before = 0;
    for (uint32_t c = 0; c < ctas; ++c) {
      const int n = ld_cluster(mine + e, c);
      if (c < cta) before += n;
      all += n;
    }
    if (cta == 0 && e < p.E) p.sizes[e] = all;
    first[e] = before;          // for now: rows of this bucket in the CTAs in front
    block_end[e] = all;         // for now: rows of this bucket
    run_rows += all;
    run_blocks += e < p.E ? (all + p.block_m - 1) / p.block_m : 0;
  }
  int all_rows, all_blocks;
  int below_rows = warp_sum_below(run_rows, lane, all_rows), below_blocks = warp_sum_below(run_blocks, lane, all_blocks);
  if (lane == 0) { warp_rows[warp] = all_rows; warp_blocks[warp] = all_blocks; }
  __syncthreads();
  for (int w = 0; w < warp; ++w) { below_rows += warp_rows[w]; below_blocks += warp_blocks[w]; }
  for (int e = e0; e < e1; ++e) {
    const int all = block_end[e], before = first[e];
    first[e] = below_rows;
    for (int w = 0; w < warps; ++w) count[w * B + e] += below_rows + before;
    below_rows += all;
    below_blocks += e < p.E ? (all + p.block_m - 1) / p.block_m : 0;
    block_end[e] = below_blocks;
  }
  __syncthreads();
  // second walk: places
  for (int i = begin + lane; i - lane < end; i += 32) {
    const bool there = i < end;
    const uint32_t active = __ballot_sync(0xffffffffu, there);
    if (there) {
      const int e = bucket(i);
      const uint32_t same = __match_any_sync(active, e);
      const int place = my_count[e] + __popc(same & ((1u << lane) - 1u));
      __syncwarp(active);
      if (lane == 31 - __clz(same)) my_count[e] = place + 1;
      p.rows[i] = e < p.E ? place : -2 - place;
    }
    __syncwarp();
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
  cluster_sync_all();  // no CTA's shared memory goes while another may still read it
}

}  // namespace qg
