// Host side of the operators around the experts' products (qgemm_moe_*, qgemm_swiglu_act_quant): argument validation, choice
// of launch shapes.  The exported functions are declared and documented in include/qgemm.h.
#include "../../include/qgemm.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "host_common.cuh"
#include "moe_blocks.cuh"
#include "moe_route.cuh"
#include "moe_rows.cuh"
#include "swiglu_quant.cuh"

namespace {

using namespace qgh;

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

constexpr int kMaxDevices = 64;
static_assert(QGEMM_MOE_MAX_EXPERTS == qg::RT_MAX_E && QGEMM_MOE_MAX_EXPERTS == qg::MB_MAX_E && QGEMM_MOE_MAX_TOP_K == qg::RT_MAX_K &&
                  QGEMM_MOE_MAX_GROUPS == qg::RT_MAX_GROUPS,
              "the limits that the header states are the kernels'");

// A persistent kernel: as many blocks as the SMs hold, or as many as there are rows for.  `resident`: blocks per SM by device, once asked.
template <typename P>
int launch_resident(void (*kernel)(P), std::atomic<int>* resident, const P& p, int64_t blocks, int threads, int smem, int sms, cudaStream_t s) {
  int dev = 0, per_sm = 0;
  CUDA_OK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return fail("device index %d out of range", dev);
  if ((per_sm = resident[dev].load(std::memory_order_acquire)) == 0) {
    CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    CUDA_OK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem));
    if (per_sm < 1) return fail("a kernel of %d threads and %d bytes of shared memory does not fit on an SM", threads, smem);
    resident[dev].store(per_sm, std::memory_order_release);
  }
  return launch_pdl(kernel, (int)std::min<int64_t>(blocks, (int64_t)per_sm * sms), threads, smem, s, p);
}
template <int TPR, int KEEP, bool BF16>
int launch_swiglu(const qg::SwigluQuantParams& p, int sms, cudaStream_t s) {
  static std::atomic<int> resident[kMaxDevices];
  constexpr int block = qg::sq_block(TPR), rows = block / TPR;
  return launch_resident(qg::swiglu_quant_kernel<TPR, KEEP, BF16>, resident, p, (p.M + rows - 1) / rows, block, qg::sq_smem_bytes(TPR, KEEP), sms, s);
}
template <int TPR, int KEEP, bool BF16>
int launch_dispatch(const qg::MoeActQuantParams& p, int sms, cudaStream_t s) {
  static std::atomic<int> resident[kMaxDevices];
  constexpr int block = qg::mq_block(TPR), rows = block / TPR;
  return launch_resident(qg::moe_act_quant_kernel<TPR, KEEP, BF16>, resident, p, (p.T + rows - 1) / rows, block, qg::mq_smem_bytes(TPR, KEEP), sms, s);
}

template <int DT, int V, bool VEC>
int launch_route(const qg::MoeRouteParams& p, int sms, cudaStream_t s) {
  // More blocks than the SMs hold, so that one that has a token to decide in fp64 is not waited for with its others; but what a warp does
  // once is worth 50 instructions a token.  us, 8 / 12 / 24 blocks per SM: 16384 x 256 22.0 / 21.7 / 21.8, 16384 x 64 9.4 / 8.5 / 9.8, 16384 x
  // 128 15.2 / 13.8 / 14.9, 9000 x 384 16.5 / 18.1 / 19.5; as many as they hold (7) 23.7 for the first.
  const int64_t blocks = std::min<int64_t>((p.T + qg::RT_WARPS - 1) / qg::RT_WARPS, (V <= 8 ? 12ll : 8ll) * sms);
  return launch_pdl(qg::moe_route_kernel<DT, V, VEC>, (int)blocks, qg::RT_WARPS * 32, qg::rt_smem_bytes(p.E), s, p);
}
template <int DT, bool VEC>
int launch_route(const qg::MoeRouteParams& p, int v, int sms, cudaStream_t s) {
  switch (v) {
    case 1: return launch_route<DT, 1, VEC>(p, sms, s);
    case 2: return launch_route<DT, 2, VEC>(p, sms, s);
    case 4: return launch_route<DT, 4, VEC>(p, sms, s);
    case 8: return launch_route<DT, 8, VEC>(p, sms, s);
    case 16: return launch_route<DT, 16, VEC>(p, sms, s);
    case 32: return launch_route<DT, 32, VEC>(p, sms, s);
    default: return launch_route<DT, 64, false>(p, sms, s);  // some 600 experts and more in groups that leave lanes idle
  }
}
template <int DT>
int launch_route(qg::MoeRouteParams p, int sms, cudaStream_t s) {
  p.log_share = 0;
  while ((2 << p.log_share) * p.groups <= 32) ++p.log_share;
  p.per_lane = (p.group_n + (1 << p.log_share) - 1) >> p.log_share;
  int v = 1;
  while (v < p.per_lane) v *= 2;
  // A lane's logits in pieces of up to 16 bytes where every row keeps that alignment and no lane has some of its places filled only.
  const int bytes = std::min(16, v * (DT == qg::RT_F32 ? 4 : 2));
  const bool vec = v <= 32 && p.group_n % v == 0 && (int64_t)p.E * (DT == qg::RT_F32 ? 4 : 2) % bytes == 0 && aligned(p.logits, bytes);
  if (vec) p.per_lane = v;
  return vec ? launch_route<DT, true>(p, v, sms, s) : launch_route<DT, false>(p, v, sms, s);
}

// One cluster of `ctas` CTAs.
template <int WARPS>
int launch_blocks(const qg::MoeBlocksParams& p, int ctas, cudaStream_t s) {
  auto kernel = qg::moe_blocks_kernel<WARPS>;
  static std::atomic<bool> ready[kMaxDevices];  // shared memory and clusters of more than eight are allowed
  int dev = 0;
  CUDA_OK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return fail("device index %d out of range", dev);
  if (!ready[dev].load(std::memory_order_acquire)) {
    CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    ready[dev].store(true, std::memory_order_release);
  }
  return launch_pdl_clusters(kernel, ctas, ctas, WARPS * 32, qg::mb_smem_bytes(WARPS, p.E), s, p);
}

}  // namespace

extern "C" {

int qgemm_moe_route(const void* logits, const float* bias, float* weights, int32_t* experts, int64_t T, int64_t E, int64_t top_k,
                    int64_t num_groups, int64_t top_groups, int group_top, int scoring, int renormalize, float scale, int logits_dtype,
                    void* stream) {
  if (T < 0 || T > (1ll << 30)) return fail("qgemm_moe_route: 0 to 2^30 tokens (got %lld)", (long long)T);
  if (E < 1 || E > QGEMM_MOE_MAX_EXPERTS) return fail("qgemm_moe_route: 1 to %d experts (got %lld)", QGEMM_MOE_MAX_EXPERTS, (long long)E);
  if (num_groups < 1 || num_groups > QGEMM_MOE_MAX_GROUPS || E % num_groups != 0)
    return fail("qgemm_moe_route: num_groups must be 1 to %d and divide the number of experts (got %lld groups, %lld experts)",
                QGEMM_MOE_MAX_GROUPS, (long long)num_groups, (long long)E);
  if (top_groups < 1 || top_groups > num_groups)
    return fail("qgemm_moe_route: top_groups must be 1 to num_groups (got %lld of %lld)", (long long)top_groups, (long long)num_groups);
  if (top_k < 1 || top_k > QGEMM_MOE_MAX_TOP_K || top_k > E / num_groups * top_groups)
    return fail("qgemm_moe_route: top_k must be 1 to %d and no more than the %lld experts of top_groups groups (got %lld)", QGEMM_MOE_MAX_TOP_K,
                (long long)(E / num_groups * top_groups), (long long)top_k);
  if (group_top != 1 && group_top != 2) return fail("qgemm_moe_route: group_top must be 1 or 2 (got %d)", group_top);
  if (scoring != QGEMM_ROUTE_SOFTMAX && scoring != QGEMM_ROUTE_SIGMOID) return fail("qgemm_moe_route: unknown scoring %d", scoring);
  if (logits_dtype != QGEMM_DT_F16 && logits_dtype != QGEMM_DT_BF16 && logits_dtype != QGEMM_DT_F32)
    return fail("qgemm_moe_route: logits_dtype must be F16, BF16 or F32 (got %d)", logits_dtype);
  if (T == 0) return 0;
  if (logits == nullptr || weights == nullptr || experts == nullptr) return fail("qgemm_moe_route: null pointer");
  if (!aligned(logits, logits_dtype == QGEMM_DT_F32 ? 4 : 2) || !aligned(bias, 4) || !aligned(weights, 4) || !aligned(experts, 4))
    return fail("qgemm_moe_route: pointers must be aligned to their elements");
  int sms = 0;
  if (ensure_device(&sms)) return -1;
  qg::MoeRouteParams p;
  p.logits = logits;
  p.bias = bias;
  p.weights = weights;
  p.experts = experts;
  p.T = T;
  p.E = (int)E;
  p.k = (int)top_k;
  p.groups = top_groups == num_groups ? 1 : (int)num_groups;  // all groups stay: nothing to choose
  p.group_n = (int)(E / p.groups);
  p.top_groups = p.groups == 1 ? 1 : (int)top_groups;
  p.group_top = group_top;
  p.softmax = scoring == QGEMM_ROUTE_SOFTMAX;
  p.renormalize = renormalize != 0;
  p.scale = scale;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (logits_dtype == QGEMM_DT_F32) return launch_route<qg::RT_F32>(p, sms, s);
  return logits_dtype == QGEMM_DT_BF16 ? launch_route<qg::RT_BF16>(p, sms, s) : launch_route<qg::RT_F16>(p, sms, s);
}

int64_t qgemm_moe_block_count(int64_t entries, int64_t num_experts, int64_t block_M) {
  if (entries <= 0 || num_experts <= 0 || block_M <= 0) return 0;
  const int64_t n = std::min(entries, num_experts);
  return n + (entries - n) / block_M;
}

int qgemm_moe_blocks(const int32_t* experts, int32_t* block_metadata, int32_t* rows, int32_t* sizes, int64_t entries, int64_t num_experts,
                     int64_t block_M, void* stream) {
  if (entries < 0 || entries > (1ll << 30)) return fail("qgemm_moe_blocks: 0 to 2^30 entries (got %lld)", (long long)entries);
  if (num_experts < 1 || num_experts > QGEMM_MOE_MAX_EXPERTS) return fail("qgemm_moe_blocks: 1 to %d experts (got %lld)", QGEMM_MOE_MAX_EXPERTS, (long long)num_experts);
  if (block_M < 1 || block_M > QGEMM_MOE_MAX_BLOCK_M)
    return fail("qgemm_moe_blocks: block_M must be 1 to %d (got %lld)", QGEMM_MOE_MAX_BLOCK_M, (long long)block_M);
  if (qgemm_moe_block_count(entries, num_experts, block_M) > QGEMM_MOE_MAX_BLOCKS)
    return fail("qgemm_moe_blocks: no more than %d blocks (got %lld entries in blocks of %lld)", QGEMM_MOE_MAX_BLOCKS, (long long)entries, (long long)block_M);
  if (sizes == nullptr || (entries > 0 && (experts == nullptr || block_metadata == nullptr || rows == nullptr)))
    return fail("qgemm_moe_blocks: null pointer");
  if (!aligned(experts, 4) || !aligned(block_metadata, 4) || !aligned(rows, 4) || !aligned(sizes, 4))
    return fail("qgemm_moe_blocks: pointers must be 4-byte aligned");
  int sms = 0;
  if (ensure_device(&sms)) return -1;
  qg::MoeBlocksParams p;
  p.experts = experts;
  p.meta = block_metadata;
  p.rows = rows;
  p.sizes = sizes;
  p.R = (int)entries;
  p.E = (int)num_experts;
  p.block_m = (int)block_M;
  p.blocks = (int)qgemm_moe_block_count(entries, num_experts, block_M);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // us, this form / the general one: 8 picks 1.5 / 3.5, 128 3.2 / 3.6 (256 experts).
  if (entries > 0 && entries <= qg::MB_FEW)
    return launch_pdl(qg::moe_blocks_few_kernel, 1, (int)((std::max(entries, num_experts) + 31) / 32 * 32), 0, st, p);
  // As many warps as keep every pick in a register, from 4096 picks on in clusters: by more CTAs a warp's walk is shorter and the sums over
  // CTAs longer.  us, CTAs x warps: 2048 picks 1 x 16 4.2, 2 x 16 4.9, 1 x 32 4.7; 8000 8 x 16 5.0, 4 x 16 5.3, 1 x 16 7.3; 16000 8 x 16 5.3,
  // 16 x 16 5.4; 32768 16 x 16 5.9, 8 x 16 6.1, 16 x 32 6.5; 131072 16 x 32 8.7, 16 x 16 9.7.
  const bool many = entries > 16 * 512 * qg::MB_ITEMS && qg::mb_smem_bytes(32, p.E) <= 227 * 1024;
  const int ctas = entries <= 4096 ? 1 : entries <= 24576 ? 8 : qg::MB_MAX_CLUSTER;
  return many ? launch_blocks<32>(p, ctas, st) : launch_blocks<16>(p, ctas, st);
}

int qgemm_moe_act_quant(const void* X, const int32_t* rows, int8_t* Y, float* S, int64_t T, int64_t N, int64_t top_k, int x_dtype,
                        int round_scale, void* stream) {
  if (T < 0 || N <= 0 || (N % 8) != 0)
    return fail("qgemm_moe_act_quant: T >= 0 and N a positive multiple of 8 required (got T=%lld, N=%lld)", (long long)T, (long long)N);
  if (N > (1ll << 30)) return fail("qgemm_moe_act_quant: N too large (%lld)", (long long)N);
  if (top_k < 1 || T > (1ll << 30) || T * top_k > (1ll << 30))
    return fail("qgemm_moe_act_quant: top_k >= 1 and no more than 2^30 rows required (got T=%lld, top_k=%lld)", (long long)T, (long long)top_k);
  if (x_dtype != QGEMM_DT_F16 && x_dtype != QGEMM_DT_BF16) return fail("qgemm_moe_act_quant: x_dtype must be F16 or BF16 (got %d)", x_dtype);
  if (T == 0) return 0;
  if (X == nullptr || rows == nullptr || Y == nullptr || S == nullptr) return fail("qgemm_moe_act_quant: null pointer");
  if (!aligned16(X) || !aligned(Y, 8) || !aligned(S, 4) || !aligned(rows, 4))
    return fail("qgemm_moe_act_quant: X must be 16-byte, Y 8-byte, S and rows 4-byte aligned");
  int sms = 0;
  if (ensure_device(&sms)) return -1;
  qg::MoeActQuantParams p;
  p.X = static_cast<const uint4*>(X);
  p.rows = rows;
  p.Y = Y;
  p.S = S;
  p.T = T;
  p.N = (int)N;
  p.k = (int)top_k;
  p.round_scale = round_scale != 0;
  // The fewest threads per row that hold it with eight chunks each: a warp needs no barrier for the row's maximum, and several chunks in
  // flight per thread do for few rows too.  us, threads x chunks: 16 tokens of 7168 128 x 8 2.8, 256 x 4 2.9, 512 x 2 3.0; 600 of 2048
  // 32 x 8 3.5, 64 x 4 3.7, 128 x 2 3.4; 4001 of 4096 64 x 8 12.9, 128 x 4 12.7, 256 x 2 15.0; 4096 of 8192 to one place 128 x 8 17.6, 256 x 4 20.9.
  const int64_t chunks = N / 8;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto launch_type = [&](auto bf16) {
    constexpr bool BF16 = decltype(bf16)::value;
    if (chunks <= 32) return launch_dispatch<32, 1, BF16>(p, sms, st);
    if (chunks <= 64) return launch_dispatch<32, 2, BF16>(p, sms, st);
    if (chunks <= 128) return launch_dispatch<32, 4, BF16>(p, sms, st);
    if (chunks <= 256) return launch_dispatch<32, 8, BF16>(p, sms, st);
    if (chunks <= 512) return launch_dispatch<64, 8, BF16>(p, sms, st);
    if (chunks <= 1024) return launch_dispatch<128, 8, BF16>(p, sms, st);
    if (chunks <= 2048) return launch_dispatch<256, 8, BF16>(p, sms, st);
    return launch_dispatch<512, 8, BF16>(p, sms, st);  // above 32768 elements the rest of a row is read a second time
  };
  return x_dtype == QGEMM_DT_BF16 ? launch_type(std::true_type{}) : launch_type(std::false_type{});
}

int qgemm_swiglu_act_quant(const void* X, int8_t* Y, float* S, int64_t M, int64_t F, int x_dtype, int round_scale, void* stream) {
  if (M < 0 || F <= 0 || (F % 8) != 0)
    return fail("qgemm_swiglu_act_quant: M >= 0 and F a positive multiple of 8 required (got M=%lld, F=%lld)", (long long)M, (long long)F);
  if (F > (1ll << 29)) return fail("qgemm_swiglu_act_quant: F too large (%lld)", (long long)F);
  if (x_dtype != QGEMM_DT_F16 && x_dtype != QGEMM_DT_BF16) return fail("qgemm_swiglu_act_quant: x_dtype must be F16 or BF16 (got %d)", x_dtype);
  if (M == 0) return 0;
  if (X == nullptr || Y == nullptr || S == nullptr) return fail("qgemm_swiglu_act_quant: null pointer");
  if (!aligned16(X) || !aligned(Y, 8) || !aligned(S, 4))
    return fail("qgemm_swiglu_act_quant: X must be 16-byte, Y 8-byte and S 4-byte aligned");
  int sms = 0;
  if (ensure_device(&sms)) return -1;
  qg::SwigluQuantParams p;
  p.X = static_cast<const uint4*>(X);
  p.Y = Y;
  p.S = S;
  p.M = M;
  p.F = (int)F;
  p.round_scale = round_scale != 0;
  const int64_t chunks = F / 8;
  // Threads per row and chunks of eight elements per thread.  While the rows leave threads idle, the fewest chunks that do not take more
  // than 450 threads per SM; otherwise the shape with the fewest empty places, and of those the one with the fewest threads per row,
  // whose maximum costs the least (a warp needs no barrier).  us, threads x chunks: 128 rows of 2048 256 x 1 2.5, 64 x 4 3.3, 32 x 8 4.0; 300 of
  // 4096 256 x 2 4.05, 128 x 4 4.1, 64 x 8 4.6; 1200 of 768 64 x 2 3.8, 32 x 3 3.3; 1500 of 2048 32 x 8 5.9, 64 x 4 6.1; 32768 of 2048
  // 32 x 8 63, 64 x 4 71; 8000 of 4096 64 x 8 34, 128 x 4 41; 5000 of 7168 128 x 7 41, 128 x 8 44, 256 x 4 52; 4000 of 14336 256 x 7 72,
  // 512 x 4 88.
  int keep = 0, tpr = 0;
  for (int k = 1; k <= 4 && keep == 0; k *= 2) {
    int t = 32;
    while (t < 512 && chunks > (int64_t)t * k) t *= 2;
    if (M * t <= 450ll * sms && chunks <= (int64_t)t * k) {
      keep = (int)((chunks + t - 1) / t);
      tpr = t;
    }
  }
  if (keep == 0) {
    keep = 8;
    tpr = 512;
    for (int t = 512; t >= 32; t /= 2) {
      const int64_t k = (chunks + t - 1) / t;
      if (k <= 8 && k * t <= (int64_t)keep * tpr) { keep = (int)k; tpr = t; }
    }
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto launch_keep = [&](auto bf16, auto keep_) {
    constexpr bool BF16 = decltype(bf16)::value;
    constexpr int KEEP = decltype(keep_)::value;
    switch (tpr) {
      case 32: return launch_swiglu<32, KEEP, BF16>(p, sms, st);
      case 64: return launch_swiglu<64, KEEP, BF16>(p, sms, st);
      case 128: return launch_swiglu<128, KEEP, BF16>(p, sms, st);
      case 256: return launch_swiglu<256, KEEP, BF16>(p, sms, st);
      default: return launch_swiglu<512, KEEP, BF16>(p, sms, st);
    }
  };
  auto launch_type = [&](auto bf16) {
    switch (keep) {
      case 1: return launch_keep(bf16, std::integral_constant<int, 1>{});
      case 2: return launch_keep(bf16, std::integral_constant<int, 2>{});
      case 3: return launch_keep(bf16, std::integral_constant<int, 3>{});
      case 4: return launch_keep(bf16, std::integral_constant<int, 4>{});
      case 5: return launch_keep(bf16, std::integral_constant<int, 5>{});
      case 6: return launch_keep(bf16, std::integral_constant<int, 6>{});
      case 7: return launch_keep(bf16, std::integral_constant<int, 7>{});
      default: return launch_keep(bf16, std::integral_constant<int, 8>{});
    }
  };
  return x_dtype == QGEMM_DT_BF16 ? launch_type(std::true_type{}) : launch_type(std::false_type{});
}

int qgemm_moe_combine(const void* Y, const int32_t* rows, const float* weights, const void* base, void* out, int64_t R, int64_t T, int64_t N,
                      int64_t top_k, int dtype, void* stream) {
  if (T < 0 || R < 0 || N <= 0 || (N % 8) != 0)
    return fail("qgemm_moe_combine: T, R >= 0 and N a positive multiple of 8 required (got T=%lld, R=%lld, N=%lld)", (long long)T, (long long)R,
                (long long)N);
  if (N > (1ll << 30) || R > (1ll << 31)) return fail("qgemm_moe_combine: dimension too large (R=%lld, N=%lld)", (long long)R, (long long)N);
  if (top_k < 1 || T > (1ll << 30) || T * top_k > (1ll << 30))
    return fail("qgemm_moe_combine: top_k >= 1 and no more than 2^30 entries required (got T=%lld, top_k=%lld)", (long long)T, (long long)top_k);
  if (dtype != QGEMM_DT_F16 && dtype != QGEMM_DT_BF16) return fail("qgemm_moe_combine: dtype must be F16 or BF16 (got %d)", dtype);
  if (T == 0) return 0;
  if ((Y == nullptr && R > 0) || rows == nullptr || weights == nullptr || out == nullptr) return fail("qgemm_moe_combine: null pointer");
  if (!aligned16(Y) || !aligned16(base) || !aligned16(out) || !aligned(rows, 4) || !aligned(weights, 4))
    return fail("qgemm_moe_combine: Y, base and out must be 16-byte, rows and weights 4-byte aligned");
  int sms = 0;
  if (ensure_device(&sms)) return -1;
  qg::MoeCombineParams p;
  p.Y = static_cast<const uint4*>(Y);
  p.rows = rows;
  p.weights = weights;
  p.base = static_cast<const uint4*>(base);
  p.out = static_cast<uint4*>(out);
  p.R = R;
  p.T = T;
  p.N = (int)N;
  p.k = (int)top_k;
  p.parts = (int)((N / 8 + qg::MC_THREADS - 1) / qg::MC_THREADS);
  const int64_t grid = T * p.parts;
  if (grid > 0x7fffffffll) return fail("qgemm_moe_combine: too many tokens (%lld of %lld)", (long long)T, (long long)N);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto launch = [&](auto kernel) { return launch_pdl(kernel, (int)grid, qg::MC_THREADS, 0, s, p); };
  const bool bf16 = dtype == QGEMM_DT_BF16;
  if (top_k <= 2) return bf16 ? launch(qg::moe_combine_kernel<true, 2>) : launch(qg::moe_combine_kernel<false, 2>);
  if (top_k <= 4) return bf16 ? launch(qg::moe_combine_kernel<true, 4>) : launch(qg::moe_combine_kernel<false, 4>);
  return bf16 ? launch(qg::moe_combine_kernel<true, 8>) : launch(qg::moe_combine_kernel<false, 8>);
}

}  // extern "C"
