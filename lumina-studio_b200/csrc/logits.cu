// Penalties, token biases and a grammar mask on logits rows, and the argmax
// (the rules are declared in lumina_cuda.h).
//
// One cluster of CTAs per row; each CTA holds the token counts of its slice
// of the vocabulary in shared memory. It counts the row's history (shared
// atomics on integers: the order does not matter), then streams its slice
// once: read, adjust, write, and keep the largest value. Bound by those
// bytes; the argmax joins over distributed shared memory, so a row needs no
// second launch and no workspace.
#include <cooperative_groups.h>

#include "weights.cuh"

namespace lumina {

namespace {

namespace cg = cooperative_groups;

constexpr int LG_THREADS = 512;
constexpr int LG_CLUSTER = 8;
constexpr int LG_SLICE = 8192;  // tokens whose counts a CTA holds at once (8 bytes each)

// larger value first, then the smaller index; a NaN is the largest
__device__ __forceinline__ unsigned long long lg_key(float v, int i) {
  const unsigned u = __float_as_uint(v);
  const unsigned ord = (u & 0x7fffffffu) > 0x7f800000u ? 0xffffffffu
                       : v == 0.f                      ? 0x80000000u
                       : (u & 0x80000000u)             ? ~u
                                                       : (u | 0x80000000u);
  return ((unsigned long long)ord << 32) | (0xffffffffu - (unsigned)i);
}

__global__ void __launch_bounds__(LG_THREADS) logits_kernel(lumina_logits_args a, int per_cta) {
  extern __shared__ int sm[];
  int* count = sm;             // [slice] occurrences in the history
  int* bias = sm + LG_SLICE;   // [slice] 1 + index of the token's last bias entry
  __shared__ unsigned long long best_s[LG_THREADS / 32], cta_best;
  cg::cluster_group cl = cg::this_cluster();
  const int row = blockIdx.x / LG_CLUSTER, rank = (int)cl.block_rank();
  const int tid = threadIdx.x;
  const float* src = a.logits_dev + (size_t)row * a.ld;
  float* dst = a.out_dev + (size_t)row * a.ldo;
  const uint32_t* mask = a.mask_dev ? a.mask_dev + (size_t)row * a.mask_ld : nullptr;
  const bool hist = a.hist_start_dev != nullptr, biased = a.bias_start_dev != nullptr;
  const int h0 = hist ? a.hist_start_dev[row] : 0, h1 = hist ? a.hist_start_dev[row + 1] : 0;
  const int b0 = biased ? a.bias_start_dev[row] : 0, b1 = biased ? a.bias_start_dev[row + 1] : 0;
  const float rep = a.repeat_dev ? a.repeat_dev[row] : 1.f;
  const float fr = a.frequency_dev ? a.frequency_dev[row] : 0.f, pr = a.presence_dev ? a.presence_dev[row] : 0.f;
  unsigned long long best = 0;
  const int v0 = rank * per_cta, v1 = min(a.vocab, v0 + per_cta);
  for (int s0 = v0; s0 < v1; s0 += LG_SLICE) {
    const int n = min(LG_SLICE, v1 - s0);
    for (int i = tid; i < n; i += LG_THREADS) {
      count[i] = 0;
      bias[i] = 0;
    }
    __syncthreads();
    for (int i = h0 + tid; i < h1; i += LG_THREADS) {
      const unsigned t = (unsigned)(a.hist_tok_dev[i] - s0);
      if (t < (unsigned)n) atomicAdd(&count[t], 1);
    }
    for (int i = b0 + tid; i < b1; i += LG_THREADS) {
      const unsigned t = (unsigned)(a.bias_tok_dev[i] - s0);
      if (t < (unsigned)n) atomicMax(&bias[t], i - b0 + 1);
    }
    __syncthreads();
    for (int i = tid; i < n; i += LG_THREADS) {
      float l = src[s0 + i];
      const int c = count[i], b = bias[i];
      if (c) {
        l = l > 0.f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
        l = __fsub_rn(__fsub_rn(l, __fmul_rn(fr, (float)c)), pr);
      }
      if (b) l = __fadd_rn(l, a.bias_val_dev[b0 + b - 1]);
      if (mask && !((mask[(s0 + i) >> 5] >> ((s0 + i) & 31)) & 1u)) l = -INFINITY;
      dst[s0 + i] = l;
      best = max(best, lg_key(l, s0 + i));
    }
    __syncthreads();
  }
  if (!a.argmax_dev) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & 31) == 0) best_s[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < LG_THREADS / 32; ++w) best = max(best, best_s[w]);
    cta_best = best;
  }
  cl.sync();
  if (rank == 0 && tid == 0) {
    for (int r = 1; r < LG_CLUSTER; ++r) best = max(best, *cl.map_shared_rank(&cta_best, r));
    a.argmax_dev[row] = (int)(0xffffffffu - (unsigned)best);
  }
  cl.sync();  // every CTA's cta_best stays until it is read
}

}  // namespace
}  // namespace lumina

using namespace lumina;

extern "C" int lumina_logits_adjust(const lumina_logits_args* args, void* stream) {
  LUMINA_CHECK_ARG(args, "logits_adjust: null arguments");
  const lumina_logits_args a = *args;
  LUMINA_CHECK_ARG(a.rows >= 0 && a.vocab >= 1 && a.rows < (1 << 24), "logits_adjust: %d rows x %d", a.rows, a.vocab);
  if (a.rows == 0) return LUMINA_OK;
  LUMINA_CHECK_ARG(a.logits_dev && a.out_dev, "logits_adjust: null pointer");
  LUMINA_CHECK_ARG(a.ld >= a.vocab && a.ldo >= a.vocab, "logits_adjust: ld %d / ldo %d smaller than %d", a.ld, a.ldo, a.vocab);
  LUMINA_CHECK_ARG((a.hist_start_dev == nullptr) == (a.hist_tok_dev == nullptr), "logits_adjust: history needs offsets and tokens");
  LUMINA_CHECK_ARG((a.bias_start_dev == nullptr) == (a.bias_tok_dev == nullptr) &&
                       (a.bias_start_dev == nullptr) == (a.bias_val_dev == nullptr),
                   "logits_adjust: biases need offsets, tokens and values");
  LUMINA_CHECK_ARG(!a.mask_dev || (long long)a.mask_ld * 32 >= a.vocab, "logits_adjust: mask rows of %d words for %d tokens",
                   a.mask_ld, a.vocab);
  int prev = -1;
  LUMINA_CUDA_TRY(cudaGetDevice(&prev));
  if (prev != a.device) LUMINA_CUDA_TRY(cudaSetDevice(a.device));
  int rc = set_smem_limit((const void*)logits_kernel, 2 * LG_SLICE * 4, "logits_adjust");
  if (!rc) {
    const int per = ((a.vocab + LG_CLUSTER - 1) / LG_CLUSTER + 31) / 32 * 32;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows * LG_CLUSTER);
    cfg.blockDim = dim3(LG_THREADS);
    cfg.dynamicSmemBytes = 2 * LG_SLICE * 4;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = LG_CLUSTER;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, logits_kernel, a, per);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_error("logits_adjust launch: %s", cudaGetErrorString(e));
      rc = LUMINA_E_CUDA;
    }
  }
  if (prev != a.device) cudaSetDevice(prev);
  return rc;
}
