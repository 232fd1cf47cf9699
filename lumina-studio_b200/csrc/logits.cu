// Penalties, token biases and a grammar mask on logits rows, and the argmax
// (the rules are declared in lumina_cuda.h).
//
// A row is one CTA's or a cluster's (the argmax joins over distributed shared
// memory, so there is no second launch and no workspace). A CTA streams its
// part of the vocabulary once (read, mask, write), bound by those bytes, with
// the next slice and its mask words in flight. The tokens that the row's
// history or biases name are few: a bit each keeps them out of the stream's
// maximum, and afterwards each is counted in the slot that its rank among
// them gives (integer atomics: the order does not matter) and adjusted.
//
// 256 rows x 131072, 3000 history tokens, 24 biases and a mask: 82 us, 3.2
// TB/s of the logits read and written, where the bytes take 42; 61 us without
// history and biases (256 rows on 148 SMs, two rows on most, account for 48).
// Naming and counting the history takes the other 20, with nothing of the
// CTA's own stream beside it. The same
// with every slice's tokens counted before it is streamed: 134 us; in a hash
// table instead of by rank: 121 us. 1 row x 32000: 9 us, launch and
// dependent loads.
#include <cooperative_groups.h>

#include "weights.cuh"

namespace lumina {

namespace {

namespace cg = cooperative_groups;

constexpr int LG_THREADS = 512;
constexpr int LG_PER = 2;                          // groups of 4 logits a thread holds
constexpr int LG_SLICE = 4 * LG_PER * LG_THREADS;  // tokens a CTA requests at once
constexpr int LG_WORDS = 8;                        // words of named bits per thread
constexpr int LG_CHUNK = 32 * LG_WORDS * LG_THREADS;  // tokens that the named bits cover
constexpr int LG_SLOTS = 4096;                     // named tokens counted at once
constexpr int LG_SMEM = (2 * LG_SLOTS + 2 * LG_CHUNK / 32) * 4;

// orders like the value; a NaN is the largest, -0 equals 0
__device__ __forceinline__ unsigned lg_order(float v) {
  const unsigned u = __float_as_uint(v);
  if ((u << 1) > 0xff000000u) return 0xffffffffu;
  return (u << 1) == 0u ? 0x80000000u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// VEC: logits and output rows are 16-byte aligned
template <bool VEC>
__global__ void __launch_bounds__(LG_THREADS, 2) logits_kernel(lumina_logits_args a, int per_cta, int cluster) {
  extern __shared__ __align__(16) int sm[];
  int *count = sm, *bias = sm + LG_SLOTS;  // bias: 1 + index of the token's last entry
  unsigned* named = reinterpret_cast<unsigned*>(sm + 2 * LG_SLOTS);
  int* first = sm + 2 * LG_SLOTS + LG_CHUNK / 32;  // named tokens below a word's
  static_assert(LG_SLOTS <= LG_CHUNK / 32, "the slots' tokens lie where the words' ranks did");
  __shared__ unsigned long long best_s[LG_THREADS / 32], cta_best;
  __shared__ int sum_s[LG_THREADS / 32];
  cg::cluster_group cl = cg::this_cluster();
  const int row = blockIdx.x / cluster, rank = blockIdx.x - row * cluster;
  const int tid = threadIdx.x;
  const float* src = a.logits_dev + (size_t)row * a.ld;
  float* dst = a.out_dev + (size_t)row * a.ldo;
  const uint32_t* mask = a.mask_dev ? a.mask_dev + (size_t)row * a.mask_ld : nullptr;
  const int v0 = rank * per_cta, v1 = min(a.vocab, v0 + per_cta);

  // logits and mask bits of this thread's groups of the slice at s0, below end
  auto load = [&](int s0, int end, float4 (&l4)[LG_PER], uint32_t (&bits)[LG_PER]) {
    const int n = end - s0;  // 0 or less: nothing left
#pragma unroll
    for (int k = 0; k < LG_PER; ++k) {
      const int i = (k * LG_THREADS + tid) * 4;
      bits[k] = ~0u;
      if (i < n) {
        if (VEC && i + 3 < n) {
          l4[k] = __ldcs(reinterpret_cast<const float4*>(src + s0 + i));
        } else {
          l4[k] = make_float4(src[s0 + i], i + 1 < n ? src[s0 + i + 1] : 0.f, i + 2 < n ? src[s0 + i + 2] : 0.f,
                              i + 3 < n ? src[s0 + i + 3] : 0.f);
        }
        if (mask) bits[k] = __ldg(mask + ((s0 + i) >> 5));  // shifted at its use: no wait here
      }
    }
  };

  const bool hist = a.hist_start_dev != nullptr, biased = a.bias_start_dev != nullptr;
  auto within = [](int i, int n) { return max(0, min(i, n)); };
  const int h0 = hist ? within(a.hist_start_dev[row], a.hist_len) : 0, h1 = hist ? within(a.hist_start_dev[row + 1], a.hist_len) : 0;
  const int b0 = biased ? within(a.bias_start_dev[row], a.bias_len) : 0, b1 = biased ? within(a.bias_start_dev[row + 1], a.bias_len) : 0;
  const bool any = h1 > h0 || b1 > b0;  // else no token is named
  unsigned top = 0;  // the stream's largest value (lg_order) and its first token
  int at = 0x7fffffff;
  unsigned long long best = 0;  // the named tokens'
  for (int c0 = v0; c0 < v1; c0 += LG_CHUNK) {
    const int c1 = min(v1, c0 + LG_CHUNK);
    float4 next4[LG_PER];
    uint32_t next_bits[LG_PER];
    load(c0, c1, next4, next_bits);
    if (any) {
      for (int i = tid; i < LG_CHUNK / 32; i += LG_THREADS) named[i] = 0u;
      __syncthreads();
      auto name = [&](int token) {
        const unsigned t = (unsigned)(token - c0);
        if (t < (unsigned)(c1 - c0)) atomicOr(&named[t >> 5], 1u << (t & 31));
      };
#pragma unroll 4
      for (int i = h0 + tid; i < h1; i += LG_THREADS) name(__ldg(a.hist_tok_dev + i));
      for (int i = b0 + tid; i < b1; i += LG_THREADS) name(__ldg(a.bias_tok_dev + i));
      __syncthreads();
    }
    for (int s0 = c0; s0 < c1; s0 += LG_SLICE) {
      const int n = min(LG_SLICE, c1 - s0);
      float4 l4[LG_PER];
      uint32_t bits[LG_PER];
#pragma unroll
      for (int k = 0; k < LG_PER; ++k) {
        l4[k] = next4[k];
        bits[k] = next_bits[k] >> ((k * LG_THREADS + tid) * 4 & 31);  // c0 and s0 are multiples of 32
      }
      load(s0 + LG_SLICE, c1, next4, next_bits);
#pragma unroll
      for (int k = 0; k < LG_PER; ++k) {
        const int i = (k * LG_THREADS + tid) * 4;
        if (i >= n) continue;
        float l[4] = {l4[k].x, l4[k].y, l4[k].z, l4[k].w};
        const unsigned skip = any ? named[(s0 - c0 + i) >> 5] >> (i & 31) : 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!((bits[k] >> e) & 1u)) l[e] = -INFINITY;
          const unsigned o = lg_order(l[e]);
          if (i + e < n && !((skip >> e) & 1u) && (o > top || at == 0x7fffffff)) {  // ascending: the first of the largest stays
            top = o;
            at = s0 + i + e;
          }
        }
        if (VEC && i + 3 < n) {
          *reinterpret_cast<float4*>(dst + s0 + i) = make_float4(l[0], l[1], l[2], l[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i + e < n) dst[s0 + i + e] = l[e];
        }
      }
    }
    if (!any) continue;
    // ---- the named tokens: a token's slot is the number of named ones below it
    int mine = 0, base = 0, total;
#pragma unroll
    for (int w = 0; w < LG_WORDS; ++w) mine += __popc(named[tid * LG_WORDS + w]);
    total = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int u = __shfl_up_sync(0xffffffffu, total, o);
      if ((tid & 31) >= o) total += u;
    }
    if ((tid & 31) == 31) sum_s[tid >> 5] = total;
    base = total - mine;
    __syncthreads();  // also: the stream's writes are seen by the whole CTA
    total = 0;
    for (int w = 0; w < LG_THREADS / 32; ++w) {
      if (w == tid >> 5) base += total;
      total += sum_s[w];
    }
    const float rep = a.repeat_dev ? a.repeat_dev[row] : 1.f;
    const float fr = a.frequency_dev ? a.frequency_dev[row] : 0.f, pr = a.presence_dev ? a.presence_dev[row] : 0.f;
    for (int r0 = 0; r0 < total; r0 += LG_SLOTS) {
      const int nr = min(LG_SLOTS, total - r0);
      for (int i = tid; i < nr; i += LG_THREADS) count[i] = bias[i] = 0;
      for (int w = 0, f = base; w < LG_WORDS; ++w) {
        first[tid * LG_WORDS + w] = f;
        f += __popc(named[tid * LG_WORDS + w]);
      }
      __syncthreads();
      auto slot = [&](int token) {  // LG_SLOTS or more: not in this pass
        const unsigned t = (unsigned)(token - c0);
        if (t >= (unsigned)(c1 - c0)) return (unsigned)LG_SLOTS;
        return (unsigned)(first[t >> 5] + __popc(named[t >> 5] & ((1u << (t & 31)) - 1u)) - r0);
      };
#pragma unroll 4
      for (int i = h0 + tid; i < h1; i += LG_THREADS) {
        const unsigned s = slot(__ldg(a.hist_tok_dev + i));
        if (s < LG_SLOTS) atomicAdd(&count[s], 1);
      }
      for (int i = b0 + tid; i < b1; i += LG_THREADS) {
        const unsigned s = slot(__ldg(a.bias_tok_dev + i));
        if (s < LG_SLOTS) atomicMax(&bias[s], i - b0 + 1);
      }
      __syncthreads();
      int* token = first;  // of each slot: the words' ranks are not needed any more
      if (base < r0 + nr && base + mine > r0)
        for (int w = tid * LG_WORDS, s = base - r0; w < (tid + 1) * LG_WORDS; ++w)
          for (unsigned m = named[w]; m; m &= m - 1, ++s)
            if ((unsigned)s < (unsigned)nr) token[s] = c0 + w * 32 + __ffs(m) - 1;
      __syncthreads();
#pragma unroll 4
      for (int i = tid; i < nr; i += LG_THREADS) {
        const int t = token[i];
        float l = dst[t];  // the logit, or -inf where the mask forbids the token
        if (!mask || ((__ldg(mask + (t >> 5)) >> (t & 31)) & 1u)) {
          if (count[i]) {
            l = l > 0.f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
            l = __fsub_rn(__fsub_rn(l, __fmul_rn(fr, (float)count[i])), pr);
          }
          if (bias[i]) l = __fadd_rn(l, __ldg(a.bias_val_dev + b0 + bias[i] - 1));
          dst[t] = l;
        }
        best = max(best, ((unsigned long long)lg_order(l) << 32) | (0xffffffffu - (unsigned)t));
      }
      __syncthreads();
    }
  }
  if (!a.argmax_dev) return;
  if (at != 0x7fffffff) best = max(best, ((unsigned long long)top << 32) | (0xffffffffu - (unsigned)at));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & 31) == 0) best_s[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < LG_THREADS / 32; ++w) best = max(best, best_s[w]);
    cta_best = best;
  }
  if (cluster > 1) cl.sync();
  if (rank == 0 && tid == 0) {
    for (int r = 1; r < cluster; ++r) best = max(best, *cl.map_shared_rank(&cta_best, r));
    a.argmax_dev[row] = (int)(0xffffffffu - (unsigned)best);
  }
  if (cluster > 1) cl.sync();  // every CTA's cta_best stays until it is read
}

}  // namespace
}  // namespace lumina

using namespace lumina;

extern "C" int lumina_logits_adjust(const lumina_logits_args* args, void* stream) {
  LUMINA_CHECK_ARG(args, "logits_adjust: null arguments");
  const lumina_logits_args a = *args;
  // tokens plus a chunk of them stay within an int
  LUMINA_CHECK_ARG(a.rows >= 0 && a.vocab >= 1 && a.rows < (1 << 24) && a.vocab <= (1 << 30), "logits_adjust: %d rows x %d",
                   a.rows, a.vocab);
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
  const bool vec = (((uintptr_t)a.logits_dev | (uintptr_t)a.out_dev) & 15) == 0 && a.ld % 4 == 0 && a.ldo % 4 == 0;
  auto kern = vec ? logits_kernel<true> : logits_kernel<false>;
  int rc = set_smem_limit((const void*)kern, LG_SMEM, "logits_adjust");
  if (!rc) {
    // CTAs of a row: enough that few rows fill the GPU, few enough that many
    // rows spend their time streaming, as each CTA reads the whole history
    // (256 rows x 131072: 82 us with 1, 98 with 2, 189 with 8)
    int cluster = 1;
    while (cluster < 8 && (long long)a.rows * cluster < 3LL * sm_count() / 2 && a.vocab > 2 * cluster * 1024) cluster *= 2;
    const int per = ((a.vocab + cluster - 1) / cluster + 31) / 32 * 32;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows * cluster);
    cfg.blockDim = dim3(LG_THREADS);
    cfg.dynamicSmemBytes = LG_SMEM;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, per, cluster);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_error("logits_adjust launch: %s", cudaGetErrorString(e));
      rc = LUMINA_E_CUDA;
    }
  }
  if (prev != a.device) cudaSetDevice(prev);
  return rc;
}
