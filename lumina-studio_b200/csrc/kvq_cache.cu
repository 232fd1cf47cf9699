// Quantized KV pages: the fused norm + RoPE + quantizing write of a step's
// new rows, and the read-back. The pool's layout and the arithmetic are
// declared in lumina_cuda.h.
#include <cfloat>
#include <cmath>

#include "kvq.cuh"

namespace lumina {

KvqDevice::KvqDevice(int dev) : ok(false), dev_(dev) {
  if (cudaGetDevice(&prev_) != cudaSuccess) {
    cudaGetLastError();
    prev_ = -1;
    return;
  }
  if (prev_ != dev && cudaSetDevice(dev) != cudaSuccess) {
    cudaGetLastError();
    return;
  }
  ok = true;
}
KvqDevice::~KvqDevice() {
  if (ok && prev_ != dev_) cudaSetDevice(prev_);
}

int kvq_view(const lumina_kvq_pool* p, const lumina_kvq_batch* b, const char* what, KvqView* v) {
  LUMINA_CHECK_ARG(p && b, "%s: null pool or batch", what);
  LUMINA_CHECK_ARG(p->pool_dev && b->row_start_dev && b->len_dev && b->pages_dev, "%s: null device pointer", what);
  LUMINA_CHECK_ARG(((uintptr_t)p->pool_dev & 15) == 0, "%s: the pool is not 16-byte aligned", what);
  LUMINA_CHECK_ARG(p->bits == 8 || p->bits == 4, "%s: %d bits per code, 8 or 4", what, p->bits);
  LUMINA_CHECK_ARG(p->n_pages >= 1 && p->n_kv >= 1 && p->n_kv <= 1024, "%s: %d pages x %d KV heads", what, p->n_pages, p->n_kv);
  LUMINA_CHECK_ARG(p->page_size == 16 || p->page_size == 32 || p->page_size == 64 || p->page_size == 128,
                   "%s: page size %d, one of 16, 32, 64, 128", what, p->page_size);
  LUMINA_CHECK_ARG(b->n_seq >= 1 && b->n_seq <= KVQ_MAX_SEQ, "%s: %d sequences, 1..%d", what, b->n_seq, KVQ_MAX_SEQ);
  LUMINA_CHECK_ARG(b->pages_ld >= 1, "%s: pages_ld %d", what, b->pages_ld);
  // positions from -n_rows to the end of the last key tile are ints
  LUMINA_CHECK_ARG((long long)b->pages_ld * p->page_size + max(0, b->n_rows) <= (1LL << 31) - 256,
                   "%s: page table of %d pages of %d tokens beside %d rows", what, b->pages_ld, p->page_size, b->n_rows);
  LUMINA_CHECK_ARG(b->n_rows >= 0 && b->max_rows >= 0 && b->max_rows <= b->n_rows &&
                       (long long)b->max_rows * b->n_seq >= b->n_rows,
                   "%s: %d rows of at most %d in %d sequences", what, b->n_rows, b->max_rows, b->n_seq);
  if (p->head_dim != 64 && p->head_dim != 128) {
    set_error("%s: head dim %d, 64 or 128", what, p->head_dim);
    return LUMINA_E_UNSUPPORTED;
  }
  v->pool = static_cast<uint8_t*>(p->pool_dev);
  v->block_bytes = (uint32_t)kvq_block_bytes(p->bits, p->head_dim, p->page_size);
  v->page_bytes = (size_t)v->block_bytes * p->n_kv;
  v->n_pages = p->n_pages;
  v->n_kv = p->n_kv;
  v->page_shift = p->page_size == 16 ? 4 : p->page_size == 32 ? 5 : p->page_size == 64 ? 6 : 7;
  v->row_start = b->row_start_dev;
  v->len = b->len_dev;
  v->pages = b->pages_dev;
  v->pages_ld = b->pages_ld;
  v->n_seq = b->n_seq;
  v->n_rows = b->n_rows;
  v->max_rows = b->max_rows;
  v->fault = serving_fault_ptr();
  if (!v->fault) {
    set_error("%s: fault word unavailable on device %d", what, p->device);
    return LUMINA_E_CUDA;
  }
  return LUMINA_OK;
}

int kvq_check_rows(const void* p, long long ld, int width, int type, const char* what, const char* name) {
  const int el = type == LUMINA_T_F32 ? 4 : 2;
  LUMINA_CHECK_ARG(p, "%s: %s is null", what, name);
  LUMINA_CHECK_ARG(ld >= width, "%s: rows of %s are %lld elements apart, %d wide", what, name, ld, width);
  LUMINA_CHECK_ARG(((uintptr_t)p & 15) == 0 && ld * el % 16 == 0, "%s: rows of %s are not 16-byte aligned", what, name);
  return LUMINA_OK;
}

namespace {

template <int N>
__device__ __forceinline__ void load_f32(const float* p, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const float4 f = __ldg(reinterpret_cast<const float4*>(p) + i);
    v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
  }
}
// N values of a row, requested now and converted when they are used
template <typename T, int N>
struct Packed {
  static constexpr int W = N * (int)sizeof(T) / 4;
  uint32_t w[W];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (W == 2) {
      const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = q.x; w[1] = q.y;
    } else {
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[N]) const {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(w[i]);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
};
template <int N>
__device__ __forceinline__ void store_row(float* p, const float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}
template <int N>
__device__ __forceinline__ void store_row(__half* p, const float (&v)[N]) {
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}

struct AppendArgs {
  KvqView v;
  const void *q, *k, *vv;
  size_t ldq, ldk, ldv, ldqo;
  int nh;
  const float *qw, *kw, *cos_t, *sin_t;
  float eps;
  int n_pos;
  int rows_per_cta;
  void* qo;
};

constexpr int APP_THREADS = 256;
constexpr int APP_ROWS = APP_THREADS / 32;  // rows per CTA at most (one warp looks up one row)
constexpr int APP_SLOTS = APP_THREADS / 8;  // heads per CTA: 8 lanes each

// One CTA: 32 of a row's nh + 2 nkv heads, 8 lanes per head, of up to 8
// consecutive batch rows. A lane holds E = HD / 16 values from each half of the
// head, so that every RoPE pair (j, j + HD / 2) sits in one lane. The sum of
// squares adds the two halves, then neighbours (a fixed tree). Bound by the
// bytes it moves: a warp per row looks the rows' pages up side by side (chains
// of dependent loads), the first row's values are requested before that and
// each next row's while this one is worked on. 5512 rows of 32 / 32 heads of
// 128, fp32, norms: 80 us, 5.0 TB/s (86 us with two rows per CTA, 99 with
// one); few rows take one row per CTA, so that every SM has work.
template <int HD, int BITS, typename T>
__global__ void __launch_bounds__(APP_THREADS, 4) kvq_append_kernel(AppendArgs a) {
  constexpr int E = HD / 16;
  __shared__ KvqRow row_s[APP_ROWS];
  const int row0 = blockIdx.x * a.rows_per_cta, tid = threadIdx.x, lane = tid & 31;
  const int slot = blockIdx.y * APP_SLOTS + (tid >> 3), j = (tid & 7) * E;
  const int nkv = a.v.n_kv, slots = a.nh + 2 * nkv;
  const int nr = min(a.rows_per_cta, a.v.n_rows - row0);
  const bool have = slot < slots;
  const int kind = slot < a.nh ? 0 : slot < a.nh + nkv ? 1 : 2;  // q, k, v
  const int head = kind == 0 ? slot : kind == 1 ? slot - a.nh : slot - a.nh - nkv;
  const size_t ld = kind == 0 ? a.ldq : kind == 1 ? a.ldk : a.ldv;
  const T* src = static_cast<const T*>(kind == 0 ? a.q : kind == 1 ? a.k : a.vv) + row0 * ld + (size_t)head * HD + j;
  Packed<T, E> next[2] = {};
  if (have) {
    next[0].load(src);
    next[1].load(src + HD / 2);
  }
  if ((tid >> 5) < nr) {
    const KvqRow r = kvq_locate(a.v, row0 + (tid >> 5), lane);
    if (lane == 0) row_s[tid >> 5] = r;
  }
  __syncthreads();
  for (int rr = 0; rr < nr; ++rr) {
    const int row = row0 + rr;
    float x[2 * E];
    next[0].get(*reinterpret_cast<float(*)[E]>(x));
    next[1].get(*reinterpret_cast<float(*)[E]>(x + E));
    if (have && rr + 1 < nr) {
      src += ld;
      next[0].load(src);
      next[1].load(src + HD / 2);
    }
    const KvqRow r = row_s[rr];
    if (r.pos < 0 || r.pos >= a.n_pos) {
      if (r.pos >= a.n_pos && tid == 0) kvq_fault(a.v, KVQ_FAULT_DATA);
      continue;
    }
    const float* nw = kind == 0 ? a.qw : kind == 1 ? a.kw : nullptr;
    // every lane of a head takes part in its shuffles (the 8 lanes agree)
    float ss = 0.f;
    {
      float p[E];
#pragma unroll
      for (int i = 0; i < E; ++i) p[i] = __fadd_rn(__fmul_rn(x[i], x[i]), __fmul_rn(x[E + i], x[E + i]));
#pragma unroll
      for (int w = 1; w < E; w *= 2)
#pragma unroll
        for (int i = 0; i + w < E; i += 2 * w) p[i] = __fadd_rn(p[i], p[i + w]);
      ss = p[0];
#pragma unroll
      for (int o = 1; o < 8; o *= 2) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, o));
    }
    if (nw) {
      const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fmul_rn(ss, 1.0f / HD), a.eps)));
      float w[2 * E];
      load_f32<E>(nw + j, *reinterpret_cast<float(*)[E]>(w));
      load_f32<E>(nw + HD / 2 + j, *reinterpret_cast<float(*)[E]>(w + E));
#pragma unroll
      for (int i = 0; i < 2 * E; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], inv), w[i]);
    }
    if (kind != 2 && have) {
      float c[E], s[E];
      load_f32<E>(a.cos_t + (size_t)r.pos * (HD / 2) + j, c);
      load_f32<E>(a.sin_t + (size_t)r.pos * (HD / 2) + j, s);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float u = x[i], w = x[E + i];
        x[i] = __fsub_rn(__fmul_rn(u, c[i]), __fmul_rn(w, s[i]));
        x[E + i] = __fadd_rn(__fmul_rn(u, s[i]), __fmul_rn(w, c[i]));
      }
    }
    // largest magnitude of the head as its bits: they order like the values,
    // and an infinity or a NaN orders above every finite one
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 2 * E; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < 8; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!have) continue;
    if (kind == 0) {
      T* dst = static_cast<T*>(a.qo) + (size_t)row * a.ldqo + (size_t)head * HD + j;
      store_row<E>(dst, *reinterpret_cast<const float(*)[E]>(x));
      store_row<E>(dst + HD / 2, *reinterpret_cast<const float(*)[E]>(x + E));
      continue;
    }
    const float amax = __uint_as_float(top);
    const bool bad = top >= 0x7f800000u, zero = amax < 7.888609052210118e-31f;  // 2^-100
    const float rcp = bad || zero ? 0.f : __fmul_rn(__fdiv_rn(1.0f, amax), BITS == 8 ? 127.0f : 7.5f);
    const float scale = bad ? __uint_as_float(0x7fffffffu) : zero ? 0.f : __fmul_rn(amax, BITS == 8 ? 1.0f / 127.0f : 1.0f / 15.0f);
    const int P = 1 << a.v.page_shift;
    constexpr int NB = HD * BITS / 8;
    uint8_t* blk = const_cast<uint8_t*>(r.page) + (size_t)head * a.v.block_bytes;
    uint8_t* code = blk + ((kind == 2 ? P : 0) + r.off) * NB;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float y = bad ? 0.f : x[h * E + i];
        if constexpr (BITS == 8) {
          const int c = __float2int_rn(__fmul_rn(y, rcp));
          w[i >> 2] |= (uint32_t)(min(127, max(-127, c)) & 0xFF) << (8 * (i & 3));
        } else {
          const int c = __float2int_rn(__fadd_rn(__fmul_rn(y, rcp), 7.5f));
          w[0] |= (uint32_t)min(15, max(0, c)) << (4 * i);
        }
      }
      const int at = (h * (HD / 2) + j) * BITS / 8;
      if constexpr (E * BITS == 64) *reinterpret_cast<uint2*>(code + at) = make_uint2(w[0], w[1]);
      else if constexpr (E * BITS == 32) *reinterpret_cast<uint32_t*>(code + at) = w[0];
      else *reinterpret_cast<uint16_t*>(code + at) = (uint16_t)w[0];
    }
    if ((tid & 7) == 0)
      reinterpret_cast<float*>(blk + 2 * P * NB)[(kind == 2 ? P : 0) + r.off] = scale;
  }
}

struct ReadArgs {
  KvqView v;
  void *k, *vv;
  size_t ld;
  int rows_per_cta;
};

constexpr int RD_THREADS = 256;
constexpr int RD_ROWS = 16;  // rows per CTA at most

// One CTA: up to 16 batch rows (a warp looks up two of them) and 256 groups
// of 16 output bytes of each (a warp's stores are whole lines); a thread turns
// its group of 8 rows at a time into values, their codes and scales requested
// together. 5512 rows x 32 heads of 128, int8 to fp32, bound by the bytes
// written: 45 us, 5.0 TB/s (68 us with 8 values per thread, whose fp32 stores
// were half lines). 8 sequences of up to 8192, int4 to fp16: 33 us where the
// bytes take 20, with neither DRAM (27 %) nor issue (2.4 of 4) full: a CTA looks
// its rows up, waits, and then streams once.
template <int HD, int BITS, typename T>
__global__ void __launch_bounds__(RD_THREADS) kvq_read_kernel(ReadArgs a) {
  constexpr int NB = HD * BITS / 8, N = 16 / (int)sizeof(T), GROUPS = HD / N, U = 8;
  constexpr int BYTES = N * BITS / 8;  // of a group's codes: 8, 4 or 2
  __shared__ const uint8_t* page_s[RD_ROWS];
  __shared__ int off_s[RD_ROWS];
  const int tid = threadIdx.x, lane = tid & 31;
  const int row0 = blockIdx.x * a.rows_per_cta;
  const int nr = min(a.rows_per_cta, a.v.n_rows - row0);
  for (int i = tid >> 5; i < nr; i += RD_THREADS / 32) {
    const KvqRow r = kvq_locate(a.v, row0 + i, lane);
    if (lane == 0) {
      page_s[i] = r.pos < 0 ? nullptr : r.page;
      off_s[i] = r.off;
    }
  }
  __syncthreads();
  const int P = 1 << a.v.page_shift, half = a.v.n_kv * GROUPS, c = blockIdx.y * RD_THREADS + tid;
  if (c >= 2 * half) return;
  const int isv = c >= half, hc = c - (isv ? half : 0), h = hc / GROUPS, e = (hc % GROUPS) * N;
  const size_t blk = (size_t)h * a.v.block_bytes;
  T* dst = static_cast<T*>(isv ? a.vv : a.k) + (size_t)row0 * a.ld + (size_t)h * HD + e;
  for (int r0 = 0; r0 < nr; r0 += U) {
    uint32_t w[U][2];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int rr = r0 + u;
      const uint8_t* page = rr < nr ? page_s[rr] : nullptr;
      if (!page) continue;
      const int t = (isv ? P : 0) + off_s[rr];
      s[u] = __ldg(reinterpret_cast<const float*>(page + blk + 2 * P * NB) + t);
      const uint8_t* code = page + blk + (size_t)t * NB + e * BITS / 8;
      if constexpr (BYTES == 8) {
        const uint2 q = __ldg(reinterpret_cast<const uint2*>(code));
        w[u][0] = q.x;
        w[u][1] = q.y;
      } else if constexpr (BYTES == 4) {
        w[u][0] = __ldg(reinterpret_cast<const uint32_t*>(code));
      } else {
        w[u][0] = __ldg(reinterpret_cast<const uint16_t*>(code));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int rr = r0 + u;
      if (rr >= nr || !page_s[rr]) continue;
      float x[N];
#pragma unroll
      for (int q = 0; q < N; ++q) {
        if constexpr (BITS == 8) x[q] = __fmul_rn((float)(int8_t)(w[u][q / 4] >> (8 * (q & 3))), s[u]);
        else x[q] = __fmul_rn((float)(2 * (int)((w[u][0] >> (4 * q)) & 15u) - 15), s[u]);
      }
      store_row<N>(dst + (size_t)rr * a.ld, x);
    }
  }
}

// Rows per CTA: as many as leave every SM several CTAs
int rows_per_cta(int rows, int parts, int most) {
  int n = most;
  while (n > 1 && ((long long)rows + n - 1) / n * parts < 4LL * sm_count()) n /= 2;
  return n;
}

#define KVQ_DISPATCH(HD_, BITS_, TYPE_, KERNEL, ...)                                        \
  do {                                                                                      \
    if (HD_ == 128 && BITS_ == 8 && TYPE_ == LUMINA_T_F16) KERNEL<128, 8, __half> __VA_ARGS__; \
    else if (HD_ == 128 && BITS_ == 8) KERNEL<128, 8, float> __VA_ARGS__;                   \
    else if (HD_ == 128 && TYPE_ == LUMINA_T_F16) KERNEL<128, 4, __half> __VA_ARGS__;       \
    else if (HD_ == 128) KERNEL<128, 4, float> __VA_ARGS__;                                 \
    else if (BITS_ == 8 && TYPE_ == LUMINA_T_F16) KERNEL<64, 8, __half> __VA_ARGS__;        \
    else if (BITS_ == 8) KERNEL<64, 8, float> __VA_ARGS__;                                  \
    else if (TYPE_ == LUMINA_T_F16) KERNEL<64, 4, __half> __VA_ARGS__;                      \
    else KERNEL<64, 4, float> __VA_ARGS__;                                                  \
  } while (0)

}  // namespace
}  // namespace lumina

using namespace lumina;

extern "C" {

int lumina_kvq_block_bytes(int bits, int head_dim, int page_size, size_t* bytes) {
  LUMINA_CHECK_ARG(bytes, "kvq_block_bytes: null output");
  LUMINA_CHECK_ARG((bits == 8 || bits == 4) && head_dim >= 1 && head_dim % 8 == 0 && page_size >= 1,
                   "kvq_block_bytes: %d bits, head dim %d, page size %d", bits, head_dim, page_size);
  *bytes = kvq_block_bytes(bits, head_dim, page_size);
  return LUMINA_OK;
}

int lumina_kvq_append(const lumina_kvq_pool* pool, const lumina_kvq_batch* batch, const void* q, int ldq, const void* k,
                      int ldk, const void* v, int ldv, int type, int n_heads, const float* q_norm, const float* k_norm,
                      float eps, const float* cos_t, const float* sin_t, int n_pos, void* q_out, int ldqo, void* stream) {
  LUMINA_CHECK_ARG(pool && batch, "kvq_append: null pool or batch");
  KvqDevice g(pool->device);
  LUMINA_CHECK_ARG(g.ok, "kvq_append: device %d not available", pool->device);
  AppendArgs a{};
  int rc = kvq_view(pool, batch, "kvq_append", &a.v);
  if (rc) return rc;
  LUMINA_CHECK_ARG(type == LUMINA_T_F32 || type == LUMINA_T_F16, "kvq_append: type %d", type);
  LUMINA_CHECK_ARG(n_heads >= 1 && n_heads <= 65536, "kvq_append: %d query heads", n_heads);
  if (batch->n_rows == 0) return LUMINA_OK;
  const int hd = pool->head_dim;
  if ((rc = kvq_check_rows(q, ldq, n_heads * hd, type, "kvq_append", "q"))) return rc;
  if ((rc = kvq_check_rows(k, ldk, pool->n_kv * hd, type, "kvq_append", "k"))) return rc;
  if ((rc = kvq_check_rows(v, ldv, pool->n_kv * hd, type, "kvq_append", "v"))) return rc;
  if ((rc = kvq_check_rows(q_out, ldqo, n_heads * hd, type, "kvq_append", "q_out"))) return rc;
  LUMINA_CHECK_ARG(cos_t && sin_t && n_pos >= 1, "kvq_append: cos / sin tables missing");
  LUMINA_CHECK_ARG((((uintptr_t)cos_t | (uintptr_t)sin_t | (uintptr_t)q_norm | (uintptr_t)k_norm) & 15) == 0,
                   "kvq_append: tables and norm weights are not 16-byte aligned");
  LUMINA_CHECK_ARG(std::isfinite(eps) && eps >= 0, "kvq_append: eps %g", eps);
  a.q = q; a.k = k; a.vv = v;
  a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldqo = ldqo;
  a.nh = n_heads;
  a.qw = q_norm; a.kw = k_norm; a.cos_t = cos_t; a.sin_t = sin_t;
  a.eps = eps;
  a.n_pos = n_pos;
  a.qo = q_out;
  const int parts = (n_heads + 2 * pool->n_kv + APP_SLOTS - 1) / APP_SLOTS;
  a.rows_per_cta = rows_per_cta(batch->n_rows, parts, APP_ROWS);
  const dim3 grid((batch->n_rows + a.rows_per_cta - 1) / a.rows_per_cta, parts);
  cudaStream_t s = (cudaStream_t)stream;
  KVQ_DISPATCH(hd, pool->bits, type, kvq_append_kernel, <<<grid, APP_THREADS, 0, s>>>(a));
  LUMINA_LAUNCH_CHECK();
  return LUMINA_OK;
}

int lumina_kvq_read(const lumina_kvq_pool* pool, const lumina_kvq_batch* batch, void* k_out, void* v_out, int ldo,
                    int type, void* stream) {
  LUMINA_CHECK_ARG(pool && batch, "kvq_read: null pool or batch");
  KvqDevice g(pool->device);
  LUMINA_CHECK_ARG(g.ok, "kvq_read: device %d not available", pool->device);
  ReadArgs a{};
  int rc = kvq_view(pool, batch, "kvq_read", &a.v);
  if (rc) return rc;
  LUMINA_CHECK_ARG(type == LUMINA_T_F32 || type == LUMINA_T_F16, "kvq_read: type %d", type);
  if (batch->n_rows == 0) return LUMINA_OK;
  const int hd = pool->head_dim;
  if ((rc = kvq_check_rows(k_out, ldo, pool->n_kv * hd, type, "kvq_read", "k_out"))) return rc;
  if ((rc = kvq_check_rows(v_out, ldo, pool->n_kv * hd, type, "kvq_read", "v_out"))) return rc;
  a.k = k_out; a.vv = v_out;
  a.ld = ldo;
  const int parts = (2 * pool->n_kv * hd * (type == LUMINA_T_F16 ? 2 : 4) / 16 + RD_THREADS - 1) / RD_THREADS;
  a.rows_per_cta = rows_per_cta(batch->n_rows, parts, RD_ROWS);
  const dim3 grid((batch->n_rows + a.rows_per_cta - 1) / a.rows_per_cta, parts);
  cudaStream_t s = (cudaStream_t)stream;
  KVQ_DISPATCH(hd, pool->bits, type, kvq_read_kernel, <<<grid, RD_THREADS, 0, s>>>(a));
  LUMINA_LAUNCH_CHECK();
  return LUMINA_OK;
}

}  // extern "C"
