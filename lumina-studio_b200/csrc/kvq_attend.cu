// Attention of a batch's rows over quantized KV pages: the general kernel
// on mma.sync, 16 packed query rows per CTA, and the entry point.
//
// out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m), x in units of log2: one
// pass over the keys with a running maximum and sum per row in fp32. The
// four warps of a CTA take 16 keys each of every 64; each keeps its own
// state, and they merge in shared memory in warp order at the end.
// p times the V scale enters the tensor pipe as fp16 relative to the
// largest V scale seen (a running power of two 2^e, times 2^14 to use
// fp16's range); fp32 rows send q and p as two fp16 parts, v = hi + lo with
// hi = fp16(v), lo = fp16(v - hi), so both keep about 22 bits.
#include <cfloat>
#include <cmath>

#include "kvq_attend.cuh"
#include "kvq_mma.cuh"

namespace lumina {

namespace {

constexpr int AT_THREADS = 128;

template <int HD, int BITS, typename T>
__global__ void __launch_bounds__(AT_THREADS) kvq_attend_kernel(AttendArgs a) {
  using F = KvqFrag<HD, BITS>;
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int KK = F::KK, NT = F::NT;
  __shared__ int scan_s[4];
  __shared__ int seq_s, rb_s;
  __shared__ float O_s[4][16][HD + 4];
  __shared__ float m_s[4][16], l_s[4][16];
  __shared__ int e_s[4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const KvqView& v = a.v;

  // this CTA's (sequence, row block): blocks in sequence order
  if (tid == 0) seq_s = -1;
  __syncthreads();
  int base = 0;
  for (int s0 = 0; s0 < v.n_seq; s0 += AT_THREADS) {
    const int s = s0 + tid;
    int first, nb = 0;
    if (s < v.n_seq) {
      const int n = kvq_seq_rows(v, s, first);
      if (n * a.G > a.few) nb = (n * a.G + 15) >> 4;
    }
    int inc = nb;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (lane == 31) scan_s[warp] = inc;
    __syncthreads();
    int before = base;
    for (int w = 0; w < warp; ++w) before += scan_s[w];
    const int lo = before + inc - nb;
    if ((int)blockIdx.x >= lo && (int)blockIdx.x < lo + nb) {
      seq_s = s;
      rb_s = blockIdx.x - lo;
    }
    base += scan_s[0] + scan_s[1] + scan_s[2] + scan_s[3];
    __syncthreads();
    if (seq_s >= 0) break;
  }
  const int s = seq_s;
  if (s < 0) return;
  const int kvh = blockIdx.y;
  int first;
  const int n = kvq_seq_rows(v, s, first);
  const int cap_tokens = v.pages_ld << v.page_shift;
  int len = __ldg(v.len + s);
  if (len < 0 || len > cap_tokens) {
    if (tid == 0) kvq_fault(v, KVQ_FAULT_DATA);
    len = len < 0 ? 0 : cap_tokens;
  }
  const int pre = a.prefix ? min(len, max(0, __ldg(a.prefix + s))) : 0;

  // packed rows g and g + 8 of the block
  int pos[2], orow[2], head[2];
  bool ok[2];
  float slope[2], qmul[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = rb_s * 16 + g + 8 * h;
    ok[h] = r < n * a.G;
    const int i = ok[h] ? r / a.G : 0;
    pos[h] = len - n + i;
    orow[h] = first + i;
    head[h] = kvh * a.G + (ok[h] ? r - i * a.G : 0);
    slope[h] = a.slopes && ok[h] ? __ldg(a.slopes + head[h]) * KVQ_LOG2E : 0.f;
    qmul[h] = a.scale;
  }
  uint32_t qh[KK][4], ql[F32 ? KK : 1][4];
  {
    float q[2][KK][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const T* src = static_cast<const T*>(a.q) + (size_t)orow[h] * a.ldq + (size_t)head[h] * HD;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e) q[h][kk][e] = ok[h] ? (float)src[F::dim_of(t, kk, e)] : 0.f;
      if constexpr (F32) {
        // bring the row's largest value near 2^14: fp16's range holds hi and lo
        float m = 0.f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
          for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(q[h][kk][e]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const int ex = min(112, max(-112, (int)(__float_as_uint(m) >> 23) - 127));
        const float up = exp2i(13 - ex);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
          for (int e = 0; e < 4; ++e) q[h][kk][e] *= up;
        qmul[h] *= exp2i(ex - 13);
      }
    }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = q[i & 1][kk][(i >> 1) * 2], y = q[i & 1][kk][(i >> 1) * 2 + 1];
        if constexpr (F32) qh[kk][i] = split_h2(x, y, ql[kk][i]);
        else qh[kk][i] = half2_bits(__floats2half2_rn(x, y));
      }
  }

  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[i][c] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  int ev = -100;  // exponent the p * scale products are relative to

  // tiles of 64 keys: those the prefix shows, then those the window shows
  const int row_lo = rb_s * 16 / a.G, row_hi = min(n, (rb_s * 16 + 15) / a.G + 1);
  const int p_lo = len - n + row_lo, p_hi = len - n + row_hi - 1;
  const int key_lo = a.window ? max(0, p_lo - a.window + 1) : 0;
  const int key_hi = max(0, min(len, p_hi + 1));
  const int tp = (pre + 63) >> 6;
  const int tl = max(tp, min(key_lo, key_hi) >> 6), te = max(tl, (key_hi + 63) >> 6);
  const int nt = tp + te - tl;
  const int P = 1 << v.page_shift;
  for (int ti = 0; ti < nt; ++ti) {
    const int j0 = (ti < tp ? ti : ti - tp + tl) * 64 + warp * 16;
    if (j0 >= len) continue;
    const int pg = __ldg(v.pages + (size_t)s * v.pages_ld + (j0 >> v.page_shift));
    if ((unsigned)pg >= (unsigned)v.n_pages) {
      if (lane == 0) kvq_fault(v, KVQ_FAULT_DATA);
      continue;
    }
    const uint8_t* blk = v.pool + (size_t)pg * v.page_bytes + (size_t)kvh * v.block_bytes;
    const int off = j0 & (P - 1);
    uint32_t kw[2][F::KW], vw[4][F::VW];
#pragma unroll
    for (int x = 0; x < 2; ++x) F::load_k(blk + (size_t)(off + x * 8 + g) * F::NB + F::k_lane(t), kw[x]);
#pragma unroll
    for (int x = 0; x < 4; ++x)
      F::load_v(blk + (size_t)(P + off + 2 * t + (x & 1) + 8 * (x >> 1)) * F::NB + F::v_lane(g), vw[x]);
    const float* sc = reinterpret_cast<const float*>(blk + 2 * P * F::NB) + off;
    float sk[4], sv[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int key = 2 * t + (x & 1) + 8 * (x >> 1);
      const bool in = j0 + key < len && (j0 + key >= key_lo || j0 + key < pre);
      sk[x] = in ? sc[key] : 0.f;
      sv[x] = in ? sc[P + key] : 0.f;
    }
    float x2[2][4];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      auto step = [&](auto kc) {
        constexpr int kk = decltype(kc)::value;
        uint32_t b0, b1;
        F::template k_frag<kk>(kw[x], b0, b1);
        if constexpr (F32) mma_16816(acc, ql[kk], b0, b1);
        mma_16816(acc, qh[kk], b0, b1);
      };
      step(std::integral_constant<int, 0>());
      step(std::integral_constant<int, 1>());
      step(std::integral_constant<int, 2>());
      step(std::integral_constant<int, 3>());
      if constexpr (KK == 8) {
        step(std::integral_constant<int, 4>());
        step(std::integral_constant<int, 5>());
        step(std::integral_constant<int, 6>());
        step(std::integral_constant<int, 7>());
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int h = c >> 1, j = j0 + x * 8 + 2 * t + (c & 1);
        float z = acc[c] * (sk[2 * x + (c & 1)] * qmul[h]);
        if (a.cap > 0.f) z = a.cap * tanhf(z / a.cap);
        z *= KVQ_LOG2E;
        z = fmaf(-slope[h], fabsf((float)(pos[h] - j)), z);
        const bool see = ok[h] && j < len && ((j <= pos[h] && (a.window == 0 || j > pos[h] - a.window)) || j < pre);
        x2[x][c] = see ? z : -INFINITY;
      }
    }
    // running maximum, one power of two for the V scales
    float svm = fmaxf(fmaxf(fabsf(sv[0]), fabsf(sv[1])), fmaxf(fabsf(sv[2]), fabsf(sv[3])));
    svm = fmaxf(svm, __shfl_xor_sync(0xffffffffu, svm, 1));
    svm = fmaxf(svm, __shfl_xor_sync(0xffffffffu, svm, 2));
    const int en = max(ev, min(100, max(-100, (int)(__float_as_uint(svm) >> 23) - 126)));
    const float es = exp2i(max(-126, ev - en)), ps = exp2i(14 - en);
    ev = en;
    float fac[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = fmaxf(fmaxf(x2[0][2 * h], x2[0][2 * h + 1]), fmaxf(x2[1][2 * h], x2[1][2 * h + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[h], mx), ms = mn == -INFINITY ? 0.f : mn;
      fac[h] = ex2(m[h] - ms);
      m[h] = mn;
      float sum = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float p = ex2(x2[x][2 * h + c] - ms);
          sum += p;
          // a masked key counts for nothing, whatever its scale holds
          x2[x][2 * h + c] = p == 0.f ? 0.f : p * (sv[2 * x + c] * ps);
        }
      l[h] = l[h] * fac[h] + sum;
    }
    uint32_t pa[4], pl[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = i & 1, x = i >> 1;
      if constexpr (F32) pa[i] = split_h2(x2[x][2 * h], x2[x][2 * h + 1], pl[i]);
      else pa[i] = half2_bits(__floats2half2_rn(x2[x][2 * h], x2[x][2 * h + 1]));
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][c] *= fac[c >> 1] * es;
    constexpr int DPW = 32 / BITS;
    auto dim = [&](auto ic, int w) {
      constexpr int i = decltype(ic)::value;
      const uint32_t b0 = F::template v_pair<i>(vw[0][w], vw[1][w]), b1 = F::template v_pair<i>(vw[2][w], vw[3][w]);
      if constexpr (F32) mma_16816(o[w * DPW + i], pl, b0, b1);
      mma_16816(o[w * DPW + i], pa, b0, b1);
    };
#pragma unroll
    for (int w = 0; w < F::VW; ++w) {
      dim(std::integral_constant<int, 0>(), w);
      dim(std::integral_constant<int, 1>(), w);
      dim(std::integral_constant<int, 2>(), w);
      dim(std::integral_constant<int, 3>(), w);
      if constexpr (DPW == 8) {
        dim(std::integral_constant<int, 4>(), w);
        dim(std::integral_constant<int, 5>(), w);
        dim(std::integral_constant<int, 6>(), w);
        dim(std::integral_constant<int, 7>(), w);
      }
    }
  }

  // merge the four warps
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (t == 0) {
      m_s[warp][g + 8 * h] = m[h];
      l_s[warp][g + 8 * h] = l[h];
    }
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + 8 * h;
    const float M = fmaxf(fmaxf(m_s[0][r], m_s[1][r]), fmaxf(m_s[2][r], m_s[3][r]));
    const float f = ex2(m[h] - (M == -INFINITY ? 0.f : M)) * exp2i(ev - 14);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < NT; ++i) O_s[warp][r][(2 * t + c) * NT + i] = o[i][2 * h + c] * f;
  }
  __syncthreads();
  for (int i = tid; i < 16 * HD; i += AT_THREADS) {
    const int r = i / HD, d = i % HD, pr = rb_s * 16 + r;
    if (pr >= n * a.G) continue;
    const float M = fmaxf(fmaxf(m_s[0][r], m_s[1][r]), fmaxf(m_s[2][r], m_s[3][r]));
    float L = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      L += l_s[w][r] * ex2(m_s[w][r] - (M == -INFINITY ? 0.f : M));
      x += O_s[w][r][d];
    }
    const float y = L == 0.f ? 0.f : x / L;
    const int li = pr / a.G;
    T* dst = static_cast<T*>(a.out) + (size_t)(first + li) * a.ldo + (size_t)(kvh * a.G + pr - li * a.G) * HD + d;
    *dst = (T)y;
  }
}

template <int HD, int BITS, typename T>
int attend_launch(AttendArgs a, cudaStream_t s) {
  // Sequences of few packed rows go to the decode kernel, the others here. A
  // batch of equal row counts needs one of the two only.
  const long long max_packed = (long long)a.v.max_rows * a.G;
  a.few = max_packed <= KVQ_DECODE_ROWS ? KVQ_DECODE_ROWS : a.G <= 8 ? 8 : KVQ_DECODE_ROWS;
  const bool equal = (long long)a.v.max_rows * a.v.n_seq == a.v.n_rows;
  if (max_packed <= a.few || !equal) {
    const int rc = kvq_decode_launch<HD, BITS, T>(a, (int)min(max_packed, (long long)a.few), s);
    if (rc) return rc;
  }
  if (max_packed <= a.few) return LUMINA_OK;
  const long long blocks = ((long long)a.v.n_rows * a.G + 15) / 16 + a.v.n_seq;
  const dim3 grid((unsigned)blocks, a.v.n_kv);
  kvq_attend_kernel<HD, BITS, T><<<grid, AT_THREADS, 0, s>>>(a);
  LUMINA_LAUNCH_CHECK();
  return LUMINA_OK;
}

}  // namespace
}  // namespace lumina

using namespace lumina;

extern "C" {

int lumina_kvq_workspace_bytes(int device, size_t* bytes) {
  LUMINA_CHECK_ARG(bytes, "kvq_workspace_bytes: null output");
  LUMINA_CHECK_ARG(device >= 0, "kvq_workspace_bytes: device %d", device);
  *bytes = kvq_ws_bytes();
  return LUMINA_OK;
}

int lumina_kvq_attend(const lumina_kvq_pool* pool, const lumina_kvq_batch* batch, const lumina_kvq_attend_args* args,
                      void* stream) {
  LUMINA_CHECK_ARG(pool && batch && args, "kvq_attend: null pool, batch or arguments");
  KvqDevice g(pool->device);
  LUMINA_CHECK_ARG(g.ok, "kvq_attend: device %d not available", pool->device);
  AttendArgs a{};
  int rc = kvq_view(pool, batch, "kvq_attend", &a.v);
  if (rc) return rc;
  LUMINA_CHECK_ARG(args->type == LUMINA_T_F32 || args->type == LUMINA_T_F16, "kvq_attend: type %d", args->type);
  LUMINA_CHECK_ARG(args->n_heads >= 1 && args->n_heads % pool->n_kv == 0, "kvq_attend: %d query heads over %d KV heads",
                   args->n_heads, pool->n_kv);
  LUMINA_CHECK_ARG(args->n_heads / pool->n_kv <= 128, "kvq_attend: %d query heads per KV head, at most 128",
                   args->n_heads / pool->n_kv);
  LUMINA_CHECK_ARG(std::isfinite(args->scale) && args->scale >= 0, "kvq_attend: scale %g", args->scale);
  LUMINA_CHECK_ARG(std::isfinite(args->softcap) && args->softcap >= 0, "kvq_attend: softcap %g", args->softcap);
  LUMINA_CHECK_ARG(args->window >= 0, "kvq_attend: window %d", args->window);
  size_t need = 0;
  if ((rc = lumina_kvq_workspace_bytes(pool->device, &need))) return rc;
  LUMINA_CHECK_ARG(args->workspace_dev && args->workspace_bytes >= need, "kvq_attend: workspace of %zu bytes, %zu needed",
                   args->workspace_bytes, need);
  LUMINA_CHECK_ARG(((uintptr_t)args->workspace_dev & 15) == 0, "kvq_attend: the workspace is not 16-byte aligned");
  if (batch->n_rows == 0) return LUMINA_OK;
  const int hd = pool->head_dim, width = args->n_heads * hd;
  if ((rc = kvq_check_rows(args->q_dev, args->ldq, width, args->type, "kvq_attend", "q"))) return rc;
  if ((rc = kvq_check_rows(args->out_dev, args->ldo, width, args->type, "kvq_attend", "out"))) return rc;
  a.q = args->q_dev;
  a.out = args->out_dev;
  a.ldq = args->ldq;
  a.ldo = args->ldo;
  a.nh = args->n_heads;
  a.G = args->n_heads / pool->n_kv;
  a.scale = args->scale > 0 ? args->scale : 1.0f / sqrtf((float)hd);
  a.cap = args->softcap;
  a.slopes = args->slopes_dev;
  a.prefix = args->prefix_dev;
  a.window = args->window;
  a.min_cells = 8;
  a.tickets = static_cast<int*>(args->workspace_dev);
  a.ws = reinterpret_cast<float*>(static_cast<uint8_t*>(args->workspace_dev) + KVQ_WS_TICKETS);
  a.spin = wait_spin_limit();
  cudaStream_t s = (cudaStream_t)stream;
  const bool f16 = args->type == LUMINA_T_F16;
  if (hd == 128 && pool->bits == 8) return f16 ? attend_launch<128, 8, __half>(a, s) : attend_launch<128, 8, float>(a, s);
  if (hd == 128) return f16 ? attend_launch<128, 4, __half>(a, s) : attend_launch<128, 4, float>(a, s);
  if (pool->bits == 8) return f16 ? attend_launch<64, 8, __half>(a, s) : attend_launch<64, 8, float>(a, s);
  return f16 ? attend_launch<64, 4, __half>(a, s) : attend_launch<64, 4, float>(a, s);
}

}  // extern "C"
