// Attention of sequences with few new rows (decode steps, short drafts) over
// quantized KV pages: bound by the bytes of the cache.
//
// A task is one (KV head, sequence): up to 8 NR packed query rows (row r =
// local row r / G, head r % G). Its keys are cut into cells of 16. All cells
// of all tasks form one line that the CTAs share evenly (one CTA per SM), so
// lengths may be as ragged as they like; a task that spans CTAs leaves
// partial states in the workspace, and the CTA that arrives last merges them
// in CTA order (the result does not depend on who that is).
//
// Every warp streams its own cells (every W-th of the CTA's segment) through
// its own ring of shared-memory slots, across task boundaries, and computes
// on its own. The copies are cp.async of 16 bytes per lane: a cell is 2 to 4
// KB, so a bulk copy per piece with its barrier cost one lane more
// instructions than the whole warp now spends (608 -> see below), and each
// chunk can land where the fragment loads meet no bank conflict. The math is the scores transposed, S^T = K Q^T
// and O^T = V^T P^T with mma.sync m16n8k16, so that 16 keys (or dims) fill
// the tensor pipe's 16 rows and the few query rows its 8 columns. Codes go
// from shared memory to fragments in registers; the scales stay outside the
// products (kvq_mma.cuh). The running maximum moves only when a score passes
// it by 2^8 (p stays below 2^8), so the steady state has no shuffles.
//
// tcgen05 would need the codes rewritten as fp16 in shared memory and 128
// rows where these sequences have at most 8 NR; the cache's bytes bound this
// kernel well before the tensor pipe does.
#include <cfloat>
#include <type_traits>

#include "kvq_attend.cuh"
#include "kvq_mma.cuh"

namespace lumina {

namespace {

// 16 bytes global -> shared, asynchronously
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <int HD, int BITS, int NR>
struct DecCfg {
  using F = KvqFrag<HD, BITS>;
  static constexpr int W = 8 / NR;              // warps: W x NR octets of rows fill the merge slabs
  static constexpr int PER_SM = 2;              // CTAs per SM: one computes while the other merges
  static constexpr int THREADS = 32 * W;
  static constexpr int R = 8 * NR;              // packed rows
  static constexpr int SLOT = 16 * (2 * F::NB + 8);  // 16 keys: K codes, V codes, K scales, V scales
  static constexpr int LD = HD + 4;
  static constexpr int SLAB = R * LD * 4;       // one warp's O
  // merging parts: 4-dim items of a row, Q threads per item, weights and joins
  static constexpr int ITEMS = R * (HD / 4), Q = THREADS / ITEMS > 0 ? THREADS / ITEMS : 1;
  static constexpr int JOIN = (R * KVQ_MAX_CTAS + (Q - 1) * ITEMS * 4) * 4;
  static constexpr int MERGE = W * SLAB > JOIN ? W * SLAB : JOIN;
  static constexpr int RING = 227 * 1024 / PER_SM - MERGE - 10 * 1024;
  static constexpr int S0 = RING / (W * SLOT);
  static constexpr int S = S0 > 6 ? 6 : S0;     // slots per warp
  static_assert(S >= 2, "at least one copy in flight beside the slot in use");
  static constexpr size_t SMEM = (size_t)MERGE + (size_t)W * S * SLOT;  // + n_seq ints
};

// One segment: cells [lo, hi) of the cell line of (KV head, sequence).
struct Seg {
  int s, kvh, lo, hi, total;  // total: the task's cells
  int first, n, len, pre, tp, tl;
};

template <int HD, int BITS, int NR, typename T>
__global__ void __launch_bounds__(DecCfg<HD, BITS, NR>::THREADS, (DecCfg<HD, BITS, NR>::PER_SM))
kvq_decode_kernel(AttendArgs a) {
  using C = DecCfg<HD, BITS, NR>;
  using F = typename C::F;
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int KK = F::KK, NT = F::NT, W = C::W, S = C::S, R = C::R;
  // fp16 rows: K codes enter with their fp16 offset (1024 + ...), which a
  // start value of the accumulator takes off again; fp32 rows use exact codes
  constexpr bool OFFSET = !F32;
  extern __shared__ __align__(16) uint8_t sm[];
  float* slab = reinterpret_cast<float*>(sm);
  uint8_t* ring_all = sm + C::MERGE;
  int* cells = reinterpret_cast<int*>(ring_all + W * S * C::SLOT);  // inclusive prefix of cells over sequences
  __shared__ float m_s[W][R], l_s[W][R], M_s[R], L_s[R];
  __shared__ int scan_s[W], last_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const KvqView& v = a.v;
  const int cap_tokens = v.pages_ld << v.page_shift;

  // what the batch says about sequence s (0 rows: not this kernel's)
  auto describe = [&](int s, Seg& x, bool report) {
    x.s = s;
    x.n = kvq_seq_rows(v, s, x.first, report);
    if (x.n * a.G > a.few) x.n = 0;
    x.len = __ldg(v.len + s);
    if (x.len < 0 || x.len > cap_tokens) {
      if (report) kvq_fault(v, KVQ_FAULT_DATA);
      x.len = x.len < 0 ? 0 : cap_tokens;
    }
    x.pre = a.prefix ? min(x.len, max(0, __ldg(a.prefix + s))) : 0;
    // cells that the prefix shows, then those that the window shows
    const int p_lo = x.len - x.n, lo = a.window ? max(0, p_lo - a.window + 1) : 0;
    x.tp = (x.pre + 15) >> 4;
    x.tl = max(x.tp, lo >> 4);
    x.total = x.n ? max(1, x.tp + max(x.tl, (x.len + 15) >> 4) - x.tl) : 0;
  };

  // the cell line
  long long T_all = 0;
  for (int s0 = 0; s0 < v.n_seq; s0 += C::THREADS) {
    const int s = s0 + tid;
    Seg x;
    x.total = 0;
    if (s < v.n_seq) describe(s, x, blockIdx.x == 0);
    int inc = x.total;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) scan_s[warp] = inc;
    __syncthreads();
    long long before = T_all;
    for (int w = 0; w < W; ++w) {
      if (w < warp) before += scan_s[w];
      T_all += scan_s[w];
    }
    if (s < v.n_seq) cells[s] = (int)(before + inc);
    __syncthreads();
  }
  if (T_all == 0 || T_all > 0x7fffffffLL) {
    if (T_all && tid == 0) kvq_fault(v, KVQ_FAULT_DATA);
    return;
  }
  const int Tn = (int)T_all;
  const long long U = (long long)Tn * v.n_kv;
  const long long share = max((U + gridDim.x - 1) / gridDim.x, (long long)a.min_cells);
  const long long u0 = blockIdx.x * share, u1 = min(U, u0 + share);
  if (u0 >= U) return;

  // the segment that starts at unit u of this CTA's range
  auto segment = [&](long long u, Seg& x) {
    const int kvh = (int)(u / Tn), c = (int)(u - (long long)kvh * Tn);
    int lo = 0, hi = v.n_seq - 1;  // first s with cells[s] > c
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (cells[mid] > c) hi = mid;
      else lo = mid + 1;
    }
    describe(lo, x, false);
    x.kvh = kvh;
    const int base = lo ? cells[lo - 1] : 0;
    x.lo = c - base;
    x.hi = (int)min((long long)x.total, x.lo + (u1 - u));
  };

  // ---- the producing side of this warp: its next cell and that cell's page
  uint8_t* ring = ring_all + warp * S * C::SLOT;
  const int P = 1 << v.page_shift;
  Seg ps;
  segment(u0, ps);
  long long pu = u0;
  int pc = ps.lo + warp, pg = -1;
  bool more = true;
  auto settle = [&]() {  // move to a cell of this warp and ask for its page
    while (pc >= ps.hi) {
      pu += ps.hi - ps.lo;
      if (pu >= u1) {
        more = false;
        return;
      }
      segment(pu, ps);
      pc = ps.lo + warp;
    }
    const int j0 = (pc < ps.tp ? pc : pc - ps.tp + ps.tl) * 16;
    pg = j0 < ps.len ? __ldg(v.pages + (size_t)ps.s * v.pages_ld + (j0 >> v.page_shift)) : -2;
  };
  settle();
  int issued = 0;
  // bit per slot: a cell without a readable page, nothing was copied
  unsigned empty = 0;
  const int line = lane >> 3, lane_dst = line * 128 + (((lane & 7) ^ F::swz(line)) << 4);
  auto issue = [&]() {
    if (more) {
      const int slot = issued % S;
      const bool good = (unsigned)pg < (unsigned)v.n_pages;
      if (good) {
        const int j0 = (pc < ps.tp ? pc : pc - ps.tp + ps.tl) * 16, off = j0 & (P - 1);
        const uint8_t* blk = v.pool + (size_t)pg * v.page_bytes + (uint32_t)ps.kvh * v.block_bytes;
        const uint8_t* src = blk + off * F::NB + lane * 16;
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(ring + slot * C::SLOT);
        constexpr int CH = F::NB;  // chunks of 16 keys' codes
#pragma unroll
        for (int i = 0; i < CH / 32; ++i) {
          // four lines further the swizzle flips bit 2 (128-byte rows) or repeats
          const uint32_t d = dst + i * 512 + (F::NB == 128 && (i & 1) ? lane_dst ^ 64 : lane_dst);
          cp_async16(d, src + i * 512);
          cp_async16(d + 16 * F::NB, src + i * 512 + P * F::NB);
        }
        if (lane < 8)
          cp_async16(dst + 32 * F::NB + lane * 16, blk + 2 * P * F::NB + 4 * off + (lane & 4 ? 4 * P : 0) + (lane & 3) * 16);
      } else if (pg != -2 && lane == 0) {
        kvq_fault(v, KVQ_FAULT_DATA);
      }
      empty = (empty & ~(1u << slot)) | ((good ? 0u : 1u) << slot);
      ++issued;
      pc += W;
      settle();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int i = 0; i < S - 1; ++i) issue();

  // ---- segments
  int used = 0;
  Seg x;
  for (long long u = u0; u < u1; u += x.hi - x.lo) {
    segment(u, x);
    // this thread's rows: 8 o + g in the Q fragments, 8 o + 2 t + c in the scores
    uint32_t qh[NR][KK][2], ql[F32 ? NR : 1][KK][2];
    float qmul[NR][2], off[NR][2], slope[NR][2];
    int pos[NR][2];
    const float scale = a.cap > 0.f ? a.scale / a.cap : a.scale * KVQ_LOG2E;
#pragma unroll
    for (int o = 0; o < NR; ++o) {
      const int r = 8 * o + g, i = r / a.G;
      const bool ok = r < x.n * a.G;
      float q[KK][4];
      const T* src = static_cast<const T*>(a.q) + (size_t)(x.first + (ok ? i : 0)) * a.ldq +
                     (size_t)(x.kvh * a.G + (ok ? r - i * a.G : 0)) * HD;
      F::load_q(src, t, q);
      float m = 0.f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!ok) q[kk][e] = 0.f;
          m = fmaxf(m, fabsf(q[kk][e]));
        }
      // bring the row's largest value near 2^10: room for 16 q, and for what
      // hi leaves to lo
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const int ex = min(112, max(-112, (int)(__float_as_uint(m) >> 23) - 127));
      const float up = exp2i(10 - ex);
      float mul = scale * exp2i(ex - 10), sum = 0.f, lo_sum = 0.f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          q[kk][e] *= up;
          sum += q[kk][e];
          // int4: e = 0, 1 are low nibbles (1024 + c), 2 and 3 high ones (1024 + 16 c)
          if (OFFSET && BITS == 4 && e < 2) {
            lo_sum += q[kk][e];
            q[kk][e] *= 16.f;
          }
        }
        if constexpr (F32) {
          qh[o][kk][0] = split_h2(q[kk][0], q[kk][1], ql[o][kk][0]);
          qh[o][kk][1] = split_h2(q[kk][2], q[kk][3], ql[o][kk][1]);
        } else {
          qh[o][kk][0] = half2_bits(__floats2half2_rn(q[kk][0], q[kk][1]));
          qh[o][kk][1] = half2_bits(__floats2half2_rn(q[kk][2], q[kk][3]));
        }
      }
      float of = 0.f;
      if constexpr (OFFSET) {
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if constexpr (BITS == 8) {
          of = -1152.f * sum;
        } else {
          lo_sum += __shfl_xor_sync(0xffffffffu, lo_sum, 1);
          lo_sum += __shfl_xor_sync(0xffffffffu, lo_sum, 2);
          of = -(1024.f * (sum - lo_sum) + 16384.f * lo_sum + 120.f * sum);
          mul *= 0.125f;
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int rr = 8 * o + 2 * t + c;
        qmul[o][c] = __shfl_sync(0xffffffffu, mul, (2 * t + c) * 4);
        off[o][c] = __shfl_sync(0xffffffffu, of, (2 * t + c) * 4);
        const int li = rr < x.n * a.G ? rr / a.G : 0;
        pos[o][c] = x.len - x.n + li;
        slope[o][c] = a.slopes && rr < x.n * a.G ? __ldg(a.slopes + x.kvh * a.G + rr - li * a.G) * KVQ_LOG2E : 0.f;
      }
    }
    float o[NR][NT / 2][4];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int i = 0; i < NT / 2; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[r][i][c] = 0.f;
    float m[NR][2], l[NR][2], ms[NR][2];  // ms: m, 0 while nothing was seen
#pragma unroll
    for (int r = 0; r < NR; ++r) m[r][0] = m[r][1] = -INFINITY, l[r][0] = l[r][1] = ms[r][0] = ms[r][1] = 0.f;
    int ev = -100;         // V scales are taken relative to 2^ev
    float vmul = exp2i(7 + 100);

    for (int c = x.lo + warp; c < x.hi; c += W) {
      const int slot = used % S;
      ++used;
      // one group per cell: all but the newest S - 2 have landed, for every lane
      asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
      __syncwarp();
      issue();  // into the slot that the previous cell left
      const bool skip = (empty >> slot) & 1u;
      const uint8_t* ks = ring + slot * C::SLOT;
      const int j0 = (c < x.tp ? c : c - x.tp + x.tl) * 16;
      if (!skip) {
        uint32_t kw[2][F::KW], vw[4][F::VW];
#pragma unroll
        for (int h = 0; h < 2; ++h) F::load_k(ks, h * 8 + g, t, kw[h]);
        const float* sc = reinterpret_cast<const float*>(ks + 32 * F::NB);
        float sk[2] = {sc[g], sc[g + 8]}, sv[2] = {sc[16 + g], sc[24 + g]};
        const bool inner = j0 + 15 < x.len && ((j0 + 15 <= x.len - x.n && (a.window == 0 || j0 > x.len - 1 - a.window)) ||
                                               j0 + 15 < x.pre);
        if (!inner) {  // scales of keys that no row sees do not count
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int j = j0 + 8 * h + g;
            if (j >= x.len || (a.window && j < x.len - x.n - a.window + 1 && j >= x.pre)) sk[h] = sv[h] = 0.f;
          }
        }
        float p[NR][4];  // [row octet][key half * 2 + row c]
        {
          float acc[NR][4];
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[r][e] = OFFSET ? off[r][e & 1] : 0.f;
          static_for<KK>([&](auto kc) {
            constexpr int kk = decltype(kc)::value;
            uint32_t f[4];
            F::template k_frag<kk, OFFSET>(kw[0], f[0], f[2]);
            F::template k_frag<kk, OFFSET>(kw[1], f[1], f[3]);
#pragma unroll
            for (int r = 0; r < NR; ++r) {
              if constexpr (F32) mma_16816(acc[r], f, ql[r][kk][0], ql[r][kk][1]);
              mma_16816(acc[r], f, qh[r][kk][0], qh[r][kk][1]);
            }
          });
#pragma unroll
          for (int x4 = 0; x4 < 4; ++x4) F::load_v(ks + 16 * F::NB, 2 * t + (x4 & 1) + 8 * (x4 >> 1), g, vw[x4]);
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) p[r][e] = acc[r][e] * (sk[e >> 1] * qmul[r][e & 1]);
        }
        if (a.cap > 0.f) {
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) p[r][e] = a.cap * KVQ_LOG2E * (F32 ? tanhf(p[r][e]) : tanh_fast(p[r][e]));
        }
        if (a.slopes) {
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              p[r][e] = fmaf(-slope[r][e & 1], fabsf((float)(pos[r][e & 1] - (j0 + 8 * (e >> 1) + g))), p[r][e]);
        }
        if (!inner) {
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = j0 + 8 * (e >> 1) + g, pp = pos[r][e & 1];
              const bool see = j < x.len && ((j <= pp && (a.window == 0 || j > pp - a.window)) || j < x.pre);
              if (!see) p[r][e] = -INFINITY;
            }
        }
        // a score past the maximum by 2^8, or a V scale past 2^ev
        bool up = fmaxf(fabsf(sv[0]), fabsf(sv[1])) * vmul > 128.f;
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) up |= p[r][e] > m[r][e & 1] + 8.f;
        if (__any_sync(0xffffffffu, up)) {
          float svm = fmaxf(fabsf(sv[0]), fabsf(sv[1]));
#pragma unroll
          for (int d = 4; d < 32; d *= 2) svm = fmaxf(svm, __shfl_xor_sync(0xffffffffu, svm, d));
          const int en = max(ev, min(100, (int)(__float_as_uint(svm) >> 23) - 126));
          const float es = exp2i(max(-126, ev - en));
          ev = en;
          vmul = exp2i(7 - en);
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            float fac[2];
#pragma unroll
            for (int c2 = 0; c2 < 2; ++c2) {
              float mx = fmaxf(p[r][c2], p[r][2 + c2]);
#pragma unroll
              for (int d = 4; d < 32; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
              const float mn = fmaxf(m[r][c2], mx);
              fac[c2] = ex2(m[r][c2] - (mn == -INFINITY ? 0.f : mn));
              m[r][c2] = mn;
              ms[r][c2] = mn == -INFINITY ? 0.f : mn;
              l[r][c2] *= fac[c2];
              fac[c2] *= es;
            }
#pragma unroll
            for (int i = 0; i < NT / 2; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[r][i][e] *= fac[e & 1];
          }
        }
        uint32_t pt[NR][2], ptl[F32 ? NR : 1][2];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float y = ex2(p[r][e] - ms[r][e & 1]);
            l[r][e & 1] += y;
            // a masked key counts for nothing, whatever its scale holds
            p[r][e] = y == 0.f ? 0.f : y * (sv[e >> 1] * vmul);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if constexpr (F32) {
              uint32_t lo;
              pt[r][h] = transpose8(split_h2(p[r][2 * h], p[r][2 * h + 1], lo));
              ptl[r][h] = transpose8(lo);
            } else {
              pt[r][h] = transpose8(half2_bits(__floats2half2_rn(p[r][2 * h], p[r][2 * h + 1])));
            }
          }
        }
        constexpr int DPW = 32 / BITS;  // dims per code word
#pragma unroll
        for (int w = 0; w < F::VW; ++w)
          static_for<DPW / 2>([&](auto ic) {
            constexpr int i = 2 * decltype(ic)::value;
            const uint32_t f[4] = {F::template v_pair<i>(vw[0][w], vw[1][w]), F::template v_pair<i + 1>(vw[0][w], vw[1][w]),
                                   F::template v_pair<i>(vw[2][w], vw[3][w]), F::template v_pair<i + 1>(vw[2][w], vw[3][w])};
#pragma unroll
            for (int r = 0; r < NR; ++r) {
              if constexpr (F32) mma_16816(o[r][(w * DPW + i) / 2], f, ptl[r][0], ptl[r][1]);
              mma_16816(o[r][(w * DPW + i) / 2], f, pt[r][0], pt[r][1]);
            }
          });
      }
    }

    // ---- merge the warps
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float s = l[r][c];
#pragma unroll
        for (int d = 4; d < 32; d *= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (g == 0) {
          m_s[warp][8 * r + 2 * t + c] = m[r][c];
          l_s[warp][8 * r + 2 * t + c] = s;
        }
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int rr = 8 * r + 2 * t + c;
        float M = m_s[0][rr];
#pragma unroll
        for (int w = 1; w < W; ++w) M = fmaxf(M, m_s[w][rr]);
        const float f = ex2(m[r][c] - (M == -INFINITY ? 0.f : M)) * exp2i(ev - 7);
        float* dst = slab + (warp * R + rr) * C::LD + g * NT;
#pragma unroll
        for (int i = 0; i < NT / 4; ++i)
          *reinterpret_cast<float4*>(dst + 4 * i) =
              make_float4(o[r][2 * i][c] * f, o[r][2 * i][2 + c] * f, o[r][2 * i + 1][c] * f, o[r][2 * i + 1][2 + c] * f);
      }
    if (tid < R) {
      float M = m_s[0][tid], L = 0.f;
      for (int w = 1; w < W; ++w) M = fmaxf(M, m_s[w][tid]);
      for (int w = 0; w < W; ++w) L += l_s[w][tid] * ex2(m_s[w][tid] - (M == -INFINITY ? 0.f : M));
      M_s[tid] = M;
      L_s[tid] = L;
    }
    __syncthreads();
    const bool split = x.hi - x.lo < x.total;
    const int rows = x.n * a.G;
    // the task's first and last CTA, by the line alone
    const long long t0 = u - x.lo, cb = t0 / share, ce = (t0 + x.total - 1) / share;
    const int my = 2 * blockIdx.x + (x.lo == 0 ? 1 : 0);  // a head piece uses the odd slot
    const size_t part = (size_t)R * (HD + 2);
    for (int i = tid; i < rows * (HD / 4); i += C::THREADS) {
      const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float4 z = *reinterpret_cast<const float4*>(slab + (w * R + r) * C::LD + d);
        y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
      }
      if (split) {
        *reinterpret_cast<float4*>(a.ws + my * part + (size_t)r * HD + d) = y;
      } else {
        const float L = L_s[r], inv = L == 0.f ? 0.f : 1.0f / L;
        if (L == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);
        kvq_store4(static_cast<T*>(a.out) + (size_t)(x.first + r / a.G) * a.ldo + (size_t)(x.kvh * a.G + r % a.G) * HD + d,
                   y.x * inv, y.y * inv, y.z * inv, y.w * inv);
      }
    }
    if (split) {
      if (tid < rows) {
        a.ws[my * part + (size_t)R * HD + 2 * tid] = M_s[tid];
        a.ws[my * part + (size_t)R * HD + 2 * tid + 1] = L_s[tid];
      }
      __threadfence();
      __syncthreads();
      if (tid == 0) last_s = atomicAdd(&a.tickets[cb], 1) == (int)(ce - cb);
      __syncthreads();
      if (last_s) {
        __threadfence();
        // weights of the parts (slab is free: its readers are past the barrier)
        const int np = (int)(ce - cb) + 1;
        float* wt = slab;  // [row][np]
        for (int r = warp; r < rows; r += W) {
          float M = -INFINITY;
          for (int p = lane; p < np; p += 32) {
            const size_t at = (size_t)(2 * (cb + p) + (p == 0 ? 1 : 0)) * part + (size_t)R * HD + 2 * r;
            M = fmaxf(M, __ldcg(a.ws + at));
          }
          M = warp_max(M);
          float L = 0.f;
          for (int p = lane; p < np; p += 32) {
            const size_t at = (size_t)(2 * (cb + p) + (p == 0 ? 1 : 0)) * part + (size_t)R * HD + 2 * r;
            const float f = ex2(__ldcg(a.ws + at) - (M == -INFINITY ? 0.f : M));
            wt[r * np + p] = f;
            L += f * __ldcg(a.ws + at + 1);
          }
          L = warp_sum(L);
          if (lane == 0) L_s[r] = L;
        }
        __syncthreads();
        // thread: 4 dims of a row, every Q-th part; the Q sums join in order
        constexpr int ITEMS = C::ITEMS, Q = C::Q;
        float* join = slab + R * KVQ_MAX_CTAS;  // past the weights
        for (int i0 = 0; i0 < ITEMS * Q; i0 += C::THREADS) {
          const int i = (i0 + tid) % ITEMS, q = (i0 + tid) / ITEMS, r = i / (HD / 4), d = (i % (HD / 4)) * 4;
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          if (r < rows) {
#pragma unroll 4
            for (int p = q; p < np; p += Q) {
              const float4 z = __ldcg(reinterpret_cast<const float4*>(
                  a.ws + (size_t)(2 * (cb + p) + (p == 0 ? 1 : 0)) * part + (size_t)r * HD + d));
              const float f = wt[r * np + p];
              y.x = fmaf(z.x, f, y.x); y.y = fmaf(z.y, f, y.y); y.z = fmaf(z.z, f, y.z); y.w = fmaf(z.w, f, y.w);
            }
          }
          if constexpr (Q > 1) {
            if (q) *reinterpret_cast<float4*>(join + ((q - 1) * ITEMS + i) * 4) = y;
            __syncthreads();
            if (q) continue;
            for (int k = 1; k < Q; ++k) {
              const float4 z = *reinterpret_cast<const float4*>(join + ((k - 1) * ITEMS + i) * 4);
              y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
            }
          }
          if (r < rows) {
            const float L = L_s[r], inv = L == 0.f ? 0.f : 1.0f / L;
            if (L == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);
            kvq_store4(static_cast<T*>(a.out) + (size_t)(x.first + r / a.G) * a.ldo +
                           (size_t)(x.kvh * a.G + r % a.G) * HD + d,
                       y.x * inv, y.y * inv, y.z * inv, y.w * inv);
          }
        }
        if (tid == 0) a.tickets[cb] = 0;
      }
    }
    __syncthreads();  // slabs and statistics are free again
  }
}

template <int HD, int BITS, int NR, typename T>
int decode_nr(const AttendArgs& a, cudaStream_t s) {
  using C = DecCfg<HD, BITS, NR>;
  auto kern = kvq_decode_kernel<HD, BITS, NR, T>;
  const size_t smem = C::SMEM + (size_t)a.v.n_seq * 4;
  const int rc = set_smem_limit((const void*)kern, C::SMEM + KVQ_MAX_SEQ * 4, "kvq_decode");
  if (rc) return rc;
  kern<<<min(C::PER_SM * sm_count(), KVQ_MAX_CTAS), C::THREADS, smem, s>>>(a);
  LUMINA_LAUNCH_CHECK();
  return LUMINA_OK;
}

}  // namespace

template <int HD, int BITS, typename T>
int kvq_decode_launch(AttendArgs a, int max_packed, cudaStream_t s) {
  return max_packed <= 8 ? decode_nr<HD, BITS, 1, T>(a, s) : decode_nr<HD, BITS, 2, T>(a, s);
}
template int kvq_decode_launch<128, 8, __half>(AttendArgs, int, cudaStream_t);
template int kvq_decode_launch<128, 8, float>(AttendArgs, int, cudaStream_t);
template int kvq_decode_launch<128, 4, __half>(AttendArgs, int, cudaStream_t);
template int kvq_decode_launch<128, 4, float>(AttendArgs, int, cudaStream_t);
template int kvq_decode_launch<64, 8, __half>(AttendArgs, int, cudaStream_t);
template int kvq_decode_launch<64, 8, float>(AttendArgs, int, cudaStream_t);
template int kvq_decode_launch<64, 4, __half>(AttendArgs, int, cudaStream_t);
template int kvq_decode_launch<64, 4, float>(AttendArgs, int, cudaStream_t);

}  // namespace lumina
