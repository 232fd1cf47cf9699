// Attention of sequences with few new rows (decode steps, short drafts) over
// quantized KV pages.
//
// A task is one (KV head, sequence, block of its new rows): up to 8 NR packed
// query rows (row r = local row r / G, head r % G); the blocks of one
// sequence share its keys through the L2. A task's keys are cut into cells of
// 32 (16 where the registers hold no more). All cells
// of all tasks form one line that the CTAs share evenly, so lengths may be as
// ragged as they like; a task that spans CTAs leaves partial states in the
// workspace, which the CTAs that arrive last join in part order (the result
// does not depend on who that is).
//
// Every warp takes its own cells (every W-th of the CTA's segment) straight
// from global memory to fragment registers, one cell ahead of its math and
// across task boundaries: the next cell's K codes are requested when this
// cell's are spent, its V codes likewise, so each waits through the other
// half's math, and no shared memory or barrier is in the loop. The scores are
// transposed, S^T = K Q^T and O^T = V^T P^T with mma.sync m16n8k16, so that
// 16 keys (or dims) fill the tensor pipe's 16 rows and the few query rows its
// 8 columns. The scales stay outside the products (kvq_mma.cuh). A row's
// reference is its own largest score times value scale (p times that scale
// has to fit fp16, and a key that the row does not see, or hardly, takes
// nothing from the others); it moves only when a key passes it by 2^8, so the
// steady state has no shuffles.
//
// Bound by the chain of a cell's math, from scores through exponentials to the
// second product: two warps per scheduler (a warp's registers hold a cell's
// codes and the output) issue 0.3 instructions a cycle, with DRAM at 27 to 45 %
// and the tensor pipe at 17 to 19 %. 64 sequences of up to 8192 tokens, 32 / 8
// heads of 128, int8, fp16 rows: 90 us, 0.69 of the copy rate (fp32 rows 106); 2
// sequences of up to 131072, 32 / 4 heads, int4: 62 us, 0.35 of it; one of 640
// tokens, 32 / 32 heads, fp32 rows: 12.4 us. CTAs of four warps, two per SM:
// one merges and joins while the other streams. A third CTA per SM spills at
// head dim 128 (the 64 sequences: 118 us).
//
// tcgen05 would need the codes rewritten as fp16 in shared memory and 128
// rows where these sequences have at most 8 NR.
#include <cfloat>
#include <type_traits>

#include "kvq_attend.cuh"
#include "kvq_mma.cuh"

namespace lumina {

namespace {

template <int HD, int BITS, int NR>
struct DecCfg {
  using F = KvqFrag<HD, BITS>;
  static constexpr int NK = NR == 2 && HD == 128 ? 1 : 2;  // 16-key tiles of one cell
  static constexpr int CELL = 16 * NK;
  // registers decide: o and q of 8 NR rows and one cell's codes
  static constexpr int W = 4;                               // warps
  static constexpr int PER_SM = 2;                          // CTAs per SM: one merges while the other streams
  static constexpr int THREADS = 32 * W;
  static constexpr int R = 8 * NR;                          // packed rows
  static constexpr int LD = HD + 4;
  static constexpr int SLAB = R * LD * 4;                   // one warp's O
  static constexpr int ITEMS = R * (HD / 4);                // 4-dim items that join parts
  static constexpr int JOIN = R * KVQ_FAN * 4;              // the parts' weights
  static constexpr int SMEM = W * SLAB > JOIN ? W * SLAB : JOIN;  // + n_seq ints
};

// One segment: cells [lo, hi) of the cell line of a task.
struct Seg {
  int s, kvh, lo, hi, total, blocks;  // total: the task's cells; blocks: the sequence's tasks of one KV head
  int first, n, len, pre, tp, tl;     // n rows from batch row `first`
  int p0;                             // position of the first
  __device__ __forceinline__ int at(int c) const { return c < tp ? c : c - tp + tl; }  // cell c's place in the cache, in cells
};

template <int HD, int BITS, int NR, typename T, bool PLAIN>
__global__ void __launch_bounds__((DecCfg<HD, BITS, NR>::THREADS), (DecCfg<HD, BITS, NR>::PER_SM)) kvq_decode_kernel(AttendArgs a) {
  constexpr bool F32 = sizeof(T) == 4;
  using C = DecCfg<HD, BITS, NR>;
  using F = typename C::F;
  constexpr int KK = F::KK, NT = F::NT, W = C::W, R = C::R, NK = C::NK, CELL = C::CELL;
  // fp16 rows spend next to no instructions on making numbers of the codes: K
  // and V enter the products raw, as fp16 subnormals (KvqFrag), and the zero
  // points come off again, K's as a start value of the accumulator, V's by one
  // more product. q is exact (to 2^-35 of its largest value) and the sums are
  // fp32 over terms of up to twice the codes' size, so a score is right to
  // about 2^-22 of sum |q k|. fp32 rows use signed codes and q as two fp16
  // parts. p is two fp16 parts for either: one alone would add 2.0e-4 of the
  // output to the 2.1e-4 of its rounding to fp16 (64 sequences of up to 8192:
  // 90 us, 89 with one part; 8 x 5 drafts 40, 39).
  constexpr bool FAST = !F32;
  // a chunk kernel of the same call may take the SMs that this one leaves
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(16) uint8_t sm[];
  float* slab = reinterpret_cast<float*>(sm);
  int* cells = reinterpret_cast<int*>(sm + C::SMEM);  // inclusive prefix of cells over sequences
  __shared__ float m_s[W][R], l_s[W][R], M_s[R], L_s[R];
  __shared__ unsigned scan_s[W];
  __shared__ int last_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const KvqView& v = a.v;
  const int cap_tokens = v.pages_ld << v.page_shift;
  const int block_rows = R / a.G;  // the launch has G <= R

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
    x.tp = (x.pre + CELL - 1) / CELL;
    x.tl = max(x.tp, lo / CELL);
    x.total = x.n ? max(1, x.tp + max(x.tl, (x.len + CELL - 1) / CELL) - x.tl) : 0;
    x.blocks = (x.n + block_rows - 1) / block_rows;
    x.p0 = p_lo;
  };

  // the cell line
  long long T_all = 0;
  for (int s0 = 0; s0 < v.n_seq; s0 += C::THREADS) {
    const int s = s0 + tid;
    Seg x;
    x.total = x.blocks = 0;
    if (s < v.n_seq) describe(s, x, blockIdx.x == 0);
    unsigned inc = (unsigned)min((long long)x.total * x.blocks, (long long)KVQ_MANY);
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const unsigned y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc = kvq_sum(inc, y);
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
  if (T_all == 0 || T_all * v.n_kv >= KVQ_MANY) {
    if (T_all && tid == 0) kvq_fault(v, KVQ_FAULT_DATA);
    return;
  }
  const unsigned Tn = (unsigned)T_all, U = Tn * (unsigned)v.n_kv;
  const unsigned share = max((U + gridDim.x - 1) / gridDim.x, (unsigned)W);  // a cell per warp
  const unsigned u0 = blockIdx.x * share, u1 = min(U, u0 + share);
  if (u0 >= U) return;

  // the segment that starts at unit u of this CTA's range
  auto segment = [&](unsigned u, Seg& x) {
    const int kvh = u / Tn, c = u - kvh * Tn;
    int lo = 0, hi = v.n_seq - 1;  // first s with cells[s] > c
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (cells[mid] > c) hi = mid;
      else lo = mid + 1;
    }
    describe(lo, x, false);
    x.kvh = kvh;
    const int base = lo ? cells[lo - 1] : 0;
    const int b = (c - base) / x.total;
    x.lo = c - base - b * x.total;
    x.first += b * block_rows;
    x.p0 += b * block_rows;
    x.n = min(block_rows, x.n - b * block_rows);
    x.hi = min(x.total, x.lo + (int)(u1 - u));
  };

  // ---- this warp's loads: the cell to load next starts at key `jn`, its
  // tile n holds keys if bit n of `have` is set (page 0 stands in where there
  // is nothing to read); its pages were asked for one cell earlier. All
  // addresses are this lane's own: kp (K codes) leads to the others.
  const int P = 1 << v.page_shift;
  const uint32_t page_bytes = (uint32_t)v.page_bytes;
  const bool one_page = P >= CELL;
  const int k_lane = g * F::NB + F::k_lane(t);
  const int v_step = P * F::NB + 2 * t * F::NB + F::v_lane(g) - k_lane;  // kp -> its V codes
  const int s_step = 2 * P * F::NB + 4 * g - k_lane;                     // page start's kp -> its first K scale
  Seg ps;
  segment(u0, ps);
  unsigned pu = u0;
  int pc = ps.lo + warp, pg[NK], pj = 0;
#pragma unroll
  for (int n = 0; n < NK; ++n) pg[n] = -2;  // a warp without a cell reads page 0 too
  const int* table = v.pages + (size_t)ps.s * v.pages_ld;
  const uint8_t* head = v.pool + (uint32_t)ps.kvh * v.block_bytes + k_lane;
  bool more = true;
  auto settle = [&]() {  // move to a cell of this warp and ask for its pages
    while (pc >= ps.hi) {
      pu += ps.hi - ps.lo;
      if (pu >= u1) {
        more = false;
        return;
      }
      segment(pu, ps);
      table = v.pages + (size_t)ps.s * v.pages_ld;
      head = v.pool + (uint32_t)ps.kvh * v.block_bytes + k_lane;
      pc = ps.lo + warp;
    }
    pj = ps.at(pc) * CELL;
    pg[0] = pj < ps.len ? __ldg(table + ((unsigned)pj >> v.page_shift)) : -2;
    if (!one_page) {
#pragma unroll
      for (int n = 1; n < NK; ++n) pg[n] = pj + 16 * n < ps.len ? __ldg(table + ((unsigned)(pj + 16 * n) >> v.page_shift)) : -2;
    }
  };
  const uint8_t *kp[NK], *sp[NK];
  int jn = 0;
  unsigned have = 0;
  auto place = [&](int n) {
    const bool good = (unsigned)pg[n] < (unsigned)v.n_pages;
    if (!good && more && pg[n] != -2 && lane == 0) kvq_fault(v, KVQ_FAULT_DATA);
    const uint8_t* page = head + (uint64_t)(good ? (uint32_t)pg[n] : 0u) * page_bytes;
    const uint32_t off = (pj + 16 * n) & (P - 1);
    kp[n] = page + off * F::NB;
    sp[n] = page + (int)(s_step + 4 * off);
    have |= good ? 1u << n : 0u;
  };
  auto advance = [&]() {
    jn = pj;
    have = 0;
    place(0);
#pragma unroll
    for (int n = 1; n < NK; ++n) {
      if (one_page) {
        kp[n] = kp[0] + 16 * n * F::NB;
        sp[n] = sp[0] + 64 * n;
        have |= have << n;
      } else {
        place(n);
      }
    }
    pc += W;
    if (more) settle();
  };
  uint32_t kw[NK][2][F::KW], vw[NK][4][F::VW];
  float sk[NK][2], sv[NK][2];
  auto load_k = [&]() {
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) F::load_k(kp[n] + h * 8 * F::NB, kw[n][h]);
  };
  auto load_v = [&]() {
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      const uint8_t* vp = kp[n] + v_step;
#pragma unroll
      for (int i = 0; i < 4; ++i) F::load_v(vp + ((i & 1) + 8 * (i >> 1)) * F::NB, vw[n][i]);
    }
  };
  auto load_s = [&]() {
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      const float *sc = reinterpret_cast<const float*>(sp[n]), *sd = sc + P;
      sk[n][0] = __ldg(sc);
      sk[n][1] = __ldg(sc + 8);
      sv[n][0] = __ldg(sd);
      sv[n][1] = __ldg(sd + 8);
    }
  };
  settle();
  advance();
  load_k();
  load_s();
  load_v();

  // ---- segments
  Seg x;
  for (unsigned u = u0; u < u1; u += x.hi - x.lo) {
    segment(u, x);
    // this thread's rows: 8 o + g in the Q fragments, 8 o + 2 t + c in the scores
    uint32_t qh[NR][KK][2], ql[F32 ? NR : 1][KK][2];
    float qmul[NR][2], off[FAST ? NR : 1][2], slope[PLAIN ? 1 : NR][2];
    int pos[NR][2];
    const float scale = !PLAIN && a.cap > 0.f ? a.scale / a.cap : a.scale * KVQ_LOG2E;
#pragma unroll
    for (int o = 0; o < NR; ++o) {
      const int r = 8 * o + g, i = r / a.G;
      const bool ok = r < x.n * a.G;
      float q[KK][4];
      F::load_q(static_cast<const T*>(a.q) + (size_t)(x.first + (ok ? i : 0)) * a.ldq +
                    (size_t)(x.kvh * a.G + (ok ? r - i * a.G : 0)) * HD,
                t, q);
      uint32_t top = 0;  // bits of the largest magnitude; past every finite one with an infinity or a NaN
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!ok) q[kk][e] = 0.f;
          top = max(top, __float_as_uint(q[kk][e]) & 0x7fffffffu);
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // bring the row's largest value near 2^10: room for 16 q, and for what
      // hi leaves to lo
      const int ex = min(112, max(-112, (int)(top >> 23) - 127));
      const float up = exp2i(10 - ex);
      float mul = scale * exp2i(ex - 10), zero = 0.f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
        for (int e = 0; e < 4; ++e) q[kk][e] *= up;
        if constexpr (F32) {
          qh[o][kk][0] = split_h2(q[kk][0], q[kk][1], ql[o][kk][0]);
          qh[o][kk][1] = split_h2(q[kk][2], q[kk][3], ql[o][kk][1]);
        } else {  // (plain, complemented) pairs as k_raw gives them
          constexpr int A = BITS == 8 ? 1 : 2, B = BITS == 8 ? 2 : 1;
          constexpr float LOW = BITS == 8 ? 1.f : 16.f;  // int4: b1's codes come times 16
          constexpr float Z0 = F::RAW_ZERO[0], Z1 = F::RAW_ZERO[1];
          zero += Z0 * (q[kk][0] + q[kk][A]) - Z1 * (q[kk][B] + q[kk][3]);
          qh[o][kk][0] = half2_bits(__floats2half2_rn(LOW * q[kk][0], -LOW * q[kk][B]));
          qh[o][kk][1] = half2_bits(__floats2half2_rn(q[kk][A], -q[kk][3]));
        }
      }
      if constexpr (FAST) {
        zero += __shfl_xor_sync(0xffffffffu, zero, 1);
        zero += __shfl_xor_sync(0xffffffffu, zero, 2);
        zero *= BITS == 8 ? -0x1p-24f : -0x1p-20f;
        mul *= BITS == 8 ? 0x1p24f : 0x1p21f;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int rr = 8 * o + 2 * t + c;
        qmul[o][c] = __shfl_sync(0xffffffffu, mul, (2 * t + c) * 4);
        if constexpr (FAST) off[o][c] = __shfl_sync(0xffffffffu, zero, (2 * t + c) * 4);
        const int li = rr < x.n * a.G ? rr / a.G : 0;
        pos[o][c] = x.p0 + li;
        if constexpr (!PLAIN)
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
    float oz[FAST ? NR : 1][4];  // the zero points' product
#pragma unroll
    for (int r = 0; r < (FAST ? NR : 1); ++r) oz[r][0] = oz[r][1] = oz[r][2] = oz[r][3] = 0.f;
    // m: the largest score plus V scale's size (kvq_size) when it last moved.
    // p = 2^(x - ms), ms = m - 7 (0 while nothing was seen): times its V scale
    // below 2^15, whatever the sizes of the V scales
    float m[NR][2], l[NR][2], ms[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) m[r][0] = m[r][1] = -INFINITY, l[r][0] = l[r][1] = ms[r][0] = ms[r][1] = 0.f;
    const float sign = FAST && (g & 1) ? -1.f : 1.f;  // odd keys' p (v_frag)

    // cells that start in [in_lo, in_hi] are seen by every row, as are those
    // that end within the prefix
    const int in_lo = a.window ? x.p0 + x.n - a.window : 0, in_hi = min(x.p0 + 1, x.len) - CELL, in_pre = x.pre - CELL;
    const int win_any = a.window ? x.p0 - a.window + 1 : -0x7fffffff;  // keys from here: some row
    for (int c = x.lo + warp; c < x.hi; c += W) {
      const int j0 = jn;
      const unsigned held = have;
      const bool inner = held == (1u << NK) - 1 && ((j0 >= in_lo && j0 <= in_hi) || j0 <= in_pre);
      float p[NK][NR][4];  // [tile][row octet][key half * 2 + row c]
#pragma unroll
      for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) p[n][r][e] = FAST ? off[FAST ? r : 0][e & 1] : 0.f;
      static_for<KK>([&](auto kc) {
        constexpr int kk = decltype(kc)::value;
#pragma unroll
        for (int n = 0; n < NK; ++n) {
          uint32_t f[4];
          F::template k_frag<kk, FAST>(kw[n][0], f[0], f[2]);
          F::template k_frag<kk, FAST>(kw[n][1], f[1], f[3]);
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            if constexpr (F32) mma_16816(p[n][r], f, ql[r][kk][0], ql[r][kk][1]);
            mma_16816(p[n][r], f, qh[r][kk][0], qh[r][kk][1]);
          }
        }
      });
      advance();
      load_k();
      if (!inner) {  // scales of keys that no row sees do not count
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int j = j0 + 16 * n + 8 * h + g;
            if (!((held >> n) & 1u) || j >= x.len || (j < win_any && j >= x.pre)) sk[n][h] = sv[n][h] = 0.f;
          }
      }
#pragma unroll
      for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) p[n][r][e] *= sk[n][e >> 1] * qmul[r][e & 1];
      if constexpr (!PLAIN) {
        if (a.cap > 0.f) {
#pragma unroll
          for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                p[n][r][e] = a.cap * KVQ_LOG2E * (F32 ? tanh_f32(p[n][r][e]) : tanh_fast(p[n][r][e]));
        }
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              p[n][r][e] = fmaf(-slope[r][e & 1], fabsf((float)(pos[r][e & 1] - (j0 + 16 * n + 8 * (e >> 1) + g))), p[n][r][e]);
      }
      if (!inner) {
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = j0 + 16 * n + 8 * (e >> 1) + g, pp = pos[r][e & 1];
              const bool see = ((held >> n) & 1u) && j < x.len &&
                               ((j <= pp && (a.window == 0 || j > pp - a.window)) || j < x.pre);
              if (!see) p[n][r][e] = -INFINITY;
            }
      }
      // past the reference by 2^8? A bound first: the thread's largest score
      // and largest V scale
      float svm = 0.f;
#pragma unroll
      for (int n = 0; n < NK; ++n) svm = fmaxf(svm, fmaxf(fabsf(sv[n][0]), fabsf(sv[n][1])));
      svm = kvq_size(svm);
      bool up = false;
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
          float mx = fmaxf(p[0][r][c2], p[0][r][2 + c2]);
#pragma unroll
          for (int n = 1; n < NK; ++n) mx = fmaxf(mx, fmaxf(p[n][r][c2], p[n][r][2 + c2]));
          up |= mx + svm > m[r][c2] + 8.f;
        }
      if (__any_sync(0xffffffffu, up)) {
        float size[NK][2];
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) size[n][h] = kvq_size(sv[n][h]);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          float fac[2];
#pragma unroll
          for (int c2 = 0; c2 < 2; ++c2) {
            float mx = m[r][c2];
#pragma unroll
            for (int n = 0; n < NK; ++n) mx = fmaxf(mx, fmaxf(p[n][r][c2] + size[n][0], p[n][r][2 + c2] + size[n][1]));
#pragma unroll
            for (int d = 4; d < 32; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            ms[r][c2] = mx == -INFINITY ? 0.f : mx - 7.f;
            fac[c2] = mx == -INFINITY ? 1.f : ex2(m[r][c2] - mx);
            m[r][c2] = mx;
            l[r][c2] *= fac[c2];
          }
#pragma unroll
          for (int i = 0; i < NT / 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[r][i][e] *= fac[e & 1];
          if constexpr (FAST) {
            oz[r][0] *= fac[0];
            oz[r][1] *= fac[1];
          }
        }
      }
      uint32_t pt[NK][NR][2], ptl[NK][NR][2];  // p's fp16 parts
      float lc[NR][2];  // sums of this cell's p: small ones would be lost beside the whole
#pragma unroll
      for (int r = 0; r < NR; ++r) lc[r][0] = lc[r][1] = 0.f;
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        const float vs[2] = {sv[n][0] * sign, sv[n][1] * sign};
#pragma unroll
        for (int r = 0; r < NR; ++r) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = p[n][r][e], y = ex2(x - ms[r][e & 1]);
            lc[r][e & 1] += y;
            // a masked key counts for nothing, whatever its scale holds
            p[n][r][e] = !inner && x == -INFINITY ? 0.f : y * vs[e >> 1];
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t lo;
            pt[n][r][h] = transpose8(split_h2(p[n][r][2 * h], p[n][r][2 * h + 1], lo));
            ptl[n][r][h] = transpose8(lo);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) l[r][0] += lc[r][0], l[r][1] += lc[r][1];
      load_s();
      constexpr int DPW = 32 / BITS;  // dims per code word
      if constexpr (FAST) {
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int w = 0; w < F::VW; ++w)
            static_for<DPW / 2>([&](auto ic) {
              constexpr int i = 2 * decltype(ic)::value;
              const uint32_t f[4] = {
                  F::template v_frag<i, true>(vw[n][0][w], vw[n][1][w]), F::template v_frag<i + 1, true>(vw[n][0][w], vw[n][1][w]),
                  F::template v_frag<i, true>(vw[n][2][w], vw[n][3][w]), F::template v_frag<i + 1, true>(vw[n][2][w], vw[n][3][w])};
#pragma unroll
              for (int r = 0; r < NR; ++r) {
                mma_16816(o[r][(w * DPW + i) / 2], f, ptl[n][r][0], ptl[n][r][1]);
                mma_16816(o[r][(w * DPW + i) / 2], f, pt[n][r][0], pt[n][r][1]);
              }
            });
      } else {
        // The tensor pipe cuts its sums off instead of rounding them, which
        // over thousands of keys shrinks an fp32 output by several 1e-6. A
        // cell's sums start at 0 and join the others by rounded additions (64
        // sequences of up to 8192: 106 us, 97 without).
#pragma unroll
        for (int w = 0; w < F::VW; ++w)
          static_for<DPW / 2>([&](auto ic) {
            constexpr int i = 2 * decltype(ic)::value;
            float d[NR][4];
#pragma unroll
            for (int r = 0; r < NR; ++r) d[r][0] = d[r][1] = d[r][2] = d[r][3] = 0.f;
#pragma unroll
            for (int n = 0; n < NK; ++n) {
              const uint32_t f[4] = {
                  F::template v_frag<i, false>(vw[n][0][w], vw[n][1][w]), F::template v_frag<i + 1, false>(vw[n][0][w], vw[n][1][w]),
                  F::template v_frag<i, false>(vw[n][2][w], vw[n][3][w]), F::template v_frag<i + 1, false>(vw[n][2][w], vw[n][3][w])};
#pragma unroll
              for (int r = 0; r < NR; ++r) {
                mma_16816(d[r], f, ptl[n][r][0], ptl[n][r][1]);
                mma_16816(d[r], f, pt[n][r][0], pt[n][r][1]);
              }
            }
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[r][(w * DPW + i) / 2][e] += d[r][e];
          });
      }
      if constexpr (FAST) {
        const uint32_t zp = half2_bits(__floats2half2_rn(F::RAW_ZERO[0], F::RAW_ZERO[1])), f[4] = {zp, zp, zp, zp};
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            mma_16816(oz[r], f, ptl[n][r][0], ptl[n][r][1]);
            mma_16816(oz[r], f, pt[n][r][0], pt[n][r][1]);
          }
      }
      load_v();
    }
    if constexpr (FAST) {  // sums of raw codes -> sums of values (int4: code = 2 c - 15, odd dims came times 16)
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int i = 0; i < NT / 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float up = BITS == 8 ? 16777216.f : e < 2 ? 33554432.f : 2097152.f;
            o[r][i][e] = fmaf(o[r][i][e], up, -(BITS == 8 ? 1.f : 2.f) * oz[r][e & 1]);
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
        const float f = ex2(m[r][c] - (M == -INFINITY ? 0.f : M));
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
    // the task's first and last CTA, by the line alone; its parts' slots: a
    // CTA's piece that begins a task is the odd one of its two
    const int cb = (u - x.lo) / share, ce = (u - x.lo + x.total - 1) / share;
    const size_t part = (size_t)R * (HD + 2);
    auto slot_of = [&](int p) { return 2 * (cb + p) + (p == 0 ? 1 : 0); };
    auto finish = [&](int r, int d, float4 y) {  // dims d .. d + 3 of packed row r
      const float L = L_s[r], inv = 1.0f / L;
      if (L == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);  // the row saw nothing
      else y = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
      const int li = r / a.G;
      kvq_store4(static_cast<T*>(a.out) + (size_t)(x.first + li) * a.ldo + (size_t)(x.kvh * a.G + r - li * a.G) * HD + d, y.x,
                 y.y, y.z, y.w);
    };
    float* mine = a.ws + slot_of(blockIdx.x - cb) * part;
    for (int i = tid; i < rows * (HD / 4); i += C::THREADS) {
      const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float4 z = *reinterpret_cast<const float4*>(slab + (w * R + r) * C::LD + d);
        y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
      }
      if (split) __stcg(reinterpret_cast<float4*>(mine + (size_t)r * HD + d), y);
      else finish(r, d, y);
    }
    if (split) {
      if (tid < rows) {
        mine[(size_t)R * HD + 2 * tid] = M_s[tid];
        mine[(size_t)R * HD + 2 * tid + 1] = L_s[tid];
      }
      // parts join in groups of KVQ_FAN, the groups' results (in their first
      // part's place) at the end; the last to arrive does each join
      const int np = (int)(ce - cb) + 1, ng = (np + KVQ_FAN - 1) / KVQ_FAN;
      for (int level = 0; level < 2; ++level) {
        const int p0 = level == 0 ? (int)(blockIdx.x - cb) / KVQ_FAN * KVQ_FAN : 0, step = level == 0 ? 1 : KVQ_FAN;
        const int cnt = level == 0 ? min(KVQ_FAN, np - p0) : ng;
        const bool last_level = level == 1 || ng == 1;
        // the CTA's writes are ordered before the barrier, and by the fence
        // of the thread that takes the ticket before the ticket
        __syncthreads();
        int* ticket = a.tickets + (level == 0 ? 0 : 2 * KVQ_MAX_CTAS) + slot_of(p0);
        if (tid == 0) {
          __threadfence();
          last_s = atomicAdd(ticket, 1) == cnt - 1;
          if (last_s) {
            __threadfence();
            *ticket = 0;
          }
        }
        __syncthreads();
        if (!last_s) break;
        auto part_at = [&](int k) { return a.ws + slot_of(p0 + k * step) * part; };
        float* wt = slab;  // [row][cnt] weights of the parts (the slab's readers are past the barrier)
        for (int r = warp; r < rows; r += W) {
          static_assert(KVQ_FAN == 64, "two parts per lane");
          float2 ml[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k = lane + 32 * h;
            ml[h] = k < cnt ? __ldcg(reinterpret_cast<const float2*>(part_at(k) + (size_t)R * HD) + r) : make_float2(-INFINITY, 0.f);
          }
          const float M = warp_max(fmaxf(ml[0].x, ml[1].x)), Ms = M == -INFINITY ? 0.f : M;
          float L = 0.f;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float f = ex2(ml[h].x - Ms);
            wt[r * KVQ_FAN + lane + 32 * h] = f;
            if (lane + 32 * h < cnt) L += f * ml[h].y;
          }
          L = warp_sum(L);
          if (lane == 0) {
            M_s[r] = M;
            L_s[r] = L;
          }
        }
        __syncthreads();
        // thread: 4 dims of a row, the parts in order
        static_assert(C::ITEMS % C::THREADS == 0, "whole passes of the CTA");
        for (int i = tid; i < C::ITEMS; i += C::THREADS) {
          const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          if (r < rows) {
#pragma unroll 16
            for (int k = 0; k < cnt; ++k) {
              const float4 z = __ldcg(reinterpret_cast<const float4*>(part_at(k) + (size_t)r * HD + d));
              const float f = wt[r * KVQ_FAN + k];
              y.x = fmaf(z.x, f, y.x); y.y = fmaf(z.y, f, y.y); y.z = fmaf(z.z, f, y.z); y.w = fmaf(z.w, f, y.w);
            }
          }
          if (r >= rows) continue;
          if (last_level) finish(r, d, y);
          else __stcg(reinterpret_cast<float4*>(part_at(0) + (size_t)r * HD + d), y);
        }
        if (last_level) break;
        if (tid < rows) {
          part_at(0)[(size_t)R * HD + 2 * tid] = M_s[tid];
          part_at(0)[(size_t)R * HD + 2 * tid + 1] = L_s[tid];
        }
      }
    }
    __syncthreads();  // slabs and statistics are free again
  }
}

template <int HD, int BITS, int NR, typename T>
int decode_nr(const AttendArgs& a, cudaStream_t s) {
  using C = DecCfg<HD, BITS, NR>;
  auto kern = a.cap > 0.f || a.slopes ? kvq_decode_kernel<HD, BITS, NR, T, false> : kvq_decode_kernel<HD, BITS, NR, T, true>;
  const size_t smem = C::SMEM + (size_t)a.v.n_seq * 4;
  const int rc = set_smem_limit((const void*)kern, C::SMEM + KVQ_MAX_SEQ * 4, "kvq_decode");
  if (rc) return rc;
  kern<<<min(C::PER_SM * sm_count(), KVQ_MAX_CTAS), C::THREADS, smem, s>>>(a);
  LUMINA_LAUNCH_CHECK();
  return LUMINA_OK;
}

}  // namespace

template <int HD, int BITS, typename T>
int kvq_decode_launch(AttendArgs a, int rows, cudaStream_t s) {
  return rows == 8 ? decode_nr<HD, BITS, 1, T>(a, s) : decode_nr<HD, BITS, 2, T>(a, s);
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
