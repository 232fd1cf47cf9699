// Attention of sequences with many new rows (prompt chunks, long drafts)
// over quantized KV pages, on the 5th-gen tensor cores.
//
// A task is one (KV head, sequence, block of packed query rows); packed row r
// is local row r / G, head r % G, so the G query heads that share a KV head
// share its dequantized tiles. Key tiles of 128:
//   S = Q K^T   tcgen05.mma, Q and K fp16 in shared memory, S in tensor memory
//   P = 2^(x - ref) * (V scale), fp16, over S's own columns in tensor memory
//   O += P V    tcgen05.mma, P from tensor memory, V fp16 in shared memory
// K and V codes are small integers, exact in fp16; the scales stay outside:
// a key's K scale multiplies its score column, its V scale its probability.
// fp32 rows send Q and P as two fp16 parts (hi + lo, about 22 bits) through
// the same tiles. fp16 rows keep one part of P: its rounding adds 2.0e-4 of the
// output to the 2.1e-4 of the output's own, and the second part costs an eighth
// of the speed (2048 rows behind 14K tokens: 928 us, 817 with one), most of it in
// the softmax warps.
//
// One CTA per SM, 13 warps:
//   warps 0-3, 4-7  softmax of row tile 0 and 1: a thread is a row, so
//                   maximum and sum need no shuffles
//   warps 8-11      codes from global memory to fp16 tiles (128-byte swizzle)
//   warp 12         issues every MMA, owns the tensor memory
// The two row tiles take turns on the tensor pipe: while one's S is being
// exponentiated the other's products run. With at most 128 packed rows (and
// always for fp32 rows) both softmax groups hold the SAME rows and take
// alternate key tiles, and merge at the end.
//
// A row's reference is its own largest score times value scale (P has to fit
// fp16, and a key that the row does not see, or hardly, takes nothing from the
// others). It moves only when P might leave fp16's range; only then O is
// rescaled in tensor memory.
//
// The key tiles of all tasks form one line that the CTAs share evenly; tasks
// that span CTAs leave partial states in the workspace, joined in part order
// by the CTA that arrives last. With more row blocks than the line holds,
// CTAs take whole tasks instead.
//
// Bound by the softmax warps, whose pass over a tile takes longer than the
// products it overlaps: by latency, with the tensor pipe at 29 % and 1.6
// instructions a cycle of 4. Two of them per scheduler walk two dependent
// passes over S in tensor memory (maximum, then exponentials), and 13 warps
// leave a thread 128 registers, which neither pass's next columns fit beside.
// 2048 rows behind 14K cached tokens, 32 / 8 heads of 128, int8, fp16 rows: 817
// us, 630 TFLOP/s (0.38 of the bf16 peak); 1024 fp32 rows behind 7K: 424 us.
// The loops' code size matters: the same with its helpers inline, twice the
// text, was 10 % slower. 301 rows of 28 / 4 heads of 64 over 4096 int4 keys,
// fp32 rows with cap, distance bias, window and prefix: 68 us.
//
// Waits are bounded: one that gives up sets bit 5 of the device fault word,
// every role leaves its loop, its rows stay unwritten (whoever joins their
// parts), and the CTA frees its tensor memory and exits.
#include <cfloat>
#include <type_traits>

#include "gemv_impl.cuh"
#include "kvq_attend.cuh"
#include "kvq_mma.cuh"

namespace lumina {

namespace {

constexpr int CK_KEYS = 128;                // keys per tile
constexpr int CK_DEQ = 8, CK_MMA = 12;      // first warp of the roles
constexpr int CK_THREADS = 32 * (CK_MMA + 1);
// P is about 2^LIFT at the key the reference was set by, and may grow to 2^15
// (fp16's range) before the reference moves. fp16 leaves a P (fp32 rows: its
// low part) an error of 2^-25 at least, which n keys add up to 2^-25 sqrt(n):
// at 128K keys 3e-5 of the largest P V for fp16 rows, 2e-7 for fp32 rows. A
// wide margin saves exact maxima (2048 rows behind 14K tokens: 838 us with
// LIFT 0, 823 with -2; fp32 rows, 1024 behind 7K: 429 us with 10, 415 with 5).
template <bool F32>
struct CkLift {
  static constexpr float LIFT = F32 ? 5.f : -2.f, MARGIN = 15.f - LIFT;
};
// The tensor pipe cuts its sums off instead of rounding them, which over
// thousands of keys shrinks an fp32 output by several 1e-6. A softmax group of
// fp32 rows takes O out of tensor memory after every CK_SUM of its tiles and
// adds it to a sum in the workspace, rounded (1024 rows behind 7K tokens: an
// error of 9.6e-7 and 424 us; 1.7e-6 after every 8 tiles, 3 % faster; 4.8e-6 at
// the end alone).
constexpr int CK_SUM = 4;
constexpr int CK_TILE = 128 * 128;          // bytes of a [128 rows][64 fp16] block
constexpr uint32_t CK_S = 0, CK_O = 256;    // tensor memory columns: S tiles, O tiles, 128 apart

template <int HD>
struct CkCfg {
  static constexpr int BLKS = HD / 64;               // 64-dim blocks of a tile
  static constexpr int BYTES = BLKS * CK_TILE;       // one K, V or Q tile
  static constexpr int Q_BYTES = 2 * 128 * HD * 2 > 128 * HD * 4 ? 2 * 128 * HD * 2 : 128 * HD * 4;
  static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + 2 * BYTES, OFF_SC = OFF_V + 2 * BYTES;
  static constexpr int OFF_LINE = OFF_SC + 2 * 3 * CK_KEYS * 4;  // [stage][K scale | V scale | its size (kvq_size)][key]
  static constexpr size_t SMEM = OFF_LINE + (size_t)KVQ_MAX_BLOCKS * 4 + 1024;  // + n_seq ints
};

__device__ __forceinline__ void ck_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ck_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ck_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void ck_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void ck_mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, int acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void ck_mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, int acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(db), "r"(idesc), "r"(acc)
      : "memory");
}
// shared-memory descriptors, 128-byte swizzle. K-major: 8-row groups 1024
// bytes apart. MN-major (V: the dims are contiguous): 64-dim blocks CK_TILE
// bytes apart (leading offset), 8-key groups 1024 bytes apart (stride offset).
__device__ __forceinline__ uint64_t ck_desc(uint32_t saddr, uint32_t lead) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lead >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// fp16 A and B, fp32 D, M = 128; bit 16: B is MN-major
__host__ __device__ constexpr uint32_t ck_idesc(int N, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void ck_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void ck_ld16(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// the loads issued so far are in their registers; v may be used after this
template <int N>
__device__ __forceinline__ void ck_wait_ld(float (&v)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void ck_get32(uint32_t addr, float (&v)[32]) {
  ck_ld32(addr, v);
  ck_wait_ld(v);
}
// two fp32 operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 a, b, c;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 a, a, b, c;\n mov.b64 {%0, %1}, a;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ void ck_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void ck_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void ck_st32(uint32_t addr, const float (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
      "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]),
      "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]),
      "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31])
      : "memory");
}
// one lane of a converged warp, always the same
__device__ __forceinline__ bool ck_elect() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void ck_ld8(uint32_t addr, float (&v)[8]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = __uint_as_float(r[i]);
    asm volatile("" : "+f"(v[i]));
  }
}
template <int N>
__device__ __forceinline__ void ck_get(uint32_t addr, float (&v)[N]) {
  if constexpr (N == 32) ck_get32(addr, v);
  else ck_ld8(addr, v);
}
template <int N>
__device__ __forceinline__ void ck_put(uint32_t addr, const uint32_t (&r)[N]) {
  if constexpr (N == 16)
    ck_st16(addr, r);
  else
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
}
__device__ __forceinline__ void ck_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One segment: key tiles [lo, hi) of one task.
struct CkSeg {
  int kvh, s, first, n, len, pre;
  int row0, rows;         // packed rows of the block
  int tp, tl;             // tiles that the prefix shows; first tile that the window shows
  int lo, hi, total;
  bool alt;               // both softmax groups hold the same rows, alternate key tiles
  __device__ __forceinline__ int key(int c) const { return (c < tp ? c : c - tp + tl) * CK_KEYS; }
};

// The line of units as a CTA sees it.
struct CkLine {
  const AttendArgs& a;
  const int *line, *blocks;
  int NBt, Tn;
  unsigned u0, u1;
  bool whole;
};

// task b of the block line (any KV head): everything but kvh, lo, hi
template <int BM>
__device__ __noinline__ void ck_describe(const CkLine& ln, int b, CkSeg& x) {
  const AttendArgs& a = ln.a;
  const KvqView& v = a.v;
  int lo = 0, hi = v.n_seq - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ln.blocks[mid] > b) hi = mid;
    else lo = mid + 1;
  }
  x.s = lo;
  x.n = kvq_seq_rows(v, lo, x.first, false);
  x.len = min(v.pages_ld << v.page_shift, max(0, __ldg(v.len + lo)));
  x.pre = a.prefix ? min(x.len, max(0, __ldg(a.prefix + lo))) : 0;
  x.row0 = (b - (lo ? ln.blocks[lo - 1] : 0)) * BM;
  x.rows = min(BM, x.n * a.G - x.row0);
  x.alt = x.rows <= 128;
  const int p0 = x.len - x.n, p_lo = p0 + x.row0 / a.G, p_hi = p0 + (x.row0 + x.rows - 1) / a.G;
  const int k_hi = min(x.len, max(0, p_hi + 1)), k_lo = a.window ? min(k_hi, max(0, p_lo - a.window + 1)) : 0;
  x.tp = (x.pre + CK_KEYS - 1) / CK_KEYS;
  x.tl = max(x.tp, k_lo / CK_KEYS);
  x.total = max(1, x.tp + max(x.tl, (k_hi + CK_KEYS - 1) / CK_KEYS) - x.tl);
}

// the segment that starts at unit u; returns the next segment's unit. Out of
// line: once per segment, and the loops that call it have to fit the
// instruction cache.
template <int BM>
__device__ __noinline__ unsigned ck_segment(const CkLine& ln, unsigned u, CkSeg& x) {
  const int kvh = u / ln.Tn, c = u - kvh * ln.Tn;
  if (ln.whole) {
    ck_describe<BM>(ln, c, x);
    x.kvh = kvh;
    x.lo = 0;
    x.hi = x.total;
    return u + gridDim.x;
  }
  int lo = 0, hi = ln.NBt - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ln.line[mid] > c) hi = mid;
    else lo = mid + 1;
  }
  ck_describe<BM>(ln, lo, x);
  x.kvh = kvh;
  x.lo = c - (lo ? ln.line[lo - 1] : 0);
  x.hi = (int)min((unsigned)x.total, x.lo + (ln.u1 - u));
  return u + (unsigned)(x.hi - x.lo);
}

template <int HD, int BITS, typename T, bool PLAIN>
__global__ void __launch_bounds__(CK_THREADS, 1) kvq_chunk_kernel(const __grid_constant__ AttendArgs a) {
  using C = CkCfg<HD>;
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int BM = F32 ? 128 : 256;                    // packed rows of a block
  constexpr int NB = HD * BITS / 8;                      // code bytes of a key
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* scale_s = reinterpret_cast<float*>(sm + C::OFF_SC);
  int* line = reinterpret_cast<int*>(sm + C::OFF_LINE);  // inclusive prefix of tiles over blocks
  int* blocks = line + KVQ_MAX_BLOCKS;                   // inclusive prefix of blocks over sequences
  __shared__ __align__(8) uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], q_full, idle;
  __shared__ uint32_t tmem_s;
  __shared__ __align__(8) float2 most_s[2][4];  // of each 32 keys of a tile: the largest K scale, the largest V scale's size
  __shared__ unsigned scan_s[CK_THREADS / 32];
  __shared__ int abort_s, last_s;
  __shared__ float m_s[128], l_s[128];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const KvqView& v = a.v;
  const int cap_tokens = v.pages_ld << v.page_shift;
  volatile int* abort_v = &abort_s;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&v_full[i], 4);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&o_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    mbar_init(&q_full, 8);
    mbar_init(&idle, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    abort_s = 0;
  }
  if (warp == CK_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }

  // ---- the line of key tiles
  auto block_scan = [&](unsigned x, unsigned& total) {  // inclusive over the CTA; two barriers
    unsigned inc = x;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const unsigned y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc = kvq_sum(inc, y);
    }
    if (lane == 31) scan_s[warp] = inc;
    __syncthreads();
    total = 0;
    for (int w = 0; w < CK_THREADS / 32; ++w) {
      if (w < warp) inc = kvq_sum(inc, scan_s[w]);
      total = kvq_sum(total, scan_s[w]);
    }
    __syncthreads();
    return inc;
  };
  int NBt = 0;
  for (int s0 = 0; s0 < v.n_seq; s0 += CK_THREADS) {
    const int s = s0 + tid;
    int first, nb = 0;
    unsigned total;
    if (s < v.n_seq) {
      const int n = kvq_seq_rows(v, s, first, blockIdx.x == 0);
      if ((long long)n * a.G > a.few) nb = (int)(((long long)n * a.G + BM - 1) / BM);
      const int len = __ldg(v.len + s);
      if (nb && (len < 0 || len > cap_tokens) && blockIdx.x == 0) kvq_fault(v, KVQ_FAULT_DATA);
    }
    const unsigned inc = block_scan(nb, total);
    if (s < v.n_seq) blocks[s] = kvq_sum(NBt, inc);
    NBt = kvq_sum(NBt, total);
  }
  __syncthreads();
  CkLine ln{a, line, blocks, 0, 0, 0u, 0u, false};
  ln.NBt = NBt;
  const bool whole = ln.whole = NBt > KVQ_MAX_BLOCKS;  // whole tasks: the line does not hold them
  int Tn = NBt;                             // units of one KV head: tiles, or tasks
  if (!whole) {
    Tn = 0;
    for (int b0 = 0; b0 < NBt; b0 += CK_THREADS) {
      CkSeg x;
      x.total = 0;
      unsigned total;
      if (b0 + tid < NBt) ck_describe<BM>(ln, b0 + tid, x);
      const unsigned inc = block_scan(x.total, total);
      if (b0 + tid < NBt) line[b0 + tid] = kvq_sum(Tn, inc);
      Tn = kvq_sum(Tn, total);
    }
  }
  ck_fence_before();
  __syncthreads();
  ck_fence_after();
  const uint32_t tmem = tmem_s;
  const long long U64 = (long long)Tn * v.n_kv;
  const unsigned U = U64 >= KVQ_MANY ? 0u : (unsigned)U64;
  if (U64 >= KVQ_MANY && tid == 0) kvq_fault(v, KVQ_FAULT_DATA);
  const unsigned share = whole ? 1u : max((U + gridDim.x - 1) / gridDim.x, 1u);  // (300 tokens x 285 rows: 29 us, 41 with two tiles at least)
  // units [u0, u1), or tasks u0, u0 + gridDim.x, ...
  const unsigned u0 = whole ? blockIdx.x : min(U, blockIdx.x * share), u1 = whole ? U : min(U, u0 + share);
  ln.Tn = Tn;
  ln.u0 = u0;
  ln.u1 = u1;
  auto segment = [&](unsigned u, CkSeg& x) { return ck_segment<BM>(ln, u, x); };  // returns the next segment's unit
  auto give_up = [&]() {
    if (!*abort_v) kvq_fault(v, KVQ_FAULT_WAIT);
    *abort_v = 1;
  };
  const unsigned spin = (unsigned)min(a.spin, 0x7fffffffLL);
  // a whole warp waits; false when this wait or, meanwhile, any role gave up
  auto wait = [&](uint64_t* bar, unsigned phase) {
    bool in = false;
#pragma unroll 1
    for (unsigned i = 0; i < spin; ++i) {
      if (mbar_try_wait(bar, phase & 1)) {
        in = true;
        break;
      }
      if ((i & 1023u) == 1023u && *abort_v) break;
    }
    in = __all_sync(0xffffffffu, in);
    if (!in && lane == 0) give_up();
    return in;
  };
  const int P = 1 << v.page_shift;

  if (warp >= CK_DEQ && warp < CK_MMA) {
    // ======== codes -> fp16 tiles. A row is LPR 16-byte words of codes, one
    // lane each; a pass of the 128 threads covers 128 / LPR rows.
    constexpr int LPR = NB / 16, RPP = 128 / LPR, NP = LPR;
    const int dt = tid - 32 * CK_DEQ, dw = warp - CK_DEQ;
    // 128-byte rows: eight consecutive lanes take half a row each of two
    // neighbouring rows, whose stores meet different banks
    const int wr = LPR == 8 ? dw * 4 + ((lane >> 2) & 1) + 2 * (lane >> 4) : dt / LPR;
    const int wc = LPR == 8 ? (lane & 3) + 4 * ((lane >> 3) & 1) : dt % LPR;
    unsigned fill = 0;  // tiles filled so far (stage = fill & 1)
    bool dead = false;
    for (unsigned u = u0; u < u1 && !dead;) {
      CkSeg x;
      u = segment(u, x);
      const uint8_t* base = v.pool + (size_t)x.kvh * v.block_bytes;
      const int* table = v.pages + (size_t)x.s * v.pages_ld;
      const float kmul = a.cap > 0.f ? a.scale / a.cap : a.scale * KVQ_LOG2E;
      const int win_any = a.window ? x.len - x.n + x.row0 / a.G - a.window + 1 : -0x7fffffff;
      // lane i & 7 knows the page of 16-key group i of a tile (-2: no key there)
      auto ask = [&](int c) {
        const int j = x.key(c) + (lane & 7) * 16;
        return c < x.hi && j < x.len ? __ldg(table + (j >> v.page_shift)) : -2;
      };
      auto load = [&](int c, int pages, bool isv, uint4 (&w)[NP]) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const int r = p * RPP + wr;
          const int pg = __shfl_sync(0xffffffffu, pages, r >> 4);
          const int off = (x.key(c) + r) & (P - 1);
          const bool good = (unsigned)pg < (unsigned)v.n_pages;
          w[p] = ldg_stream(base + (size_t)(good ? pg : 0) * v.page_bytes + (size_t)((isv ? P : 0) + off) * NB + wc * 16);
        }
      };
      auto store = [&](const uint4 (&w)[NP], uint8_t* tile) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const int r = p * RPP + wr;
          const uint32_t ws[4] = {w[p].x, w[p].y, w[p].z, w[p].w};
          if constexpr (BITS == 8) {
            // 16 dims: chunks 2 wc, 2 wc + 1 (of 8 dims) of block wc / 4
            uint4 q[2];
            uint32_t* qq = reinterpret_cast<uint32_t*>(q);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t f = ws[i] ^ 0x80808080u;
              qq[2 * i] = s8_pair<0x4140>(f);
              qq[2 * i + 1] = s8_pair<0x4342>(f);
            }
            uint8_t* dst = tile + (wc >> 2) * CK_TILE + r * 128;
            const int c0 = 2 * (wc & 3);
#pragma unroll
            for (int i = 0; i < 2; ++i) *reinterpret_cast<uint4*>(dst + (((c0 + i) ^ (r & 7)) << 4)) = q[i];
          } else {
            // 32 dims, one chunk per word, order 0 4 1 5 2 6 3 7 within it
            uint8_t* dst = tile + (wc >> 1) * CK_TILE + r * 128;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t n = ws[i];
              const uint4 q = make_uint4(u4_pair(n << 4), u4_pair(n), u4_pair(n >> 4), u4_pair(n >> 8));
              *reinterpret_cast<uint4*>(dst + (((4 * (wc & 1) + i) ^ (r & 7)) << 4)) = q;
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      };
      // order: K 0, K 1, V 0, K 2, V 1, ...: S of a tile is wanted before P V
      // of the one before it. A step's codes (and scales) are asked for when
      // the step before is stored, its page numbers a step earlier.
      const int nt = x.hi - x.lo;
      auto after = [&](int s) {  // steps are 2 * tile + (V ? 1 : 0); 2 nt: the end
        const int c = s >> 1;
        if (s & 1) return c + 2 < nt ? s + 3 : s + 2 < 2 * nt ? s + 2 : 2 * nt;
        return c == 0 ? (nt > 1 ? 2 : 1) : s - 1;
      };
      uint4 w[NP];
      float sk = 0.f, sv = 0.f;
      int s0 = -1, s1 = 0, pg1 = ask(x.lo);  // the step in registers, the next one and its pages
#pragma unroll 1
      while (true) {
        if (s0 >= 0) {
          const unsigned f = fill + (s0 >> 1);
          const int st = f & 1;
          if (f >= 2 && !wait((s0 & 1 ? v_empty : k_empty) + st, (f >> 1) + 1)) {
            dead = true;
            break;
          }
          store(w, sm + (s0 & 1 ? C::OFF_V : C::OFF_K) + st * C::BYTES);
          if (s0 & 1) {
            scale_s[st * 384 + dt] = sk;
            scale_s[st * 384 + 128 + dt] = sv;
            scale_s[st * 384 + 256 + dt] = kvq_size(sv);
            // largest scales of 32 keys (bits order like the values; a NaN does not count)
            const uint32_t kb = __float_as_uint(sk) & 0x7fffffffu, vb = __float_as_uint(sv) & 0x7fffffffu;
            const uint32_t km = __reduce_max_sync(0xffffffffu, kb > 0x7f800000u ? 0u : kb);
            const uint32_t vm = __reduce_max_sync(0xffffffffu, vb > 0x7f800000u ? 0u : vb);
            if (lane == 0) {
              most_s[st][dw] = make_float2(__uint_as_float(km), kvq_size(__uint_as_float(vm)));
            }
          }
          __syncwarp();
          if (lane == 0) ck_arrive((s0 & 1 ? v_full : k_full) + st);
        }
        if (s1 >= 2 * nt) break;
        load(x.lo + (s1 >> 1), pg1, s1 & 1, w);
        if (s1 & 1) {  // the tile's scales (thread = key)
          const int j = x.key(x.lo + (s1 >> 1)) + dt;
          const int pg = __shfl_sync(0xffffffffu, pg1, dt >> 4);
          const bool there = j < x.len && (unsigned)pg < (unsigned)v.n_pages;
          if (j < x.len && !there && pg != -2) kvq_fault(v, KVQ_FAULT_DATA);
          sk = sv = 0.f;
          if (there && (j >= win_any || j < x.pre)) {
            const float* sc = reinterpret_cast<const float*>(base + (size_t)pg * v.page_bytes + 2 * P * NB) + (j & (P - 1));
            sk = __ldg(sc);
            sv = __ldg(sc + P);
          }
          sk *= kmul;
        }
        s0 = s1;
        s1 = after(s1);
        pg1 = ask(x.lo + (s1 >> 1));
      }
      fill += x.hi - x.lo;
    }
  } else if (warp == CK_MMA) {
    // ======== every MMA. Step j of a segment: softmax group j & 1, key tile
    // j (alternating) or j / 2; S of step j + 2 follows P V of step j, and
    // the groups' steps alternate, so that one group exponentiates while the
    // other's products run. The whole warp walks the loop and one elected
    // lane issues: what is uniform stays in uniform registers, and eight MMAs
    // issue in 70 to 150 cycles where a lone thread took 390 (they run for 515).
    constexpr uint32_t ID_S = ck_idesc(128, false), ID_O = ck_idesc(HD, true);
    const bool lead = ck_elect();
    const uint32_t sb = __shfl_sync(0xffffffffu, smem_u32(sm), 0);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    unsigned fill = 0, seg = 0, np0 = 0, np1 = 0;
    bool dead = false;
    for (unsigned u = u0; u < u1 && !dead; ++seg) {
      CkSeg x;
      u = segment(u, x);
      const bool alt = x.alt;
      const int nt = x.hi - x.lo, J = alt ? nt : 2 * nt;
      dead = !wait(&q_full, seg);
      // j = -2, -1 only ask for the first S of each group
#pragma unroll 1
      for (int j = -2; j < J && !dead; ++j) {
        const int t = __shfl_sync(0xffffffffu, j & 1, 0);
        if (j >= 0) {
          const unsigned f = fill + (alt ? j : j >> 1);
          const int st = __shfl_sync(0xffffffffu, f & 1, 0);
          dead = ((alt || t == 0) && !wait(&v_full[st], f >> 1)) || !wait(&p_full[t], t ? np1 : np0);
          if (dead) break;
          if (t) ++np1;
          else ++np0;
          ck_fence_after();
          const uint64_t vd = ck_desc(sb + C::OFF_V + st * C::BYTES, CK_TILE);
          const uint32_t d = tm + CK_O + t * 128, p = tm + CK_S + t * 128;
          const int fresh = F32 ? (j >> 1) % CK_SUM == 0 : j < 2;  // O starts here
          if (lead) {
#pragma unroll
            for (int part = 0; part < (F32 ? 2 : 1); ++part)
#pragma unroll
              for (int kk = 0; kk < CK_KEYS / 16; ++kk)
                ck_mma_ts(d, p + (kk >> 1) * 32 + (kk & 1) * 8 + (F32 ? (1 - part) * 16 : 0), vd + kk * (2048 >> 4), ID_O,
                          (part | kk) != 0 || !fresh);
            if (alt || t == 1) ck_commit(&v_empty[st]);
            if (j + 2 >= J) ck_commit(&o_full[t]);
          }
          __syncwarp();
        }
        if (j + 2 < J) {
          const unsigned f = fill + (alt ? j + 2 : (j + 2) >> 1);
          const int st = __shfl_sync(0xffffffffu, f & 1, 0);
          dead = (alt || t == 0) && !wait(&k_full[st], f >> 1);
          if (dead) break;
          ck_fence_after();
          const uint64_t kd = ck_desc(sb + C::OFF_K + st * C::BYTES, 16);
          const uint64_t qd = ck_desc(sb + (F32 || alt ? 0 : t * C::BYTES), 16);
          const uint32_t d = tm + CK_S + t * 128;
          if (lead) {
#pragma unroll
            for (int part = 0; part < (F32 ? 2 : 1); ++part)  // fp32 rows: lo, then hi
#pragma unroll
              for (int kk = 0; kk < HD / 16; ++kk) {
                const uint32_t o = ((kk >> 2) * CK_TILE + (kk & 3) * 32) >> 4;
                ck_mma_ss(d, qd + (F32 ? (1 - part) * C::BYTES >> 4 : 0) + o, kd + o, ID_S, (part | kk) != 0);
              }
            ck_commit(&s_full[t]);
            if (alt || t == 1) ck_commit(&k_empty[st]);
          }
          __syncwarp();
        }
      }
      fill += nt;
    }
    if (lead) ck_commit(&idle);  // completes once every MMA issued above is done
  } else {
    // ======== softmax: thread = row
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;  // row of its tile
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_tm = tmem + lanes + CK_S + t * 128, o_tm = tmem + lanes + CK_O + t * 128;
    unsigned fill = 0, ns = 0, no = 0;
    bool dead = false;
    auto pair_bar = [&]() { asm volatile("bar.sync 1, 256;" ::: "memory"); };
    for (unsigned u = u0; u < u1;) {
      CkSeg x;
      const unsigned un = segment(u, x);
      const int nt = x.hi - x.lo;
      const int pr = x.row0 + (x.alt ? 0 : t * 128) + row;  // packed row
      const bool ok = pr < x.row0 + x.rows;
      const int li = ok ? pr / a.G : x.row0 / a.G, head = x.kvh * a.G + (ok ? pr - li * a.G : 0);
      const int pos = x.len - x.n + li;
      // ---- Q to shared memory: this thread's row (alternating: group 1 writes half of it)
      float rmul = 1.f;
      {
        const T* src = static_cast<const T*>(a.q) + (size_t)(x.first + li) * a.ldq + (size_t)head * HD;
        uint8_t* dst = sm + (F32 || x.alt ? 0 : t * C::BYTES) + row * 128;
        constexpr int CH = HD / 8;  // chunks of 8 dims
        int c0 = 0, c1 = CH;
        if constexpr (F32) {
          uint32_t top = 0;
#pragma unroll 8
          for (int c = 0; c < HD / 4; ++c) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(src) + c);
            top = max(max(top, __float_as_uint(f.x) & 0x7fffffffu), __float_as_uint(f.y) & 0x7fffffffu);
            top = max(max(top, __float_as_uint(f.z) & 0x7fffffffu), __float_as_uint(f.w) & 0x7fffffffu);
          }
          const int ex = min(112, max(-112, (int)(top >> 23) - 127));
          rmul = exp2i(ex - 13);
        }
        if (x.alt) {
          c0 = t * (CH / 2);
          c1 = c0 + CH / 2;
        }
        const float up = F32 ? __int_as_float((254 << 23) - __float_as_int(rmul)) : 1.f;  // 1 / rmul
#pragma unroll 4
        for (int c = c0; c < c1; ++c) {
          float q[8];
          if constexpr (F32) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(src) + 2 * c), g = __ldg(reinterpret_cast<const float4*>(src) + 2 * c + 1);
            q[0] = f.x * up; q[1] = f.y * up; q[2] = f.z * up; q[3] = f.w * up;
            q[4] = g.x * up; q[5] = g.y * up; q[6] = g.z * up; q[7] = g.w * up;
          } else {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(src) + c);
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = __half22float2(bits_half2(ws[i]));
              q[2 * i] = f.x;
              q[2 * i + 1] = f.y;
            }
          }
          if (!ok) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = 0.f;
          }
          constexpr int ord[8] = {0, BITS == 4 ? 4 : 1, BITS == 4 ? 1 : 2, BITS == 4 ? 5 : 3,
                                  BITS == 4 ? 2 : 4, BITS == 4 ? 6 : 5, BITS == 4 ? 3 : 6, 7};
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) hi[i] = split_h2(q[ord[2 * i]], q[ord[2 * i + 1]], lo[i]);
          uint8_t* at = dst + (c >> 3) * CK_TILE + (((c & 7) ^ (row & 7)) << 4);
          *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          if constexpr (F32) *reinterpret_cast<uint4*>(at + C::BYTES) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) ck_arrive(&q_full);
      }
      const float slope = a.slopes && ok ? __ldg(a.slopes + head) * KVQ_LOG2E : 0.f;
      // keys that every row of the block sees; this row's own limits
      const int p_lo = x.len - x.n + x.row0 / a.G, p_hi = x.len - x.n + (x.row0 + x.rows - 1) / a.G;
      const int in_lo = a.window ? p_hi - a.window + 1 : 0, in_hi = min(p_lo + 1, x.len) - CK_KEYS, in_pre = x.pre - CK_KEYS;
      const int r_lo = a.window ? pos - a.window + 1 : 0, r_hi = min(pos, x.len - 1);  // sees r_lo .. r_hi and 0 .. pre - 1
      // m: the largest score plus V scale's size when the reference last moved
      float m = -INFINITY, l = 0.f, ref = 0.f;
      // fp32 rows: the sum of earlier O tiles, relative to 2^sum_ref (-inf:
      // nothing seen yet); behind the parts (a slot holds 128 of its 256 rows)
      static_assert(!F32 || (size_t)2 * KVQ_CHUNK_CTAS * BM * (2 * HD + 2) <= KVQ_WS_CHUNK, "parts and sums");
      float sum_ref = -INFINITY;
      bool summed = false;
      auto against = [](float r, float top) { return r == -INFINITY ? 0.f : ex2(r - top); };
      float4* sum_at = reinterpret_cast<float4*>(a.ws + (size_t)2 * KVQ_CHUNK_CTAS * BM * (HD + 2)) +
                       (size_t)(2 * blockIdx.x + t) * 128 * (HD / 4) + row;
      auto add_sum = [&](int c, float (&o)[32], float fo, float fs) {  // columns 32 c .. of O and of the sum
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 z = __ldcg(sum_at + (8 * c + i) * 128);
          o[4 * i] = fmaf(z.x, fs, o[4 * i] * fo); o[4 * i + 1] = fmaf(z.y, fs, o[4 * i + 1] * fo);
          o[4 * i + 2] = fmaf(z.z, fs, o[4 * i + 2] * fo); o[4 * i + 3] = fmaf(z.w, fs, o[4 * i + 3] * fo);
        }
      };
      const int J = x.alt ? nt : 2 * nt;
#pragma unroll 1
      for (int j = t; j < J && !dead; j += 2) {
        const int kt = x.alt ? j : j >> 1, j0 = x.key(x.lo + kt);
        const unsigned f = fill + kt;
        const int st = f & 1;
        dead = !wait(&v_full[st], f >> 1) || !wait(&s_full[t], ns++);
        if (dead) break;
        ck_fence_after();
        const float4* ksc = reinterpret_cast<const float4*>(scale_s + st * 384);
        const float4 *vsc = ksc + 32, *size4 = ksc + 64;
        const bool inner = (j0 >= in_lo && j0 <= in_hi) || j0 <= in_pre;
        // x of columns GC c .. GC c + GC - 1; where the common tile has its own
        // code this one is kept small
        constexpr int GC = PLAIN && !F32 ? 8 : 32;  // (fp32 rows' low parts go to columns that have to be read first)
        auto scores = [&](int c, float (&z)[GC]) {
          ck_get<GC>(s_tm + GC * c, z);
#pragma unroll
          for (int i = 0; i < GC / 4; ++i) {
            const float4 k4 = ksc[GC / 4 * c + i];
            const float k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) z[4 * i + e] *= F32 ? k[e] * rmul : k[e];
          }
          if (!PLAIN && a.cap > 0.f) {
#pragma unroll
            for (int i = 0; i < GC; ++i) z[i] = a.cap * KVQ_LOG2E * (F32 ? tanh_f32(z[i]) : tanh_fast(z[i]));
          }
          if (!PLAIN && a.slopes) {
#pragma unroll
            for (int i = 0; i < GC; ++i) z[i] = fmaf(-slope, fabsf((float)(pos - (j0 + GC * c + i))), z[i]);
          }
          if (!inner) {
#pragma unroll
            for (int i = 0; i < GC; ++i) {
              const int k = j0 + GC * c + i;
              if (!((k >= r_lo && k <= r_hi) || k < x.pre)) z[i] = -INFINITY;
            }
          }
        };
        // Does the reference hold? The common tile (no cap, no bias, nothing
        // masked) asks a bound first, the largest raw product of 32 keys times
        // their largest K scale, plus their largest V scale's size, which needs
        // no key's own scales.
        const bool fast = PLAIN && inner;
        float mx = m;
        const float hold = m + CkLift<F32>::MARGIN;
        if (fast) {
          float z[2][32];
          ck_ld32(s_tm, z[0]);
#pragma unroll 1
          for (int c2 = 0; c2 < 4; c2 += 2)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int c = c2 + h;
            ck_wait_ld(z[h]);
            if (c < 3) ck_ld32(s_tm + 32 * (c + 1), z[h ^ 1]);
            float(&w)[32] = z[h];
            float top[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              top[0] = fmaxf(top[0], fmaxf(w[i], w[i + 1]));
              top[1] = fmaxf(top[1], fmaxf(w[i + 2], w[i + 3]));
            }
            const float2 most = most_s[st][c];
            if (__any_sync(0xffffffffu, !(fmaf(fmaxf(top[0], top[1]), most.x * rmul, most.y) <= hold))) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 k4 = ksc[8 * c + i], z4 = size4[8 * c + i];
                const float e0 = fmaxf(fmaf(w[4 * i] * rmul, k4.x, z4.x), fmaf(w[4 * i + 1] * rmul, k4.y, z4.y));
                const float e1 = fmaxf(fmaf(w[4 * i + 2] * rmul, k4.z, z4.z), fmaf(w[4 * i + 3] * rmul, k4.w, z4.w));
                mx = fmaxf(mx, fmaxf(e0, e1));
              }
            }
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < 128 / GC; ++c) {
            float z[GC];
            scores(c, z);
#pragma unroll
            for (int i = 0; i < GC / 4; ++i) {
              const float4 z4 = size4[GC / 4 * c + i];
              mx = fmaxf(mx, fmaxf(fmaxf(z[4 * i] + z4.x, z[4 * i + 1] + z4.y), fmaxf(z[4 * i + 2] + z4.z, z[4 * i + 3] + z4.w)));
            }
            if constexpr (GC == 32) ck_st32(s_tm + GC * c, z);  // tanh, bias and mask once only
          }
          if constexpr (GC == 32) ck_wait_st();
        }
        if (F32 && j >= 2 && (j >> 1) % CK_SUM == 0) {  // (the products of O's tiles are done, as below)
          const float own = m == -INFINITY ? m : ref, top = fmaxf(sum_ref, own), fo = against(own, top), fs = against(sum_ref, top);
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            float o[32];
            ck_get32(o_tm + 32 * c, o);
            if (summed) add_sum(c, o, fo, fs);  // (else fo is 1, or O is 0)
#pragma unroll
            for (int i = 0; i < 8; ++i) __stcg(sum_at + (8 * c + i) * 128, make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
          }
          sum_ref = top;
          summed = true;
        }
        if (__any_sync(0xffffffffu, mx > hold)) {
          const float rn = (mx == -INFINITY ? 0.f : mx) - CkLift<F32>::LIFT;
          const float fac = m == -INFINITY ? 0.f : ex2(ref - rn);
          m = mx;
          ref = rn;
          l *= fac;
          // O holds this group's earlier tiles (their products are done: S of this tile came after them)
          if (F32 ? (j >> 1) % CK_SUM != 0 : j >= 2) {
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
              float o[32];
              ck_get32(o_tm + 32 * c, o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= fac;
              ck_st32(o_tm + 32 * c, o);
            }
          }
        }
        if (fast) {
          const float2 nref = make_float2(-ref, -ref);
          float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};  // of this tile: small weights would be lost beside the whole
          auto weigh = [&](int q, const float* w, float2& u0, float2& u1) {  // keys 4 q .. + 3
            const float4 k4 = ksc[q], v4 = vsc[q];
            u0 = make_float2(w[0], w[1]);
            u1 = make_float2(w[2], w[3]);
            if constexpr (F32) {
              u0 = mul2(u0, make_float2(rmul, rmul));
              u1 = mul2(u1, make_float2(rmul, rmul));
            }
            u0 = fma2(u0, make_float2(k4.x, k4.y), nref);
            u1 = fma2(u1, make_float2(k4.z, k4.w), nref);
            u0.x = ex2(u0.x); u0.y = ex2(u0.y); u1.x = ex2(u1.x); u1.y = ex2(u1.y);
            l2[0] = add2(l2[0], u0);
            l2[1] = add2(l2[1], u1);
            u0 = mul2(u0, make_float2(v4.x, v4.y));
            u1 = mul2(u1, make_float2(v4.z, v4.w));
          };
          if constexpr (F32) {
            // 16 keys at a time: two parts of 32 spill (461 us where this takes 424)
            float za[16], zb[16];
            uint32_t ph[8], pa[8], pb[8];
            auto parts = [&](int c, const float (&z)[16], uint32_t (&lo)[8]) {  // keys 16 c ..
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float2 u0, u1;
                weigh(4 * c + i, z + 4 * i, u0, u1);
                ph[2 * i] = split_h2(u0.x, u0.y, lo[2 * i]);
                ph[2 * i + 1] = split_h2(u1.x, u1.y, lo[2 * i + 1]);
              }
            };
            ck_ld16(s_tm, za);
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              ck_wait_ld(za);
              ck_ld16(s_tm + 32 * c + 16, zb);
              parts(2 * c, za, pa);
              ck_st8(s_tm + 32 * c, ph);
              ck_wait_ld(zb);
              if (c < 3) ck_ld16(s_tm + 32 * (c + 1), za);
              ck_st8(s_tm + 32 * c + 16, pa);  // over scores that are in registers now
              parts(2 * c + 1, zb, pb);
              ck_st8(s_tm + 32 * c + 8, ph);
              ck_st8(s_tm + 32 * c + 24, pb);
            }
          } else {
            float z[2][32];
            ck_ld32(s_tm, z[0]);
#pragma unroll 1
            for (int c2 = 0; c2 < 4; c2 += 2)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c = c2 + h;
              ck_wait_ld(z[h]);
              if (c < 3) ck_ld32(s_tm + 32 * (c + 1), z[h ^ 1]);
              uint32_t ph[16];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float2 u0, u1;
                weigh(8 * c + i, z[h] + 4 * i, u0, u1);
                ph[2 * i] = half2_bits(__floats2half2_rn(u0.x, u0.y));
                ph[2 * i + 1] = half2_bits(__floats2half2_rn(u1.x, u1.y));
              }
              ck_st16(s_tm + 32 * c, ph);
            }
          }
          l += (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
        } else {
          float lt = 0.f;
#pragma unroll 1
          for (int c = 0; c < 128 / GC; ++c) {
            float z[GC];
            if constexpr (GC == 32) ck_get32(s_tm + GC * c, z);
            else scores(c, z);
            uint32_t ph[GC / 2], pl[F32 ? GC / 2 : 1];
#pragma unroll
            for (int i = 0; i < GC / 4; ++i) {
              const float4 v4 = vsc[GC / 4 * c + i];
              const float vs[4] = {v4.x, v4.y, v4.z, v4.w};
              float p[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float y = ex2(z[4 * i + e] - ref);
                lt += y;
                p[e] = z[4 * i + e] == -INFINITY ? 0.f : y * vs[e];  // a masked key counts for nothing, whatever its scale holds
              }
              if constexpr (F32) {
                ph[2 * i] = split_h2(p[0], p[1], pl[2 * i]);
                ph[2 * i + 1] = split_h2(p[2], p[3], pl[2 * i + 1]);
              } else {
                ph[2 * i] = half2_bits(__floats2half2_rn(p[0], p[1]));
                ph[2 * i + 1] = half2_bits(__floats2half2_rn(p[2], p[3]));
              }
            }
            // keys 32 k ..: 16 columns of pairs at 32 k (and 16 of low parts).
            // GC = 8 overwrites columns 32 k + 4 r ..: of chunk r = 0 the first
            // four of its own, later ones columns that were read before.
            const uint32_t to = s_tm + (GC * c & ~31) + (GC * c & 31) / 2;
            ck_put<GC / 2>(to, ph);
            if constexpr (F32) ck_put<GC / 2>(to + 16, pl);
          }
          l += lt;
        }
        ck_wait_st();
        ck_fence_before();
        __syncwarp();
        if (lane == 0) ck_arrive(&p_full[t]);
      }
      fill += nt;

      // ---- the segment's end: O from tensor memory
      const bool mine = J > t;  // this group had a tile
      bool have = !dead;
      if (mine && have) {
        have = wait(&o_full[t], no);
        ck_fence_after();
      }
      if (mine) ++no;
      dead |= !have;
      // O of the whole segment, relative to 2^ref, columns 32 c ..
      const float own = m == -INFINITY ? m : ref, whole_ref = fmaxf(sum_ref, own);
      const float end_o = against(own, whole_ref), end_s = against(sum_ref, whole_ref);
      auto get_o = [&](int c, float (&o)[32]) {
        ck_get32(o_tm + 32 * c, o);
        if (F32 && summed) add_sum(c, o, end_o, end_s);
      };
      if (F32 && summed) {
        l *= end_o;
        ref = whole_ref;
      }
      float* merge = reinterpret_cast<float*>(sm);  // the Q tiles are free: [128 rows][HD] floats, 16-byte chunks swizzled
      auto at = [&](int r, int c4) { return reinterpret_cast<float4*>(merge + r * HD) + (c4 ^ (r & (HD / 4 - 1))); };
      float f1 = 1.f;  // this group's weight (alternating: against the other's)
      if (x.alt) {
        // group 1 hands its state to group 0
        if (t == 1) {
          l_s[row] = dead ? -1.f : mine ? l : 0.f;
          if (mine && have) {
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
              float o[32];
              get_o(c, o);
#pragma unroll
              for (int i = 0; i < 8; ++i) *at(row, 8 * c + i) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
          }
          // the reference exponent stands in for the maximum: l and O are relative to it
          m_s[row] = mine && m != -INFINITY ? ref : -INFINITY;
        }
        pair_bar();
      }
      const bool split = x.hi - x.lo < x.total;
      const int cb = whole ? 0 : (u - x.lo) / share, ce = whole ? 0 : (u - x.lo + x.total - 1) / share;
      auto slot_of = [&](int p) { return 2 * (cb + p) + (p == 0 ? 1 : 0); };
      const size_t part = (size_t)BM * (HD + 2);
      float* my_part = a.ws + slot_of(blockIdx.x - cb) * part;
      // dims of output column 8 c + k (int4 codes unpack in another order)
      auto put = [&](int packed, int c, const float (&o)[32], float inv) {  // columns 32 c .. + 31 of a packed row
        const int i = packed / a.G;
        T* dst = static_cast<T*>(a.out) + (size_t)(x.first + i) * a.ldo + (size_t)(x.kvh * a.G + packed - i * a.G) * HD + 32 * c;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int b = 8 * (k >> 1);
          if constexpr (BITS == 4) {
            // dim d of a group of 8 sits at column 2 (d & 3) + (d >> 2)
            const int h = k & 1;
            kvq_store4(dst + 4 * k, o[b + h] * inv, o[b + 2 + h] * inv, o[b + 4 + h] * inv, o[b + 6 + h] * inv);
          } else {
            kvq_store4(dst + 4 * k, o[4 * k] * inv, o[4 * k + 1] * inv, o[4 * k + 2] * inv, o[4 * k + 3] * inv);
          }
        }
      };
      if (!(x.alt && t == 1)) {
        float R = m == -INFINITY ? -INFINITY : ref, f2 = 0.f, L = l;
        bool gone = dead;  // this row's state is not whole
        if (x.alt) {
          gone |= l_s[row] < 0.f;
          const float r1 = m_s[row], M = fmaxf(R, r1);
          f1 = R == -INFINITY ? 0.f : ex2(R - M);
          f2 = r1 == -INFINITY ? 0.f : ex2(r1 - M);
          // a NaN sum stays one, whatever its weight
          L = (l == l ? l * f1 : l) + (l_s[row] == l_s[row] ? l_s[row] * f2 : l_s[row]);
          R = M;
        }
        const bool other = x.alt && J > 1;
        const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          float o[32];
          get_o(c, o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= f1;
          if (other) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 z = *at(row, 8 * c + i);
              o[4 * i] = fmaf(z.x, f2, o[4 * i]); o[4 * i + 1] = fmaf(z.y, f2, o[4 * i + 1]);
              o[4 * i + 2] = fmaf(z.z, f2, o[4 * i + 2]); o[4 * i + 3] = fmaf(z.w, f2, o[4 * i + 3]);
            }
          }
          if (L == 0.f) {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.f;
          }
          if (ok && !gone) {
            if (split) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                __stcg(reinterpret_cast<float4*>(my_part) + (8 * c + i) * BM + pr - x.row0,
                       make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
            } else {
              put(pr, c, o, inv);
            }
          }
        }
        // (a sum below 0: the part is not there, and the row stays unwritten)
        if (split && ok)
          __stcg(reinterpret_cast<float2*>(my_part + (size_t)BM * HD) + (pr - x.row0), make_float2(R, gone ? -1.f : L));
      }
      ck_fence_before();
      pair_bar();  // Q tiles, merge buffer and O are free for the next segment
      if (split) {
        if (tid == 0) {
          __threadfence();
          last_s = atomicAdd(a.tickets + slot_of(0), 1) == ce - cb;
          if (last_s) {
            __threadfence();
            a.tickets[slot_of(0)] = 0;
          }
        }
        pair_bar();
        if (last_s) {
          // The parts' weights of each row first (the Q tiles are free), then
          // 8 dims of two rows per thread and pass, the parts in order; eight
          // lanes hold neighbouring rows, four neighbouring dims.
          constexpr int WT = C::Q_BYTES / (4 * 256) - 2;  // parts whose weights fit; those of further ones are found anew
          const int np = ce - cb + 1;
          float2* stat = reinterpret_cast<float2*>(sm);
          float* wt = reinterpret_cast<float*>(stat + 256);  // [part][256 rows]
          auto stat_of = [&](int p) { return reinterpret_cast<const float2*>(a.ws + slot_of(p) * part + (size_t)BM * HD); };
          auto weight = [](float2 rl, float M) { return rl.x == -INFINITY ? (rl.y == rl.y ? 0.f : rl.y) : ex2(rl.x - M); };
          if (tid < x.rows) {
            float M = -INFINITY, L = 0.f;
            bool gone = false;
#pragma unroll 4
            for (int p = 0; p < np; ++p) M = fmaxf(M, __ldcg(stat_of(p) + tid).x);
#pragma unroll 4
            for (int p = 0; p < np; ++p) {
              const float2 rl = __ldcg(stat_of(p) + tid);
              const float w = weight(rl, M);
              L += rl.y * w;
              gone |= rl.y < 0.f;
              if (p < WT) wt[p * 256 + tid] = w;
            }
            stat[tid] = make_float2(M, gone ? -1.f : L);
          }
          pair_bar();
          constexpr int K = 2, GROUPS = HD / 32;
          const int octets = (x.rows + 7) / 8;  // items: (octet of rows, group of 32 dims, lane)
          for (int i0 = tid; i0 < octets * GROUPS * 32; i0 += 256 * K) {
            int r[K], d8[K];
            bool there[K];
            float4 y[K][2];
#pragma unroll
            for (int k = 0; k < K; ++k) {
              const int i = (i0 + 256 * k) >> 5, o = i / GROUPS;
              r[k] = o * 8 + (lane & 7);
              d8[k] = 4 * (i - o * GROUPS) + (lane >> 3);
              there[k] = r[k] < x.rows;
              if (!there[k]) r[k] = 0;
              y[k][0] = y[k][1] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll 2
            for (int p = 0; p < np; ++p) {
              const float4* at_p = reinterpret_cast<const float4*>(a.ws + slot_of(p) * part);
#pragma unroll
              for (int k = 0; k < K; ++k) {
                const float w = p < WT ? wt[p * 256 + r[k]] : weight(__ldcg(stat_of(p) + r[k]), stat[r[k]].x);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const float4 z = __ldcg(at_p + (2 * d8[k] + h) * BM + r[k]);
                  y[k][h].x = fmaf(z.x, w, y[k][h].x); y[k][h].y = fmaf(z.y, w, y[k][h].y);
                  y[k][h].z = fmaf(z.z, w, y[k][h].z); y[k][h].w = fmaf(z.w, w, y[k][h].w);
                }
              }
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
              if (!there[k] || stat[r[k]].y < 0.f) continue;
              const float L = stat[r[k]].y, inv = L == 0.f ? 0.f : 1.0f / L;
              const bool none = L == 0.f;
              float o[8] = {y[k][0].x, y[k][0].y, y[k][0].z, y[k][0].w, y[k][1].x, y[k][1].y, y[k][1].z, y[k][1].w};
#pragma unroll
              for (int e = 0; e < 8; ++e) o[e] = none ? 0.f : o[e] * inv;
              const int packed = x.row0 + r[k], li2 = packed / a.G;
              T* dst = static_cast<T*>(a.out) + (size_t)(x.first + li2) * a.ldo + (size_t)(x.kvh * a.G + packed - li2 * a.G) * HD + 8 * d8[k];
              if constexpr (BITS == 4) {  // dim d of a group of 8 sits at column 2 (d & 3) + (d >> 2)
                kvq_store4(dst, o[0], o[2], o[4], o[6]);
                kvq_store4(dst + 4, o[1], o[3], o[5], o[7]);
              } else {
                kvq_store4(dst, o[0], o[1], o[2], o[3]);
                kvq_store4(dst + 4, o[4], o[5], o[6], o[7]);
              }
            }
          }
        }
        pair_bar();
      }
      u = un;
    }
  }
  ck_fence_before();
  __syncthreads();
  if (warp == CK_MMA) {
    if (lane == 0) mbar_wait_bounded(&idle, 0u, MBAR_SPIN_LIMIT);  // no MMA may still write the memory that is freed
    __syncwarp();
    ck_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  // the call's decode kernel, if any, has ended too when this one ends
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace

template <int HD, int BITS, typename T>
int kvq_chunk_launch(AttendArgs a, bool beside, cudaStream_t s) {
  using C = CkCfg<HD>;
  auto kern = a.cap > 0.f || a.slopes ? kvq_chunk_kernel<HD, BITS, T, false> : kvq_chunk_kernel<HD, BITS, T, true>;
  const int rc = set_smem_limit((const void*)kern, C::SMEM + KVQ_MAX_SEQ * 4, "kvq_chunk");
  if (rc) return rc;
  // Beside a decode kernel: it lets this one start as its CTAs leave, and this
  // one's end waits for it. Nothing passes between the two (workspaces and
  // outputs are apart), and what came before it ended before it began.
  // 317 rows of 17 sequences, one of them for this kernel: 82 us, 88 in turn.
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(min(sm_count(), KVQ_CHUNK_CTAS));
  cfg.blockDim = dim3(CK_THREADS);
  cfg.dynamicSmemBytes = C::SMEM + (size_t)a.v.n_seq * 4;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = beside ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("kvq_chunk launch: %s", cudaGetErrorString(e));
    return LUMINA_E_CUDA;
  }
  return LUMINA_OK;
}
template int kvq_chunk_launch<128, 8, __half>(AttendArgs, bool, cudaStream_t);
template int kvq_chunk_launch<128, 8, float>(AttendArgs, bool, cudaStream_t);
template int kvq_chunk_launch<128, 4, __half>(AttendArgs, bool, cudaStream_t);
template int kvq_chunk_launch<128, 4, float>(AttendArgs, bool, cudaStream_t);
template int kvq_chunk_launch<64, 8, __half>(AttendArgs, bool, cudaStream_t);
template int kvq_chunk_launch<64, 8, float>(AttendArgs, bool, cudaStream_t);
template int kvq_chunk_launch<64, 4, __half>(AttendArgs, bool, cudaStream_t);
template int kvq_chunk_launch<64, 4, float>(AttendArgs, bool, cudaStream_t);

}  // namespace lumina
