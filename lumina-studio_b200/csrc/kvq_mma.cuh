// Pieces of the attention over quantized KV pages: codes to fragments of
// mma.sync m16n8k16 (the decode kernel) and to fp16 numbers, the exponential
// and tanh, and the sizes of V scales (both kernels).
//
// The decode kernel's products are transposed, S^T = K Q^T and O^T = V^T P^T:
// 16 keys (dims) fill a fragment's rows, up to 8 packed query rows (row r =
// local row r / G, head r % G of one KV head's G query heads) its columns.
// Codes are small integers, exact in fp16, so K and V enter the tensor pipe as
// they are stored and the scales stay outside the products: a key's K scale
// multiplies its scores, its V scale its probabilities.
//
// Fragment layouts (lane = 4 g + t): a thread's four k-indices of a step may
// be any four dims of key g as long as q uses the same, so thread t owns runs
// of the key's codes that load as 16-byte words (load_q takes q's dims in that
// order). In V^T, row g of 8-dim tile i is dim g * HD / 8 + i, so a thread
// loads one contiguous run per key and ends with HD / 8 contiguous dims of its
// two output columns.
#pragma once
#include "kvq.cuh"

namespace lumina {

constexpr float KVQ_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh by 1 - 2 / (1 + e^2x): absolute error near 2^-23
__device__ __forceinline__ float tanh_fast(float x) {
  return fmaf(-2.f, rcp_approx(1.f + ex2(2.f * KVQ_LOG2E * x)), 1.f);
}
// tanh to about 2 ulp without a branch: its Taylor polynomial below 0.35,
// (1 - e^-2|x|) / (1 + e^-2|x|) above
__device__ __forceinline__ float tanh_f32(float x) {
  const float s = x * x, t = ex2(-2.f * KVQ_LOG2E * fabsf(x));
  float c = fmaf(s, -1382.f / 155925.f, 62.f / 2835.f);
  c = fmaf(s, c, -17.f / 315.f);
  c = fmaf(s, c, 2.f / 15.f);
  c = fmaf(s, c, -1.f / 3.f);
  const float far = copysignf((1.f - t) * rcp_approx(1.f + t), x);
  return fabsf(x) < 0.35f ? fmaf(x * s, c, x) : far;
}
// 8 x 8 fp16 tile: (row g, columns 2t, 2t + 1) per lane -> (column g, rows 2t, 2t + 1)
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// 2^e as a float, e in [-126, 127]
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }

// A V scale's size as attention's references count it: the e with |s| < 2^e,
// -90 at least (a NaN too), so that 2^(15 - e) times any number of keys stays
// within fp32. (Keys whose V scales are 2^126 apart may lose each other's
// weights.)
__device__ __forceinline__ float kvq_size(float s) {
  const uint32_t b = __float_as_uint(s) & 0x7fffffffu;
  return (float)(b > 0x7f800000u ? -90 : max(-90, (int)(b >> 23) - 126));
}

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_half2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
// (a, b) -> fp16 pair, and the fp16 pair of what it leaves
__device__ __forceinline__ uint32_t split_h2(float a, float b, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  lo = half2_bits(__floats2half2_rn(a - __low2float(h), b - __high2float(h)));
  return half2_bits(h);
}

// Codes to fp16 through the fp16 number 1024 + u: its low mantissa bits are u.
constexpr uint32_t H_1024 = 0x64006400u;
// signed bytes with the sign bit flipped (u = c + 128): two of them -> (c0, c1)
template <int SEL>
__device__ __forceinline__ uint32_t s8_pair(uint32_t flipped) {
  const __half2 v = bits_half2(__byte_perm(flipped, 0x64646464u, SEL));
  return half2_bits(__hsub2(v, __floats2half2_rn(1152.f, 1152.f)));
}
// nibbles at bits 4-7 of each 16-bit half -> 2 c - 15 = (1024 + 16 c) / 8 - 143
// (at bits 0-3 the subtrahend, 2063, would not be an fp16 number)
__device__ __forceinline__ uint32_t u4_pair(uint32_t w) {
  return half2_bits(__hfma2(bits_half2((w & 0x00F000F0u) | H_1024), __floats2half2_rn(0.125f, 0.125f),
                            __floats2half2_rn(-143.f, -143.f)));
}

template <int HD, int BITS>
struct KvqFrag {
  static constexpr int NB = HD * BITS / 8;  // code bytes of one key
  static constexpr int KK = HD / 16;        // MMA steps of q . k
  static constexpr int KW = NB / 16;        // 32-bit words of K codes per thread and key
  static constexpr int NT = HD / 8;         // n-tiles of p . v = dims per thread and key
  static constexpr int VW = NT * BITS / 32; // 32-bit words of V codes per thread and key

  // q[kk][e] of a row from its head_dim values at src (16-byte aligned): the
  // thread's runs of consecutive dims by 16-byte loads
  template <typename T>
  __device__ static __forceinline__ void load_q(const T* src, int t, float (&q)[KK][4]) {
    constexpr int RUN = BITS == 8 ? 16 : HD / 4, V = 16 / sizeof(T);
#pragma unroll
    for (int u = 0; u < KK * 4 / RUN; ++u) {
      float x[RUN];
#pragma unroll
      for (int i = 0; i < RUN / V; ++i) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(src + (u * 4 + t) * RUN) + i);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(T) == 4) {
            x[4 * i + e] = __uint_as_float(ws[e]);
          } else {
            const float2 f = __half22float2(bits_half2(ws[e]));
            x[8 * i + 2 * e] = f.x;
            x[8 * i + 2 * e + 1] = f.y;
          }
        }
      }
#pragma unroll
      for (int kk = 0; kk < RUN / 4; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          q[u * (RUN / 4) + kk][e] = x[BITS == 8 ? kk * 4 + e : (kk >> 1) * 8 + 2 * (kk & 1) + (e >> 1) + 4 * (e & 1)];
    }
  }
  // where a thread's code words of a key row start, and the words themselves
  __device__ static __forceinline__ int k_lane(int t) { return t * (KW >= 4 ? 16 : 8); }
  __device__ static __forceinline__ int v_lane(int g) { return g * VW * 4; }
  __device__ static __forceinline__ void load_k(const uint8_t* p, uint32_t (&w)[KW]) {
    if constexpr (KW >= 4) {
#pragma unroll
      for (int i = 0; i < KW / 4; ++i) {
        const uint4 q = ldg_stream(p + i * 64);
        w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
      }
    } else {
      const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = q.x; w[1] = q.y;
    }
  }
  // fragment of step kk: k-indices e = 0, 1 in b0 and 2, 3 in b1, the codes'
  // values c (int8) or 2 c - 15 (int4). RAW: unsigned codes at the bottom of
  // an fp16 mantissa, that is the subnormal code * 2^-24 (exact on the tensor
  // pipe), the second of each pair complemented: u = c + 128 and 255 - u
  // (int8; e = 0, 2 in b0 and 1, 3 in b1); c and 15 - c, in b1 times 16 (int4).
  // With q negated for the complemented ones, sum q (u - zero) = sum +-q u' -
  // sum +-q w, w = RAW_ZERO of the place in the pair, and both sums stay small
  // also where the q have a common offset.
  template <int kk, bool RAW = false>
  __device__ static __forceinline__ void k_frag(const uint32_t (&w)[KW], uint32_t& b0, uint32_t& b1) {
    if constexpr (BITS == 8 && RAW) {
      const uint32_t x = w[kk] ^ 0x7F7F8080u;
      b0 = x & 0x00FF00FFu;
      b1 = __byte_perm(x, 0u, 0x4341);  // bytes 1 and 3 (a shift and a mask: 93 us, 88 so, with 64 sequences of up to 8192)
    } else if constexpr (BITS == 8) {
      const uint32_t f = w[kk] ^ 0x80808080u;
      b0 = s8_pair<0x4140>(f);
      b1 = s8_pair<0x4342>(f);
    } else if constexpr (RAW) {
      const uint32_t v = (kk & 1) ? w[kk >> 1] >> 8 : w[kk >> 1];
      b0 = (v ^ 0x000F0000u) & 0x000F000Fu;
      b1 = (v ^ 0x00F00000u) & 0x00F000F0u;
    } else {
      const uint32_t v = w[kk >> 1];
      b0 = u4_pair((kk & 1) ? v >> 4 : v << 4);
      b1 = u4_pair((kk & 1) ? v >> 8 : v);
    }
  }
  __device__ static __forceinline__ void load_v(const uint8_t* p, uint32_t (&w)[VW]) {
    if constexpr (VW == 4) {
      const uint4 q = ldg_stream(p);
      w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    } else if constexpr (VW == 2) {
      const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = q.x; w[1] = q.y;
    } else {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    }
  }
  // fp16 pairs (key a, key b) of dims DPW * j + i of the thread's run, where
  // word j of each key holds DPW = 32 / BITS dims: c (int8) or 2 c - 15 (int4).
  // RAW (as in k_frag): the odd key's codes are complemented, to be met by a
  // negated p; for odd i int4 codes come times 16.
  static constexpr float RAW_ZERO[2] = {BITS == 8 ? 128.f : 7.5f, BITS == 8 ? 127.f : 7.5f};
  template <int i, bool RAW>
  __device__ static __forceinline__ uint32_t v_frag(uint32_t a, uint32_t b) {
    if constexpr (BITS == 8 && RAW) {
      const uint32_t x = __byte_perm(a, b, (i & 2) ? 0x7632 : 0x5410);  // a_i' a_i'+1 | b_i' b_i'+1
      return (((i & 1) ? x >> 8 : x) ^ 0x007F0080u) & 0x00FF00FFu;
    } else if constexpr (BITS == 8) {
      const uint32_t x = __byte_perm(a, b, (i & 2) ? 0x7362 : 0x5140);  // a_i' b_i' a_i'+1 b_i'+1
      return s8_pair<(i & 1) ? 0x4342 : 0x4140>(x ^ 0x80808080u);
    } else {
      const uint32_t x = __byte_perm(a, b, (i & 4) ? 0x7632 : 0x5410);
      if constexpr (RAW) return (((i & 2) ? x >> 8 : x) ^ 0xFFFF0000u) & ((i & 1) ? 0x00F000F0u : 0x000F000Fu);
      else return u4_pair((i & 3) == 0 ? x << 4 : x >> (4 * ((i & 3) - 1)));
    }
  }
};

}  // namespace lumina
