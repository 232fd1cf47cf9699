// What the attention kernels over quantized KV pages share: arguments and
// the launches that lumina_kvq_attend chooses from.
#pragma once
#include <type_traits>

#include "kvq.cuh"

namespace lumina {

constexpr int KVQ_MAX_CTAS = 512;    // CTAs that may leave partial states (two each)
constexpr int KVQ_FAN = 64;          // partial states that one CTA joins at a time
constexpr int KVQ_DECODE_ROWS = 16;  // packed rows of a decode task at most
constexpr int KVQ_DECODE_BLOCKS = 4;  // times so many: a sequence's packed rows for the decode kernel at most (fp32 rows)

struct AttendArgs {
  KvqView v;
  const void* q;
  void* out;
  size_t ldq, ldo;
  int nh, G;
  float scale, cap;
  const float* slopes;
  const int* prefix;
  int window;
  int few;        // sequences of up to this many packed rows (rows x G) are the decode kernel's
  float* ws;      // partial states
  int* tickets;   // two per partial state, zero between launches
  long long spin;
};

// sequences of up to a.few packed rows, in blocks of up to `rows` (8 or 16; kvq_decode.cu)
template <int HD, int BITS, typename T>
int kvq_decode_launch(AttendArgs a, int rows, cudaStream_t s);

// sequences of more than a.few packed rows (kvq_chunk.cu). beside: the decode
// kernel was launched just before, and this one may start while it runs
template <int HD, int BITS, typename T>
int kvq_chunk_launch(AttendArgs a, bool beside, cudaStream_t s);

constexpr int KVQ_MAX_BLOCKS = 2048;  // row blocks whose key tiles the chunk kernel lines up
constexpr int KVQ_CHUNK_CTAS = 160;   // CTAs of the chunk kernel at most
constexpr int KVQ_CHUNK_ROWS = 256;   // packed rows of its partial states

// workspace: tickets, then partial states (and the chunk kernel's sums of fp32
// rows); the two kernels of a mixed batch overlap, so each has its own of both
constexpr size_t KVQ_WS_DECODE_TICKETS = 4 * KVQ_MAX_CTAS, KVQ_WS_CHUNK_TICKETS = 2 * KVQ_CHUNK_CTAS;
constexpr size_t KVQ_WS_TICKETS = (KVQ_WS_DECODE_TICKETS + KVQ_WS_CHUNK_TICKETS) * sizeof(int);
constexpr size_t KVQ_WS_DECODE = (size_t)KVQ_MAX_CTAS * 2 * KVQ_DECODE_ROWS * (128 + 2);  // floats
constexpr size_t KVQ_WS_CHUNK = (size_t)KVQ_CHUNK_CTAS * 2 * KVQ_CHUNK_ROWS * (128 + 2);
constexpr size_t kvq_ws_bytes() { return KVQ_WS_TICKETS + (KVQ_WS_DECODE + KVQ_WS_CHUNK) * sizeof(float); }
static_assert(KVQ_WS_TICKETS % 16 == 0 && KVQ_WS_DECODE % 4 == 0, "16-byte aligned partial states");

// rows of sequence s as the batch says (0 where row_start is out of order)
__device__ __forceinline__ int kvq_seq_rows(const KvqView& v, int s, int& first, bool report = true) {
  first = __ldg(v.row_start + s);
  const int end = __ldg(v.row_start + s + 1);
  if (first < 0 || end < first || end > v.n_rows || end - first > v.max_rows) {
    if (report) kvq_fault(v, KVQ_FAULT_DATA);
    return 0;
  }
  return end - first;
}

__device__ __forceinline__ void kvq_store4(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
__device__ __forceinline__ void kvq_store4(__half* p, float a, float b, float c, float d) {
  const __half2 x = __floats2half2_rn(a, b), y = __floats2half2_rn(c, d);
  *reinterpret_cast<uint2*>(p) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// a + b for the prefix sums of the work lines, no further than KVQ_MANY (which
// a + b of two such sums does not pass 32 bits for, and no line may reach)
constexpr unsigned KVQ_MANY = 0x40000000u;
__device__ __forceinline__ unsigned kvq_sum(unsigned a, unsigned b) { return min(a + b, KVQ_MANY); }

// f(integral_constant<int, 0>), ..., f(integral_constant<int, N - 1>)
template <int N, int I = 0, typename Fn>
__device__ __forceinline__ void static_for(Fn&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    static_for<N, I + 1>(f);
  }
}

}  // namespace lumina
