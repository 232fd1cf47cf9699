// Quantized KV pages of several sequences: what the append, read and attend
// kernels share (pool geometry, batch lookup, argument checks).
#pragma once
#include "weights.cuh"

namespace lumina {

constexpr int KVQ_MAX_SEQ = 4096;   // sequences of one batch
constexpr int KVQ_FAULT_WAIT = 32;  // fault word: a bounded wait gave up
constexpr int KVQ_FAULT_DATA = 64;  // fault word: row, length or page out of range

// A pool and a batch as the kernels take them.
struct KvqView {
  uint8_t* pool;
  size_t page_bytes;      // n_kv blocks
  uint32_t block_bytes;
  int n_pages, n_kv;
  int page_shift;         // log2(page_size)
  const int* row_start;
  const int* len;
  const int* pages;
  int pages_ld, n_seq, n_rows, max_rows;
  int* fault;
};

inline size_t kvq_block_bytes(int bits, int hd, int page) { return (size_t)page * (2 * (hd * bits / 8) + 8); }

// LUMINA_OK and the view, or the status of what is wrong with the arguments
// (the device of the pool must be current: fault word).
int kvq_view(const lumina_kvq_pool* pool, const lumina_kvq_batch* batch, const char* what, KvqView* v);
// rows of `ld` elements of `type` at p: 16-byte aligned, at least `width` wide
int kvq_check_rows(const void* p, long long ld, int width, int type, const char* what, const char* name);

class KvqDevice {
 public:
  explicit KvqDevice(int dev);
  ~KvqDevice();
  bool ok;

 private:
  int prev_ = -1, dev_;
};

__device__ __forceinline__ void kvq_fault(const KvqView& v, int bit) { atomicOr(v.fault, bit); }

// Sequence of batch row `row`: the last s with row_start[s] <= row, by a
// search 32 wide (one load per lane and level; a whole warp calls it).
// -1 when row_start does not hold it.
__device__ __forceinline__ int kvq_find_seq(const KvqView& v, int row, int lane) {
  int lo = 0, n = v.n_seq;
  while (true) {
    const int step = (n + 31) >> 5;
    const int at = lo + lane * step;
    const bool in = lane * step < n && __ldg(v.row_start + at) <= row;
    const unsigned m = __ballot_sync(0xffffffffu, in);
    if (m == 0) return -1;
    const int c = 31 - __clz(m);
    lo += c * step;
    n = min(step, n - c * step);
    if (step == 1) return lo;
  }
}

// A batch row's place in the cache. pos = -1: not stored (data out of range;
// the fault bit is set).
struct KvqRow {
  int pos;
  const uint8_t* page;  // its page (the block of KV head 0)
  int off;              // token within the page
};
__device__ __forceinline__ KvqRow kvq_locate(const KvqView& v, int row, int lane) {
  KvqRow r{-1, nullptr, 0};
  // one row per sequence: the row is the sequence
  int s = v.max_rows == 1 && v.n_rows == v.n_seq ? row : kvq_find_seq(v, row, lane);
  if (s >= 0) {
    const int end = __ldg(v.row_start + s + 1), ln = __ldg(v.len + s);
    const int p = ln - (end - row);
    if (__ldg(v.row_start + s) <= row && end > row && p >= 0 && (p >> v.page_shift) < v.pages_ld) {
      const int pg = __ldg(v.pages + (size_t)s * v.pages_ld + (p >> v.page_shift));
      if ((unsigned)pg < (unsigned)v.n_pages) {
        r.pos = p;
        r.page = v.pool + (size_t)pg * v.page_bytes;
        r.off = p & ((1 << v.page_shift) - 1);
        return r;
      }
    }
  }
  if (lane == 0) kvq_fault(v, KVQ_FAULT_DATA);
  return r;
}

}  // namespace lumina
