// Attention of a batch's rows over quantized KV pages: the entry point and
// the choice between the two kernels.
//
// A sequence of few packed rows (new rows x query heads per KV head) is bound
// by reading its cache and goes to the decode kernel (kvq_decode.cu), in tasks
// of up to 16 packed rows per KV head; one of more than 48 (fp32 rows: 64)
// goes to the chunk kernel (kvq_chunk.cu), bound by its softmax work. A task
// holds whole rows, so where the heads do not divide 16 there are more tasks
// than 48 / 16, and the decode kernel is still the faster one (below).
// Each kernel takes its own sequences out of the batch, so a batch may mix
// them. Decode / chunk kernel, int8, head dim 128, 8 KV heads, lengths up to
// 4096, fp16 rows unless said:
//   8 sequences,  20 packed rows     39 /  57 us, fp32 rows 43 / 65 us
//   8 sequences,  48 packed rows     50 /  59 us
//   8 sequences,  64 packed rows     59 /  59 us, fp32 rows 67 / 72 us
//   32 sequences, 32 packed rows    104 / 131 us
//   32 sequences, 48 packed rows    146 / 136 us
//   32 sequences, 64 packed rows    190 / 136 us, fp32 rows 221 / 165 us
//   8 sequences x 5 rows of 9 heads  40 /  59 us (4 KV heads; five tasks of a row)
//   8 sequences x 4 rows of 12 heads 33 /  60 us (2 KV heads; four tasks)
// Sequences for the decode kernel take at least a cell per warp and CTA
// (1 x 640 tokens, 32 KV heads: 12.4 us; 14.4 with two cells, 16.4 with three).
// Beside a sequence for the chunk kernel the others mostly bring one row, so
// the decode kernel's blocks are 8 rows there.
#include <cmath>

#include "kvq_attend.cuh"

namespace lumina {

namespace {

template <int HD, int BITS, typename T>
int attend_launch(AttendArgs a, cudaStream_t s) {
  // a batch of equal row counts needs one of the two kernels only
  const long long max_packed = (long long)a.v.max_rows * a.G;
  const bool equal = (long long)a.v.max_rows * a.v.n_seq == a.v.n_rows;
  const int blocks = sizeof(T) == 4 ? KVQ_DECODE_BLOCKS : KVQ_DECODE_BLOCKS - 1;
  const int most = blocks * KVQ_DECODE_ROWS;
  const int rows = max_packed <= 8 || (max_packed > most && a.G <= 8) ? 8 : KVQ_DECODE_ROWS;  // of a decode block
  a.few = a.G <= rows ? blocks * rows : 0;
  const bool decode = a.few && (max_packed <= a.few || !equal);
  if (decode) {
    const int rc = kvq_decode_launch<HD, BITS, T>(a, rows, s);
    if (rc) return rc;
  }
  if (max_packed <= a.few) return LUMINA_OK;
  a.tickets += KVQ_WS_DECODE_TICKETS;
  a.ws += KVQ_WS_DECODE;
  return kvq_chunk_launch<HD, BITS, T>(a, decode, s);
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
  // no shorter than the cache: it hides nothing (and a position less the
  // window stays within an int)
  a.window = args->window >= (long long)batch->pages_ld * pool->page_size ? 0 : args->window;
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
