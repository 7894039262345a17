// Beam search's reordering of a paged cache: row r takes over the cached tokens of row parents[r] (of the same length), in every pool.
//
// Pages that are full are shared: the row's block table names its parent's.  The open page of a row is the row's own (the entries from
// seq_lens / 16 on never change), so that it gets the parent's bytes.  Nothing is allocated and no full page is ever copied or written again.
// Rows read what other rows write: a CTA owns a stretch of bytes (of columns) for ALL rows, and reads all of them before it writes any.
// Bytes: 2 * page bytes for each pool and row that changes its parent inside a page, 8 for each table entry; for few rows the chain parents -> lengths
// -> table -> page.  Rows that change are looked up once a CTA; stretches are powers of two (16 sequences x 4 beams, 32 layers of 8 heads of 128: 31.2 us with
// a lookup and two divisions for each 16 bytes, 21.4 now).
#include "common.cuh"

namespace tsb {
namespace {

constexpr int kThreads = 256, kPieces = 8, kMaxRows = kThreads * kPieces;

struct ReorderArgs {
  int64_t page_bytes, num_pages, bt_stride;
  int rows, pools, scales, width;          // width: floats of a row of scales
  int page_log, page_ctas, table_log, table_ctas, scale_log, scale_ctas;     // stretch of a CTA (16-byte pieces, entries, floats; its logarithm); CTAs
};

// Up to kPieces elements a thread, from row to row (where they start: from[], to[]), columns [at, at + 2^log) below the row's limit.
template <typename E, typename Limit>
__device__ __forceinline__ void move(E* base, const int64_t* from, const int64_t* to, int count, int at, int log, Limit limit) {
  E v[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int idx = threadIdx.x + i * kThreads, r = idx >> log, col = at + (idx & ((1 << log) - 1));
    if (r < count && col < limit(r)) v[i] = base[from[r] + col];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int idx = threadIdx.x + i * kThreads, r = idx >> log, col = at + (idx & ((1 << log) - 1));
    if (r < count && col < limit(r)) base[to[r] + col] = v[i];
  }
}

__global__ void __launch_bounds__(kThreads)
kv_reorder_kernel(uint8_t* const* __restrict__ pools, float* const* __restrict__ scales, int32_t* table, const int32_t* __restrict__ lens,
                  const int32_t* __restrict__ parents, ReorderArgs a) {
  extern __shared__ int64_t s_rows[];                        // [2][rows]: where a row that changes reads and writes; then int [rows]: its limit
  __shared__ int s_count;
  int64_t* s_from = s_rows;
  int64_t* s_to = s_rows + a.rows;
  int* s_full = reinterpret_cast<int*>(s_rows + 2 * a.rows);
  // Nothing that follows is let in before the end: an append or attention two launches on looks its table up ahead of its own wait, and the launch
  // between the two may have begun, and let that one begin, while this one runs.
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();
  pdl_wait();
  int block = (int)blockIdx.x;
  const bool is_page = block < a.pools * a.page_ctas;
  if (!is_page) block -= a.pools * a.page_ctas;
  const bool is_table = !is_page && block < a.table_ctas;
  if (!is_page && !is_table) block -= a.table_ctas;
  for (int r = threadIdx.x; r < a.rows; r += kThreads) {
    const int parent = parents[r], len = lens[r], full = len >> 4;
    // rows whose tokens change hands: another parent, in range, of the row's own length
    if (parent == r || parent < 0 || parent >= a.rows || len <= 0 || lens[parent] != len) continue;
    int64_t from, to;
    if (is_page) {
      if (!(len & 15) || full >= a.bt_stride) continue;
      from = table[parent * a.bt_stride + full];
      to = table[r * a.bt_stride + full];
      if (from < 0 || from >= a.num_pages || to < 0 || to >= a.num_pages) continue;
      from *= a.page_bytes / 16;
      to *= a.page_bytes / 16;
    } else {
      from = parent * (is_table ? a.bt_stride : a.width);
      to = r * (is_table ? a.bt_stride : a.width);
    }
    const int slot = atomicAdd(&s_count, 1);
    s_from[slot] = from;
    s_to[slot] = to;
    s_full[slot] = (int)min((int64_t)full, a.bt_stride);
  }
  __syncthreads();
  const int count = s_count;
  if (is_page) {
    const int pieces = (int)(a.page_bytes / 16);
    move(reinterpret_cast<uint4*>(pools[block / a.page_ctas]), s_from, s_to, count, block % a.page_ctas << a.page_log, a.page_log, [=](int) { return pieces; });
  } else if (is_table) {
    move(table, s_from, s_to, count, block << a.table_log, a.table_log, [=](int r) { return s_full[r]; });
  } else {
    const int width = a.width;
    move(scales[block / a.scale_ctas], s_from, s_to, count, block % a.scale_ctas << a.scale_log, a.scale_log, [=](int) { return width; });
  }
  if (!is_page) __threadfence();        // (pages so read are older than a row's open one; all CTAs' fences: 64 x 4 rows 23.4 -> 26.6 us)
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" int tsb200_kv_reorder(void* const* pools, int n_pools, int64_t page_bytes, int64_t num_pages, float* const* scales, int n_scales, int scale_width,
                                 int32_t* block_table, int64_t bt_stride, const int32_t* seq_lens, const int32_t* parents, int64_t rows, void* stream) {
  TSB_REQUIRE_DEVICE();
  if (n_pools < 0 || n_scales < 0 || rows < 0 || bt_stride < 0 || num_pages < 0) return TSB200_ERR_ARG;
  if (rows == 0) return TSB200_OK;
  if (rows > kMaxRows) return TSB200_ERR_UNSUPPORTED;
  if (!block_table || !seq_lens || !parents || bt_stride == 0) return TSB200_ERR_ARG;
  if (n_pools && (!pools || page_bytes <= 0 || page_bytes % 16)) return TSB200_ERR_ARG;
  if (n_scales && (!scales || scale_width <= 0)) return TSB200_ERR_ARG;
  ReorderArgs a;
  a.page_bytes = page_bytes; a.num_pages = num_pages; a.bt_stride = bt_stride;
  a.rows = (int)rows; a.pools = n_pools; a.scales = n_scales; a.width = scale_width;
  if (page_bytes / 16 > 0x7fffffffLL || bt_stride > 0x7fffffffLL) return TSB200_ERR_UNSUPPORTED;
  auto split = [&](int64_t width, int& log, int& ctas) {
    log = 0;
    while ((2LL << log) * rows <= kMaxRows && (1LL << log) < width) ++log;
    const int64_t n = (width + (1LL << log) - 1) >> log;
    ctas = (int)n;
    return n;
  };
  int64_t total = split(bt_stride, a.table_log, a.table_ctas);
  a.page_log = a.scale_log = 0;
  a.page_ctas = a.scale_ctas = 0;
  if (n_pools) total += n_pools * split(page_bytes / 16, a.page_log, a.page_ctas);
  if (n_scales) total += n_scales * split(scale_width, a.scale_log, a.scale_ctas);
  if (total > 0x7fffffffLL) return TSB200_ERR_UNSUPPORTED;
  TSB_CUDA(launch_kernel(kv_reorder_kernel, dim3((unsigned)total), dim3(kThreads), (size_t)rows * 20, as_stream(stream), (uint8_t* const*)pools, scales, block_table, seq_lens,
                         parents, a));
  return TSB200_OK;
}
