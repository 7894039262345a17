// Beam search's reordering of a paged cache: row r takes over the cached tokens of row parents[r] (of the same length), in every pool.
//
// Pages that are full are shared: the row's block table names its parent's.  The open page of a row is the row's own (the entries from
// seq_lens / 16 on never change), so that it gets the parent's bytes.  Nothing is allocated and no full page is ever copied or written again.
// Rows read what other rows write: a CTA owns a stretch of bytes (of columns) for ALL rows, and reads all of them before it writes any.
// Bytes: 2 * page bytes for each pool and row that changes its parent inside a page, 8 for each table entry; a few microseconds of latency.
#include "common.cuh"

namespace tsb {
namespace {

constexpr int kThreads = 256, kPieces = 8, kMaxRows = kThreads * kPieces;

struct ReorderArgs {
  int64_t page_bytes, num_pages, bt_stride;
  int rows, pools, scales, width;          // width: floats of a row of scales
  int page_cols, page_ctas, table_cols, table_ctas, scale_cols, scale_ctas;     // stretch of a CTA (16-byte pieces, entries, floats); CTAs
};

// Rows whose tokens change hands: another parent, in range, of the row's own length.
__device__ __forceinline__ bool taken_over(const int32_t* __restrict__ parents, const int32_t* __restrict__ lens, int rows, int r, int& parent, int& len) {
  parent = parents[r];
  len = lens[r];
  return parent != r && parent >= 0 && parent < rows && len > 0 && lens[parent] == len;
}

__global__ void __launch_bounds__(kThreads)
kv_reorder_kernel(uint8_t* const* __restrict__ pools, float* const* __restrict__ scales, int32_t* table, const int32_t* __restrict__ lens,
                  const int32_t* __restrict__ parents, ReorderArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  int block = (int)blockIdx.x;
  if (block < a.pools * a.page_ctas) {
    uint8_t* pool = pools[block / a.page_ctas];
    const int64_t at = (int64_t)(block % a.page_ctas) * a.page_cols, cols = min((int64_t)a.page_cols, a.page_bytes / 16 - at);
    uint4 v[kPieces];
    uint4* dst[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int idx = threadIdx.x + i * kThreads;
      dst[i] = nullptr;
      const int r = (int)(idx / cols);
      int parent, len;
      if (r < a.rows && taken_over(parents, lens, a.rows, r, parent, len) && (len & 15) && (len >> 4) < a.bt_stride) {
        const int64_t from = table[parent * a.bt_stride + (len >> 4)], to = table[r * a.bt_stride + (len >> 4)];
        if (from >= 0 && from < a.num_pages && to >= 0 && to < a.num_pages) {
          const int64_t off = (at + idx % cols) * 16;
          v[i] = *reinterpret_cast<const uint4*>(pool + from * a.page_bytes + off);
          dst[i] = reinterpret_cast<uint4*>(pool + to * a.page_bytes + off);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      if (dst[i]) *dst[i] = v[i];
    return;
  }
  block -= a.pools * a.page_ctas;
  const bool is_table = block < a.table_ctas;
  if (!is_table) block -= a.table_ctas;
  unsigned* base = is_table ? reinterpret_cast<unsigned*>(table) : reinterpret_cast<unsigned*>(scales[block / a.scale_ctas]);
  const int64_t stride = is_table ? a.bt_stride : a.width;
  const int64_t per = is_table ? a.table_cols : a.scale_cols;
  const int64_t at = (is_table ? block : block % a.scale_ctas) * per, cols = min(per, stride - at);
  unsigned v[kPieces];
  unsigned* dst[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int idx = threadIdx.x + i * kThreads;
    dst[i] = nullptr;
    const int r = (int)(idx / cols);
    int parent, len;
    if (r < a.rows && taken_over(parents, lens, a.rows, r, parent, len)) {
      const int64_t col = at + idx % cols;
      if (!is_table || col < (len >> 4)) {
        v[i] = base[parent * stride + col];
        dst[i] = base + r * stride + col;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPieces; ++i)
    if (dst[i]) *dst[i] = v[i];
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
  const int64_t cols = kMaxRows / rows;
  auto split = [&](int64_t width, int& per, int& ctas) {
    per = (int)(cols < width ? cols : width);
    const int64_t n = (width + per - 1) / per;
    ctas = (int)n;
    return n;
  };
  int64_t total = split(bt_stride, a.table_cols, a.table_ctas);
  a.page_cols = a.scale_cols = 1;
  a.page_ctas = a.scale_ctas = 0;
  if (n_pools) total += n_pools * split(page_bytes / 16, a.page_cols, a.page_ctas);
  if (n_scales) total += n_scales * split(scale_width, a.scale_cols, a.scale_ctas);
  if (total > 0x7fffffffLL) return TSB200_ERR_UNSUPPORTED;
  TSB_CUDA(launch_kernel(kv_reorder_kernel, dim3((unsigned)total), dim3(kThreads), 0, as_stream(stream), (uint8_t* const*)pools, scales, block_table, seq_lens,
                         parents, a));
  return TSB200_OK;
}
