// paged.cuh -- the paged KV cache as the kernels see it (ie_b200_kv_pages, include/ie_b200.h): where a position's rows lie, and
// the host's checks of the description.
#pragma once

#include "common.cuh"

namespace ieb {

constexpr uint32_t ERR_PAGES = 6u;  // error word: a length or position outside the table, or a page number outside the pools

// Checks of a description that every entry makes. page_multiple: what the entry wants the positions of a page to be a multiple of.
int check_pages(const char *who, const ie_b200_kv_pages *p, uint32_t page_multiple);

#ifdef __CUDACC__
// Positions that the table can name (below 2^31: check_pages).
__host__ __device__ __forceinline__ uint32_t table_positions(const ie_b200_kv_pages &p) { return p.table_cols * p.page; }
// The page number of column `col` of sequence `seq` (both inside the table).
__device__ __forceinline__ uint32_t page_number(const ie_b200_kv_pages &p, uint32_t seq, uint32_t col) { return p.table[(size_t)seq * p.table_stride + col]; }
// Byte offset, in either pool, of row `row` of KV head `head` in page `number`.
__device__ __forceinline__ size_t page_row(const ie_b200_kv_pages &p, uint32_t number, uint32_t head, uint32_t row, uint32_t row_bytes) {
  return (size_t)number * p.page_stride + ((size_t)head * p.page + row) * row_bytes;
}
#endif

}  // namespace ieb
