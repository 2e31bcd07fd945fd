// Shared definitions of the operators on a paged cache of head_dim-512 keys and values.
//
// A cache is two tensors of pages (num_pages, page_size, heads_kv, 512). Slot j of sequence b is row j % page_size of
// page page_table[b][j / page_size]. Every page id is checked against num_pages before it becomes an address: a row of
// a page that does not exist is neither read nor written, and the call leaves ST_BAD_PAGE in the status word.
#pragma once
#include "common.cuh"
#include "ptx.cuh"

namespace sd {

constexpr int kRowBytes = kHeadDim * 2;

struct PageMap {
  const int* table;      // (batch, table_stride)
  int64_t table_stride;  // elements
  int max_pages;         // entries of a row of the table that belong to it
  int page_size;
  int num_pages;
  int shift;             // log2(page_size), or -1
};

// Slots that the table can address.
__host__ __device__ inline int page_capacity(const PageMap& m) {
  const int64_t n = static_cast<int64_t>(m.max_pages) * m.page_size;
  constexpr int64_t kMost = 0x7fffffff - 65536;  // a slot plus a step of any loop over slots stays below 2^31
  return static_cast<int>(n < kMost ? n : kMost);
}
__host__ inline int page_shift(int page_size) {
  for (int s = 0; s < 31; ++s)
    if (page_size == (1 << s)) return s;
  return -1;
}
// slot (>= 0, < page_capacity) -> entry of the table's row and row inside the page
__device__ __forceinline__ void split_slot(const PageMap& m, int slot, int& entry, int& row) {
  entry = m.shift >= 0 ? slot >> m.shift : slot / m.page_size;
  row = slot - (m.shift >= 0 ? entry << m.shift : entry * m.page_size);
}
__device__ __forceinline__ int page_of(const PageMap& m, int b, int entry) {
  return __ldg(m.table + static_cast<int64_t>(b) * m.table_stride + entry);
}
__device__ __forceinline__ bool page_ok(const PageMap& m, int page) {
  return static_cast<unsigned>(page) < static_cast<unsigned>(m.num_pages);
}

}  // namespace sd
