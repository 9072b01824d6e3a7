// Device view of a paged key-value cache (RecPagedKV / RecPagedTable) and the
// slot arithmetic that the batched-decode kernels share.
#pragma once
#include "capi_common.h"
#include "common.cuh"

namespace rec {

// t / d for 0 <= t < 2^31 and 1 <= d < 2^31 by one high multiplication:
// with l = ceil(log2 d), mul = floor(2^32 (2^l - d) / d) + 1,
// t / d = (mulhi(t, mul) + t) >> l (Granlund and Montgomery's round-up method).
struct FastDiv {
  uint32_t d, mul, shift;
};
inline FastDiv make_fastdiv(uint32_t d) {
  uint32_t l = 0;
  while (l < 31 && (1u << l) < d) ++l;
  const uint64_t mul = (((uint64_t(1) << l) - d) << 32) / d + 1;
  return {d, uint32_t(mul), l};
}
__device__ __forceinline__ uint32_t fdiv(uint32_t t, const FastDiv& f) { return (__umulhi(t, f.mul) + t) >> f.shift; }

// One tensor of the pool.  The page, head and row strides are in 16-byte
// units (rows) or 2-byte units (scales), so that a row's place fits 32 bits
// while the pool may span 64 GB (8 GB of scales); the host checks the spans.
struct PagedRows {
  uint8_t* base;
  uint32_t page, head, row;
};
struct PagedScales {
  uint16_t *s, *b;
  uint32_t page, head, row;
};
struct PagedView {
  PagedRows k, v;
  PagedScales ks, vs;
  int n_pages, hkv, d, k_bits, v_bits, fp16;
  FastDiv ps;
  const int* table;
  int64_t table_stride;
  int width, batch;
  int64_t slots;  // width * page_size
};

// The page of slot t of session b, or -1 (outside the table, or a page
// outside the pool).
__device__ __forceinline__ int slot_page(const PagedView& p, int b, int t, int& off) {
  const uint32_t e = fdiv(uint32_t(t), p.ps);
  off = t - int(e * p.ps.d);
  if (int64_t(e) >= p.width) return -1;
  const int page = p.table[int64_t(b) * p.table_stride + e];
  return uint32_t(page) < uint32_t(p.n_pages) ? page : -1;
}
// Place of (page, head, off) in a tensor with one value per slot.
__device__ __forceinline__ int64_t slot_index(const PagedView& p, int page, int h, int off) {
  return (int64_t(page) * p.hkv + h) * p.ps.d + off;
}
__device__ __forceinline__ uint8_t* row_ptr(const PagedRows& r, int page, int h, int off) {
  return r.base + (size_t(uint32_t(page) * r.page + uint32_t(h) * r.head + uint32_t(off) * r.row) << 4);
}
__device__ __forceinline__ size_t scale_at(const PagedScales& r, int page, int h, int off) {
  return size_t(uint32_t(page) * r.page + uint32_t(h) * r.head + uint32_t(off) * r.row);
}

// Checks a cache and a table and fills the view; `who` names the caller in
// messages.  Host only.
int paged_view(const RecPagedKV* kv, const RecPagedTable* table, const char* who, PagedView* out);

}  // namespace rec
