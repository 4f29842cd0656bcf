// The paged KV cache on the device: addresses of rows, and the argument checks of its entry points.
#pragma once
#include "axm.h"
#include "axm_common.h"

// One layer's pool and the sequences' tables, as kernels take it.
struct PagedKv {
  uint8_t* k;
  uint8_t* v;
  uint8_t* ks;
  uint8_t* vs;
  const int* table;
  int64_t page_stride, scale_stride;  // bytes
  int kv_dtype, Hkv, hd, page_shift, n_pages, n_seqs, max_pages;
};

__host__ __device__ static inline int paged_row_bytes(int kv_dtype, int hd) {
  return kv_dtype == AXM_KV_FP16 ? 2 * hd : kv_dtype == AXM_KV_FP8 ? hd : hd / 2;
}

// Page of slot `slot` (>= 0) of sequence b; -1 outside the table or the pool.
__device__ __forceinline__ int paged_page(const PagedKv& kv, int b, int slot) {
  const int i = slot >> kv.page_shift;
  if (i >= kv.max_pages) return -1;
  const int page = kv.table[(size_t)b * kv.max_pages + i];
  return (unsigned)page < (unsigned)kv.n_pages ? page : -1;
}

// Offsets of a row inside one layer's codes / scales, 64 bits wide: pools pass 4 GiB.
__device__ __forceinline__ int64_t paged_row(const PagedKv& kv, int page, int h, int slot, int row_bytes) {
  const int in_page = (h << kv.page_shift) + (slot & ((1 << kv.page_shift) - 1));
  return page * kv.page_stride + (int64_t)in_page * row_bytes;
}
__device__ __forceinline__ int64_t paged_scale_row(const PagedKv& kv, int page, int h, int slot) {
  const int in_page = (h << kv.page_shift) + (slot & ((1 << kv.page_shift) - 1));
  return page * kv.scale_stride + (int64_t)in_page * (kv.hd / 64 * 2);
}

// Checks a descriptor and fills the kernel's view of it; 0 or an error code with its message set.
int paged_view(const axm_paged_kv* d, const char* who, PagedKv* out);
