// The paged key-value cache as the kernels see it (struct ecah_kv_cache), and
// the host checks its launchers share.
#pragma once

#include <algorithm>

#include "common.cuh"
#include "host_util.h"

namespace ecah {
namespace kv {

// One of the cache's two tensors: rows of head_dim at page, slot and head
// strides (elements).
struct Side {
  void* base;
  long long page, slot, head;
  float* scale;               // [pages, heads, page_size], e4m3 only
};

struct Cache {
  Side k, v;
  const int* indptr;
  const int* indices;
  long long num_indices;
  int num_pages, page_size, heads, batch;
};

// Page list of request b, clamped into the index array.
__device__ __forceinline__ void page_range(const Cache& c, int b, long long* first, long long* count) {
  const long long lo = min(max(static_cast<long long>(c.indptr[b]), 0ll), c.num_indices);
  const long long hi = min(max(static_cast<long long>(c.indptr[b + 1]), lo), c.num_indices);
  *first = lo;
  *count = hi - lo;
}

// One side of the cache in 16-byte units from its base.
struct Side16 {
  const unsigned char* base;
  unsigned page, slot, head;
  const float* scale;
};

inline bool head_dim_ok(int d) { return d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

// Shape and pointer checks of a cache with a model dtype of 2 bytes.
inline int check_cache(const ecah_kv_cache& c, int dtype) {
  if (dtype != ECAH_DTYPE_F16 && dtype != ECAH_DTYPE_BF16) return ECAH_ERR_DTYPE;
  if (c.kv_dtype != dtype && c.kv_dtype != ECAH_KV_E4M3) return ECAH_ERR_DTYPE;
  if (c.num_pages < 0 || c.page_size < 1 || c.num_kv_heads < 1 || !head_dim_ok(c.head_dim) || c.batch < 0 || c.num_indices < 0)
    return ECAH_ERR_SHAPE;
  if (!c.kv_indptr || (c.num_indices && !c.kv_indices)) return ECAH_ERR_NULL;
  if (c.num_pages == 0) return ECAH_OK;
  if (!c.k_cache || !c.v_cache) return ECAH_ERR_NULL;
  const bool e4m3 = c.kv_dtype == ECAH_KV_E4M3;
  if (e4m3 && (!c.k_scale || !c.v_scale)) return ECAH_ERR_NULL;
  const long long unit = e4m3 ? 16 : 8;   // elements of 16 bytes
  for (long long s : {c.k_page_stride, c.k_slot_stride, c.k_head_stride, c.v_page_stride, c.v_slot_stride, c.v_head_stride})
    if (s < 0 || s % unit) return ECAH_ERR_SHAPE;
  if (!aligned16(c.k_cache) || !aligned16(c.v_cache)) return ECAH_ERR_SHAPE;
  return ECAH_OK;
}

inline Cache make_cache(const ecah_kv_cache& c) {
  Cache r = {};
  r.k = Side{c.k_cache, c.k_page_stride, c.k_slot_stride, c.k_head_stride, c.k_scale};
  r.v = Side{c.v_cache, c.v_page_stride, c.v_slot_stride, c.v_head_stride, c.v_scale};
  r.indptr = c.kv_indptr;
  r.indices = c.kv_indices;
  r.num_indices = c.num_indices;
  r.num_pages = c.num_pages;
  r.page_size = c.page_size;
  r.heads = c.num_kv_heads;
  r.batch = c.batch;
  return r;
}

// A side of the cache in 16-byte units; false where a row lies past 2^32 of them
// (64 GB from the base).
inline bool side16(const Side& s, int pages, int page_size, int heads, int elem, Side16* r) {
  const long long unit = 16 / elem;
  const long long most = (std::max(pages, 1) - 1ll) * (s.page / unit) + (page_size - 1ll) * (s.slot / unit) + (heads - 1ll) * (s.head / unit);
  if (s.page / unit > 0xFFFFFFFFll || s.slot / unit > 0xFFFFFFFFll || s.head / unit > 0xFFFFFFFFll || most + 64 > 0xFFFFFFFFll) return false;
  *r = Side16{static_cast<const unsigned char*>(s.base), static_cast<unsigned>(s.page / unit), static_cast<unsigned>(s.slot / unit),
              static_cast<unsigned>(s.head / unit), s.scale};
  return true;
}

// log2 of a page size that is a power of two, or -1.
inline int page_shift(int page_size) {
  for (int i = 0; i < 31; ++i)
    if (page_size == 1 << i) return i;
  return -1;
}

}  // namespace kv
}  // namespace ecah
