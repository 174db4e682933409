// The paged key-value cache as the kernels see it (struct ecah_kv_cache), and
// the host checks its launchers share.
#pragma once

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

}  // namespace kv
}  // namespace ecah
