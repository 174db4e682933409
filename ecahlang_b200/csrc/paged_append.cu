// Norm, rotation and cache write of new tokens: ecah_paged_append (contract
// in include/ecah_sampler.h).

#include <cuda_fp8.h>

#include "host_util.h"
#include "paged.cuh"

namespace ecah {
namespace append {

constexpr int kT = 256;

struct Params {
  const void *q, *k, *v;
  void* q_out;
  const void *q_norm, *k_norm;
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head, qo_tok, qo_head;
  const float* cos_sin;
  const int* positions;
  const int* batch_index;
  int tokens, hq, D, table_rows, interleaved;
  float eps;
  kv::Cache cache;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
// keeps a NaN, so that its row's scale is one
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}

// One warp per token and head (queries, then keys, then values); lane l takes
// the pairs l, l + 32, ...
template <int DT, bool E4M3>
__global__ void __launch_bounds__(kT) append_kernel(const Params P) {
  using DTy = DType<DT>;
  constexpr int kPairs = 4;   // head_dim 256 / 2 / 32
  const int lane = threadIdx.x & 31;
  const int heads = P.hq + 2 * P.cache.heads;
  const long long unit = static_cast<long long>(blockIdx.x) * (kT / 32) + (threadIdx.x >> 5);
  if (unit >= static_cast<long long>(P.tokens) * heads) return;
  const int t = static_cast<int>(unit / heads), hh = static_cast<int>(unit % heads);
  const bool is_q = hh < P.hq, is_v = hh >= P.hq + P.cache.heads;
  const int h = is_q ? hh : is_v ? hh - P.hq - P.cache.heads : hh - P.hq;
  const uint16_t* x = static_cast<const uint16_t*>(is_q ? P.q : is_v ? P.v : P.k);
  x += is_q ? t * P.q_tok + h * P.q_head : is_v ? t * P.v_tok + h * P.v_head : t * P.k_tok + h * P.k_head;
  const int half = P.D / 2, pos = P.positions[t];
  float a[kPairs], b[kPairs];
  int ia[kPairs], ib[kPairs];
  for (int i = 0; i < kPairs; ++i) {
    const int p = lane + 32 * i;
    ia[i] = P.interleaved ? 2 * p : p;
    ib[i] = P.interleaved ? 2 * p + 1 : p + half;
    a[i] = p < half ? DTy::to_f32(x[ia[i]]) : 0.0f;
    b[i] = p < half ? DTy::to_f32(x[ib[i]]) : 0.0f;
  }
  const uint16_t* w = static_cast<const uint16_t*>(is_q ? P.q_norm : P.k_norm);
  if (!is_v && w) {
    float ss = 0.0f;
    for (int i = 0; i < kPairs; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
    const float inv = rsqrtf(warp_sum(ss) / static_cast<float>(P.D) + P.eps);
    for (int i = 0; i < kPairs; ++i)
      if (lane + 32 * i < half) {
        a[i] = a[i] * inv * DTy::to_f32(w[ia[i]]);
        b[i] = b[i] * inv * DTy::to_f32(w[ib[i]]);
      }
  }
  if (!is_v && P.cos_sin) {
    const float* cs = P.cos_sin + static_cast<long long>(min(max(pos, 0), P.table_rows - 1)) * P.D;
    for (int i = 0; i < kPairs; ++i) {
      const int p = lane + 32 * i;
      if (p >= half) continue;
      const float c = cs[p], s = cs[half + p], u = a[i], v = b[i];
      a[i] = u * c - v * s;
      b[i] = v * c + u * s;
    }
  }
  if (is_q) {
    uint16_t* o = static_cast<uint16_t*>(P.q_out) + t * P.qo_tok + h * P.qo_head;
    for (int i = 0; i < kPairs; ++i)
      if (lane + 32 * i < half) {
        o[ia[i]] = DTy::to_raw(a[i]);
        o[ib[i]] = DTy::to_raw(b[i]);
      }
    return;
  }
  const int req = P.batch_index[t];
  if (req < 0 || req >= P.cache.batch || pos < 0) return;
  long long first, count;
  kv::page_range(P.cache, req, &first, &count);
  const int nth = pos / P.cache.page_size, slot = pos % P.cache.page_size;
  if (nth >= count) return;
  const int page = P.cache.indices[first + nth];
  if (page < 0 || page >= P.cache.num_pages) return;
  const kv::Side& side = is_v ? P.cache.v : P.cache.k;
  const long long at = page * side.page + slot * side.slot + h * side.head;
  if (!E4M3) {
    uint16_t* o = static_cast<uint16_t*>(side.base) + at;
    for (int i = 0; i < kPairs; ++i)
      if (lane + 32 * i < half) {
        o[ia[i]] = DTy::to_raw(a[i]);
        o[ib[i]] = DTy::to_raw(b[i]);
      }
    return;
  }
  float big = 0.0f;
  for (int i = 0; i < kPairs; ++i) big = max_nan(big, max_nan(fabsf(a[i]), fabsf(b[i])));
  big = max_nan(warp_max_nan(big), 448e-12f);
  const float scale = big / 448.0f;
  if (lane == 0) side.scale[(static_cast<long long>(page) * P.cache.heads + h) * P.cache.page_size + slot] = scale;
  __nv_fp8_storage_t* o = static_cast<__nv_fp8_storage_t*>(side.base) + at;
  for (int i = 0; i < kPairs; ++i)
    if (lane + 32 * i < half) {
      o[ia[i]] = __nv_cvt_float_to_fp8(a[i] / scale, __NV_SATFINITE, __NV_E4M3);
      o[ib[i]] = __nv_cvt_float_to_fp8(b[i] / scale, __NV_SATFINITE, __NV_E4M3);
    }
}

}  // namespace append
}  // namespace ecah

using namespace ecah;

extern "C" int ecah_paged_append(const ecah_append_args* a, void* stream) {
  if (!a) return ECAH_ERR_NULL;
  if (a->abi_version != ECAH_SAMPLER_ABI_VERSION) return ECAH_ERR_ABI;
  const int st = kv::check_cache(a->cache, a->dtype);
  if (st != ECAH_OK) return st;
  if (a->tokens < 0 || a->num_qo_heads < 0 || (a->cos_sin && a->table_rows < 1)) return ECAH_ERR_SHAPE;
  for (long long s : {a->q_token_stride, a->q_head_stride, a->k_token_stride, a->k_head_stride, a->v_token_stride,
                      a->v_head_stride, a->qo_token_stride, a->qo_head_stride})
    if (s < 0 || s % 8) return ECAH_ERR_SHAPE;
  if (a->tokens == 0) return ECAH_OK;
  if (!a->k || !a->v || !a->positions || !a->batch_index) return ECAH_ERR_NULL;
  if (a->q ? (!a->q_out || a->num_qo_heads < 1) : a->num_qo_heads != 0) return a->q && !a->q_out ? ECAH_ERR_NULL : ECAH_ERR_SHAPE;
  for (const void* p : {a->q, a->k, a->v, static_cast<const void*>(a->q_out), a->q_norm, a->k_norm,
                        static_cast<const void*>(a->cos_sin)})
    if (!kv::aligned16(p)) return ECAH_ERR_SHAPE;
  append::Params P = {};
  P.q = a->q; P.k = a->k; P.v = a->v; P.q_out = a->q_out;
  P.q_norm = a->q_norm; P.k_norm = a->k_norm;
  P.q_tok = a->q_token_stride; P.q_head = a->q_head_stride;
  P.k_tok = a->k_token_stride; P.k_head = a->k_head_stride;
  P.v_tok = a->v_token_stride; P.v_head = a->v_head_stride;
  P.qo_tok = a->qo_token_stride; P.qo_head = a->qo_head_stride;
  P.cos_sin = a->cos_sin;
  P.positions = a->positions; P.batch_index = a->batch_index;
  P.tokens = a->tokens; P.hq = a->q ? a->num_qo_heads : 0; P.D = a->cache.head_dim;
  P.table_rows = a->table_rows; P.interleaved = a->interleaved;
  P.eps = a->eps;
  P.cache = kv::make_cache(a->cache);
  const long long units = static_cast<long long>(P.tokens) * (P.hq + 2ll * P.cache.heads);
  const long long blocks = (units + append::kT / 32 - 1) / (append::kT / 32);
  if (blocks > 0x7FFFFFFF) return ECAH_ERR_SHAPE;
  const bool e4m3 = a->cache.kv_dtype == ECAH_KV_E4M3, f16 = a->dtype == ECAH_DTYPE_F16;
  auto fn = f16 ? (e4m3 ? append::append_kernel<ECAH_DTYPE_F16, true> : append::append_kernel<ECAH_DTYPE_F16, false>)
                : (e4m3 ? append::append_kernel<ECAH_DTYPE_BF16, true> : append::append_kernel<ECAH_DTYPE_BF16, false>);
  return launch_kernel(fn, dim3(static_cast<unsigned>(blocks)), append::kT, 0, reinterpret_cast<cudaStream_t>(stream), P)
             ? ECAH_OK : ECAH_ERR_LAUNCH;
}
