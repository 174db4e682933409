// Attention of several new tokens per request over the paged key-value cache:
// ecah_paged_prefill (contract in include/ecah_sampler.h).

#include <cuda_fp8.h>

#include <algorithm>

#include "host_util.h"
#include "paged.cuh"

namespace ecah {
namespace prefill {

// One warp to a token and query head, keys one after another.

constexpr int kT = 128;

struct Params {
  const void* q;
  void* out;
  float* lse;
  const int *qo_indptr, *last_page_len;
  long long q_tok, q_head, o_tok, o_head;
  int tokens, hq, group, causal;
  float scale;               // sm_scale * log2 e
  kv::Cache cache;
};

template <int DT, bool E4M3>
__device__ __forceinline__ float value(const void* base, long long at) {
  if (E4M3) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<const __nv_fp8_storage_t*>(base)[at], __NV_E4M3);
    return __half2float(__half(h));
  }
  return DType<DT>::to_f32(static_cast<const uint16_t*>(base)[at]);
}

template <int DT, bool E4M3, int D>
__global__ void __launch_bounds__(kT) prefill_kernel(const Params P) {
  grid_start();
  constexpr int kN = D / 32;
  const int lane = threadIdx.x & 31;
  const long long id = static_cast<long long>(blockIdx.x) * (kT / 32) + (threadIdx.x >> 5);
  const int t = static_cast<int>(id / P.hq), h = static_cast<int>(id % P.hq);
  if (t >= P.tokens) return;
  int b = -1, lo = 0, hi = 0;
  for (int i = 0; i < P.cache.batch; ++i) {
    lo = min(max(P.qo_indptr[i], 0), P.tokens);
    hi = min(max(P.qo_indptr[i + 1], lo), P.tokens);
    if (t >= lo && t < hi) { b = i; break; }
  }
  if (b < 0) return;
  long long at, count;
  kv::page_range(P.cache, b, &at, &count);
  long long len = 0;
  if (count > 0 && P.cache.num_pages > 0)
    len = (count - 1) * P.cache.page_size + min(max(P.last_page_len[b], 0), P.cache.page_size);
  const long long seen = P.causal ? min(len, max(len - (hi - lo) + (t - lo) + 1, 0ll)) : len;
  const int kh = h / P.group;
  // the sum in blocks of 64 keys: one chain over a long row would lose its last digits
  float q[kN], o[kN], m = -INFINITY, l = 0.0f, some = 0.0f;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    q[i] = DType<DT>::to_f32(static_cast<const uint16_t*>(P.q)[t * P.q_tok + h * P.q_head + 32 * i + lane]);
    o[i] = 0.0f;
  }
  for (long long j = 0; j < seen; ++j) {
    const long long page = min(max(P.cache.indices[at + j / P.cache.page_size], 0), P.cache.num_pages - 1);
    const long long slot = j % P.cache.page_size;
    const long long ka = page * P.cache.k.page + slot * P.cache.k.slot + kh * P.cache.k.head + lane;
    const long long va = page * P.cache.v.page + slot * P.cache.v.slot + kh * P.cache.v.head + lane;
    const long long sa = (page * P.cache.heads + kh) * P.cache.page_size + slot;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kN; ++i) s = fmaf(q[i], value<DT, E4M3>(P.cache.k.base, ka + 32 * i), s);
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, x);
    s *= P.scale * (E4M3 ? P.cache.k.scale[sa] : 1.0f);
    const float top = fmaxf(m, s), f = m == top ? 1.0f : ex2_approx(m - top);
    const float p = s == -INFINITY ? 0.0f : ex2_approx(s - top);
    m = top;
    l *= f;
    some = fmaf(some, f, p);
    if ((j & 63) == 63) { l += some; some = 0.0f; }
    const float w = p * (E4M3 ? P.cache.v.scale[sa] : 1.0f);
#pragma unroll
    for (int i = 0; i < kN; ++i) o[i] = fmaf(o[i], f, w * value<DT, E4M3>(P.cache.v.base, va + 32 * i));
  }
  l += some;
  const float r = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < kN; ++i)
    static_cast<uint16_t*>(P.out)[t * P.o_tok + h * P.o_head + 32 * i + lane] = DType<DT>::to_raw(o[i] * r);
  if (P.lse && lane == 0) P.lse[static_cast<long long>(t) * P.hq + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

using KernelFn = void (*)(const Params);

template <int DT, bool E4M3>
static KernelFn kernel_for(int D) {
  switch (D) {
    case 64: return prefill_kernel<DT, E4M3, 64>;
    case 96: return prefill_kernel<DT, E4M3, 96>;
    case 128: return prefill_kernel<DT, E4M3, 128>;
    case 192: return prefill_kernel<DT, E4M3, 192>;
    default: return prefill_kernel<DT, E4M3, 256>;
  }
}

}  // namespace prefill
}  // namespace ecah

using namespace ecah;

extern "C" {

size_t ecah_paged_prefill_workspace_bytes(int32_t head_dim) {
  if (!kv::head_dim_ok(head_dim) || device_sms() <= 0) return 0;
  return 256;
}

int ecah_paged_prefill(const ecah_prefill_args* a, void* stream) {
  if (!a) return ECAH_ERR_NULL;
  if (a->abi_version != ECAH_SAMPLER_ABI_VERSION) return ECAH_ERR_ABI;
  const int st = kv::check_cache(a->cache, a->dtype);
  if (st != ECAH_OK) return st;
  const ecah_kv_cache& c = a->cache;
  if (a->tokens < 0 || a->num_qo_heads < 1 || a->num_qo_heads % c.num_kv_heads || !(a->sm_scale > 0.0f)) return ECAH_ERR_SHAPE;
  for (long long s : {a->q_token_stride, a->q_head_stride, a->out_token_stride, a->out_head_stride})
    if (s < 0 || s % 8) return ECAH_ERR_SHAPE;
  if (c.batch == 0 || a->tokens == 0) return ECAH_OK;
  if (!a->q || !a->out || !a->qo_indptr || !a->kv_last_page_len) return ECAH_ERR_NULL;
  if (!aligned16(a->q) || !aligned16(a->out)) return ECAH_ERR_SHAPE;
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < ecah_paged_prefill_workspace_bytes(c.head_dim))
    return ECAH_ERR_WORKSPACE;
  if (device_sms() <= 0) return ECAH_ERR_LAUNCH;
  prefill::Params P = {};
  P.q = a->q; P.out = a->out; P.lse = a->lse;
  P.qo_indptr = a->qo_indptr; P.last_page_len = a->kv_last_page_len;
  P.q_tok = a->q_token_stride; P.q_head = a->q_head_stride;
  P.o_tok = a->out_token_stride; P.o_head = a->out_head_stride;
  P.tokens = a->tokens; P.hq = a->num_qo_heads; P.group = a->num_qo_heads / c.num_kv_heads; P.causal = a->causal;
  P.scale = a->sm_scale * kLog2e;
  P.cache = kv::make_cache(c);
  const bool e4m3 = c.kv_dtype == ECAH_KV_E4M3;
  const prefill::KernelFn fn =
      a->dtype == ECAH_DTYPE_F16 ? (e4m3 ? prefill::kernel_for<ECAH_DTYPE_F16, true>(c.head_dim) : prefill::kernel_for<ECAH_DTYPE_F16, false>(c.head_dim))
                                 : (e4m3 ? prefill::kernel_for<ECAH_DTYPE_BF16, true>(c.head_dim) : prefill::kernel_for<ECAH_DTYPE_BF16, false>(c.head_dim));
  const long long blocks = (static_cast<long long>(a->tokens) * a->num_qo_heads + prefill::kT / 32 - 1) / (prefill::kT / 32);
  if (blocks > 0x7FFFFFFF) return ECAH_ERR_SHAPE;
  return launch_kernel(fn, dim3(static_cast<unsigned>(blocks)), prefill::kT, 0, reinterpret_cast<cudaStream_t>(stream), P)
             ? ECAH_OK : ECAH_ERR_LAUNCH;
}

}  // extern "C"
