// Attention of one new token per request over the paged key-value cache:
// ecah_paged_decode (contract in include/ecah_sampler.h).

#include <cuda_fp8.h>

#include "host_util.h"
#include "paged.cuh"

namespace ecah {
namespace decode {

constexpr int kT = 128;
constexpr int kW = kT / 32;

struct Params {
  const void* q;
  void* out;
  float* lse;
  const int* last_page_len;
  long long q_tok, q_head, o_tok, o_head;
  int hq, group;
  float scale;               // sm_scale * log2 e
  kv::Cache cache;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

template <int DT, bool E4M3>
__device__ __forceinline__ float load_elem(const void* base, long long at) {
  if (E4M3) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<const __nv_fp8_storage_t*>(base)[at], __NV_E4M3);
    return __half2float(__half(h));
  }
  return DType<DT>::to_f32(static_cast<const uint16_t*>(base)[at]);
}

// One CTA per request and query head; warp w takes the keys w, w + 4, ... with
// a running maximum and sum, and the warps are joined at the end.
template <int DT, bool E4M3, int D>
__global__ void __launch_bounds__(kT) decode_kernel(const Params P) {
  constexpr int E = D / 32;
  __shared__ float sm[kW], sl[kW], so[kW][D];
  const int b = blockIdx.x, hq = blockIdx.y, h = hq / P.group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long first, count;
  kv::page_range(P.cache, b, &first, &count);
  const int ps = P.cache.page_size;
  const long long len = count > 0 && P.cache.num_pages > 0
                            ? (count - 1) * ps + min(max(P.last_page_len[b], 0), ps) : 0;
  const uint16_t* q = static_cast<const uint16_t*>(P.q) + b * P.q_tok + hq * P.q_head;
  float qv[E], acc[E];
  for (int e = 0; e < E; ++e) { qv[e] = DType<DT>::to_f32(q[lane + 32 * e]); acc[e] = 0.0f; }
  float m = -INFINITY, l = 0.0f;
  for (long long j = warp; j < len; j += kW) {
    const long long page = min(max(P.cache.indices[first + j / ps], 0), P.cache.num_pages - 1);
    const int slot = static_cast<int>(j % ps);
    const long long sat = (page * P.cache.heads + h) * ps + slot;
    const long long ka = page * P.cache.k.page + slot * P.cache.k.slot + h * P.cache.k.head;
    const long long va = page * P.cache.v.page + slot * P.cache.v.slot + h * P.cache.v.head;
    float s = 0.0f;
    for (int e = 0; e < E; ++e) s = fmaf(qv[e], load_elem<DT, E4M3>(P.cache.k.base, ka + lane + 32 * e), s);
    s = warp_sum(s) * P.scale;
    if (E4M3) s *= P.cache.k.scale[sat];
    const float mn = s == -INFINITY ? m : fmaxf(m, s);
    const float p = s == -INFINITY ? 0.0f : exp2f(s - mn), f = m == mn ? 1.0f : exp2f(m - mn);
    const float pv = E4M3 ? p * P.cache.v.scale[sat] : p;
    l = fmaf(l, f, p);
    for (int e = 0; e < E; ++e)
      acc[e] = fmaf(pv, load_elem<DT, E4M3>(P.cache.v.base, va + lane + 32 * e), acc[e] * f);
    m = mn;
  }
  if (lane == 0) { sm[warp] = m; sl[warp] = l; }
  for (int e = 0; e < E; ++e) so[warp][lane + 32 * e] = acc[e];
  __syncthreads();
  float M = sm[0];
  for (int w = 1; w < kW; ++w) M = fmaxf(M, sm[w]);
  float L = 0.0f, f[kW];
  for (int w = 0; w < kW; ++w) {
    f[w] = sm[w] == -INFINITY ? 0.0f : exp2f(sm[w] - M);
    L = fmaf(sl[w], f[w], L);
  }
  uint16_t* o = static_cast<uint16_t*>(P.out) + b * P.o_tok + hq * P.o_head;
  for (int d = threadIdx.x; d < D; d += kT) {
    float v = 0.0f;
    for (int w = 0; w < kW; ++w) v = fmaf(so[w][d], f[w], v);
    o[d] = DType<DT>::to_raw(L == 0.0f ? 0.0f : v / L);
  }
  if (threadIdx.x == 0 && P.lse)
    P.lse[static_cast<long long>(b) * P.hq + hq] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

template <int DT, bool E4M3>
static auto kernel_for(int D) {
  switch (D) {
    case 64: return decode_kernel<DT, E4M3, 64>;
    case 96: return decode_kernel<DT, E4M3, 96>;
    case 128: return decode_kernel<DT, E4M3, 128>;
    case 192: return decode_kernel<DT, E4M3, 192>;
    default: return decode_kernel<DT, E4M3, 256>;
  }
}

}  // namespace decode
}  // namespace ecah

using namespace ecah;

extern "C" {

size_t ecah_paged_decode_workspace_bytes(int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim) {
  if (batch < 0 || num_kv_heads < 1 || num_qo_heads < 1 || num_qo_heads % num_kv_heads || !kv::head_dim_ok(head_dim) ||
      device_sms() <= 0)
    return 0;
  return 256;
}

int ecah_paged_decode(const ecah_decode_args* a, void* stream) {
  if (!a) return ECAH_ERR_NULL;
  if (a->abi_version != ECAH_SAMPLER_ABI_VERSION) return ECAH_ERR_ABI;
  const int st = kv::check_cache(a->cache, a->dtype);
  if (st != ECAH_OK) return st;
  const ecah_kv_cache& c = a->cache;
  if (a->num_qo_heads < 1 || a->num_qo_heads % c.num_kv_heads || !(a->sm_scale > 0.0f)) return ECAH_ERR_SHAPE;
  for (long long s : {a->q_token_stride, a->q_head_stride, a->out_token_stride, a->out_head_stride})
    if (s < 0 || s % 8) return ECAH_ERR_SHAPE;
  if (c.batch == 0) return ECAH_OK;
  if (!a->q || !a->out || !a->kv_last_page_len) return ECAH_ERR_NULL;
  if (!kv::aligned16(a->q) || !kv::aligned16(a->out)) return ECAH_ERR_SHAPE;
  if (!a->workspace || a->workspace_bytes < ecah_paged_decode_workspace_bytes(c.batch, a->num_qo_heads, c.num_kv_heads, c.head_dim))
    return ECAH_ERR_WORKSPACE;
  decode::Params P = {};
  P.q = a->q; P.out = a->out; P.lse = a->lse; P.last_page_len = a->kv_last_page_len;
  P.q_tok = a->q_token_stride; P.q_head = a->q_head_stride;
  P.o_tok = a->out_token_stride; P.o_head = a->out_head_stride;
  P.hq = a->num_qo_heads; P.group = a->num_qo_heads / c.num_kv_heads;
  P.scale = a->sm_scale * kLog2e;
  P.cache = kv::make_cache(c);
  const bool e4m3 = c.kv_dtype == ECAH_KV_E4M3, f16 = a->dtype == ECAH_DTYPE_F16;
  auto fn = f16 ? (e4m3 ? decode::kernel_for<ECAH_DTYPE_F16, true>(c.head_dim) : decode::kernel_for<ECAH_DTYPE_F16, false>(c.head_dim))
                : (e4m3 ? decode::kernel_for<ECAH_DTYPE_BF16, true>(c.head_dim) : decode::kernel_for<ECAH_DTYPE_BF16, false>(c.head_dim));
  if (a->num_qo_heads > 65535) return ECAH_ERR_SHAPE;
  return launch_kernel(fn, dim3(c.batch, a->num_qo_heads), decode::kT, 0, reinterpret_cast<cudaStream_t>(stream), P)
             ? ECAH_OK : ECAH_ERR_LAUNCH;
}

}  // extern "C"
