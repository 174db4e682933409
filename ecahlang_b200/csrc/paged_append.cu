// Norm, rotation and cache write of new tokens: ecah_paged_append (contract
// in include/ecah_sampler.h).

#include "host_util.h"
#include "paged.cuh"

namespace ecah {
namespace append {

// The mathematics is elementwise but for two sums over a head: the mean square of
// the norm and the largest magnitude of an e4m3 row.
//
// Bound: HBM; every value is read once and written once (4 bytes for 16-bit
// caches), about 8 instructions a value against the 22 that the bandwidth leaves.
//
// Split: a head vector is held by D / 16 lanes of a group of 4, 8 or 16, 16 values a
// lane in two 16-byte loads, placed so that both members of every rotated pair are
// in one lane: 8 values of each half of the head, or 16 neighbours where pairs are
// interleaved.  A warp holds several heads of one token and, with many tokens, goes
// through kMany heads a group with all their loads in flight and one reading of the
// token's table row; with few tokens one head a group spreads over more warps.
//
// Measured on one B200, device time of graph replays: 8192 tokens of 32/8 heads of
// 128 with norm and rotation into a bf16 cache 37.8 us (5.4 TB/s), into an e4m3 cache
// 42.9 us (4.3 TB/s), 128 tokens into an e4m3 cache 3.4 us, one token 2.1 us (a launch).

constexpr int kT = 64;               // 8192 tokens: 37.5 us, with 128 threads 37.8, with 256 39.3
constexpr int kMany = 2;             // with 4 38.7 us, with 6 43.2

struct Params {
  const void *q, *k, *v;
  void* q_out;
  const void *q_norm, *k_norm;
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head, qo_tok, qo_head;
  const float* cos_sin;
  const int* positions;
  const int* batch_index;
  int tokens, hq, table_rows, interleaved;
  int warps_per_token;
  float eps;
  kv::Cache cache;
};

// keeps a NaN, so that its row's scale is one
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <int DT>
__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = DType<DT>::to_f32(w[i] & 0xFFFFu);
    x[2 * i + 1] = DType<DT>::to_f32(w[i] >> 16);
  }
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (DT == ECAH_DTYPE_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// eight values to e4m3 codes, rounded to nearest even
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    asm("{ .reg .b16 l, h; cvt.rn.satfinite.e4m3x2.f32 l, %2, %1; cvt.rn.satfinite.e4m3x2.f32 h, %4, %3; mov.b32 %0, {l, h}; }"
        : "=r"(w[i]) : "f"(x[4 * i] * inv), "f"(x[4 * i + 1] * inv), "f"(x[4 * i + 2] * inv), "f"(x[4 * i + 3] * inv));
  return make_uint2(w[0], w[1]);
}

template <int DT, bool E4M3, int D, int ITERS>
__global__ void __launch_bounds__(kT) append_kernel(const Params P) {
  grid_start();
  constexpr int kLanes = D / 16;                                     // of a head
  constexpr int kGroup = kLanes <= 4 ? 4 : kLanes <= 8 ? 8 : 16;     // lanes set aside for it
  constexpr int kGroups = 32 / kGroup;
  const int lane = threadIdx.x & 31, l = lane % kGroup, g = lane / kGroup;
  const long long id = static_cast<long long>(blockIdx.x) * (kT / 32) + (threadIdx.x >> 5);
  const int t = static_cast<int>(id / P.warps_per_token);
  if (t >= P.tokens) return;
  const int first = static_cast<int>(id % P.warps_per_token) * kGroups * ITERS + g;
  const int hk = P.cache.heads, heads = P.hq + 2 * hk;
  const bool on = l < kLanes;
  const int lo = P.interleaved ? 16 * l : 8 * l, hi = P.interleaved ? lo + 8 : lo + D / 2;

  // the vectors, all in flight
  uint4 raw[ITERS][2];
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    const int hh = first + i * kGroups;
    if (on && hh < heads) {
      const uint16_t* x = hh < P.hq        ? static_cast<const uint16_t*>(P.q) + t * P.q_tok + hh * P.q_head
                          : hh < P.hq + hk ? static_cast<const uint16_t*>(P.k) + t * P.k_tok + (hh - P.hq) * P.k_head
                                           : static_cast<const uint16_t*>(P.v) + t * P.v_tok + (hh - P.hq - hk) * P.v_head;
      raw[i][0] = *reinterpret_cast<const uint4*>(x + lo);
      raw[i][1] = *reinterpret_cast<const uint4*>(x + hi);
    } else {
      raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
    }
  }
  const int pos = P.positions[t];
  // the cache slot of the token: none when it has no place
  long long page = -1;
  int slot = 0;
  if (first - g + kGroups * ITERS > P.hq) {                          // this warp holds keys or values
    const int req = P.batch_index[t];
    if (req >= 0 && req < P.cache.batch && pos >= 0) {
      long long at, count;
      kv::page_range(P.cache, req, &at, &count);
      const int nth = pos / P.cache.page_size;
      slot = pos - nth * P.cache.page_size;
      if (nth < count) {
        page = P.cache.indices[at + nth];
        if (page >= P.cache.num_pages) page = -1;
      }
    }
  }
  alignas(16) float c[8], s[8];
  const bool rotate = P.cos_sin != nullptr;
  if (rotate && on && first < P.hq + hk) {
    const float* cs = P.cos_sin + static_cast<long long>(min(max(pos, 0), P.table_rows - 1)) * D + 8 * l;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<float4*>(c + 4 * i) = *reinterpret_cast<const float4*>(cs + 4 * i);
      *reinterpret_cast<float4*>(s + 4 * i) = *reinterpret_cast<const float4*>(cs + D / 2 + 4 * i);
    }
  }

#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    const int hh = first + i * kGroups;
    const bool is_q = hh < P.hq, is_v = hh >= P.hq + hk;
    float a[8], b[8];
    unpack8<DT>(raw[i][0], a);
    unpack8<DT>(raw[i][1], b);
    const uint16_t* w = static_cast<const uint16_t*>(is_q ? P.q_norm : is_v ? nullptr : P.k_norm);
    // the warp's lanes take these sums together, whatever their heads need of them
    if (P.q_norm || P.k_norm) {
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(a[j], a[j], fmaf(b[j], b[j], ss));
#pragma unroll
      for (int o = kGroup / 2; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
      if (w && on) {
        const float inv = rsqrtf(ss / static_cast<float>(D) + P.eps);
        float wa[8], wb[8];
        unpack8<DT>(*reinterpret_cast<const uint4*>(w + lo), wa);
        unpack8<DT>(*reinterpret_cast<const uint4*>(w + hi), wb);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          a[j] *= inv * wa[j];
          b[j] *= inv * wb[j];
        }
      }
    }
    if (rotate && !is_v && on) {
      if (P.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float u = a[2 * j], v = a[2 * j + 1], x = b[2 * j], y = b[2 * j + 1];
          a[2 * j] = fmaf(u, c[j], -(v * s[j]));
          a[2 * j + 1] = fmaf(v, c[j], u * s[j]);
          b[2 * j] = fmaf(x, c[j + 4], -(y * s[j + 4]));
          b[2 * j + 1] = fmaf(y, c[j + 4], x * s[j + 4]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float u = a[j], v = b[j];
          a[j] = fmaf(u, c[j], -(v * s[j]));
          b[j] = fmaf(v, c[j], u * s[j]);
        }
      }
    }
    float scale = 1.0f;
    if (E4M3) {
      float big = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) big = max_nan(big, max_nan(fabsf(a[j]), fabsf(b[j])));
#pragma unroll
      for (int o = kGroup / 2; o; o >>= 1) big = max_nan(big, __shfl_xor_sync(0xFFFFFFFFu, big, o));
      scale = max_nan(big, 448e-12f) / 448.0f;
    }
    if (!on || hh >= heads) continue;
    if (is_q) {
      uint16_t* o = static_cast<uint16_t*>(P.q_out) + t * P.qo_tok + hh * P.qo_head;
      *reinterpret_cast<uint4*>(o + lo) = pack8<DT>(a);
      *reinterpret_cast<uint4*>(o + hi) = pack8<DT>(b);
    } else if (page >= 0) {
      const kv::Side& side = is_v ? P.cache.v : P.cache.k;
      const int h = is_v ? hh - P.hq - hk : hh - P.hq;
      const long long at = page * side.page + slot * side.slot + h * side.head;
      if (!E4M3) {
        uint16_t* o = static_cast<uint16_t*>(side.base) + at;
        *reinterpret_cast<uint4*>(o + lo) = pack8<DT>(a);
        *reinterpret_cast<uint4*>(o + hi) = pack8<DT>(b);
      } else {
        if (l == 0) side.scale[(page * hk + h) * P.cache.page_size + slot] = scale;
        const float inv = 1.0f / scale;
        uint8_t* o = static_cast<uint8_t*>(side.base) + at;
        *reinterpret_cast<uint2*>(o + lo) = codes8(a, inv);
        *reinterpret_cast<uint2*>(o + hi) = codes8(b, inv);
      }
    }
  }
}

using KernelFn = void (*)(const Params);

template <int DT, bool E4M3, int ITERS>
static KernelFn kernel_for(int D) {
  switch (D) {
    case 64: return append_kernel<DT, E4M3, 64, ITERS>;
    case 96: return append_kernel<DT, E4M3, 96, ITERS>;
    case 128: return append_kernel<DT, E4M3, 128, ITERS>;
    case 192: return append_kernel<DT, E4M3, 192, ITERS>;
    default: return append_kernel<DT, E4M3, 256, ITERS>;
  }
}

template <int DT>
static KernelFn kernel_for(int D, bool e4m3, bool many) {
  return e4m3 ? (many ? kernel_for<DT, true, kMany>(D) : kernel_for<DT, true, 1>(D))
              : (many ? kernel_for<DT, false, kMany>(D) : kernel_for<DT, false, 1>(D));
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
    if (!aligned16(p)) return ECAH_ERR_SHAPE;
  append::Params P = {};
  P.q = a->q; P.k = a->k; P.v = a->v; P.q_out = a->q_out;
  P.q_norm = a->q_norm; P.k_norm = a->k_norm;
  P.q_tok = a->q_token_stride; P.q_head = a->q_head_stride;
  P.k_tok = a->k_token_stride; P.k_head = a->k_head_stride;
  P.v_tok = a->v_token_stride; P.v_head = a->v_head_stride;
  P.qo_tok = a->qo_token_stride; P.qo_head = a->qo_head_stride;
  P.cos_sin = a->cos_sin;
  P.positions = a->positions; P.batch_index = a->batch_index;
  P.tokens = a->tokens; P.hq = a->q ? a->num_qo_heads : 0;
  P.table_rows = a->table_rows; P.interleaved = a->interleaved;
  P.eps = a->eps;
  P.cache = kv::make_cache(a->cache);
  const int sms = device_sms();
  if (sms <= 0) return ECAH_ERR_LAUNCH;
  const int D = a->cache.head_dim, group = D <= 64 ? 4 : D <= 128 ? 8 : 16, groups = 32 / group;
  const long long heads = P.hq + 2ll * P.cache.heads;
  // kMany heads a group once one head a group would be more than a full wave of
  // 32 warps an SM.
  const bool many = P.tokens * ((heads + groups - 1) / groups) > 32ll * sms;
  const long long step = static_cast<long long>(groups) * (many ? append::kMany : 1);
  const long long per_token = (heads + step - 1) / step;
  const long long blocks = (P.tokens * per_token + append::kT / 32 - 1) / (append::kT / 32);
  if (heads > 0x7FFFFFFF || blocks > 0x7FFFFFFF) return ECAH_ERR_SHAPE;
  P.warps_per_token = static_cast<int>(per_token);
  const bool e4m3 = a->cache.kv_dtype == ECAH_KV_E4M3;
  const append::KernelFn fn = a->dtype == ECAH_DTYPE_F16 ? append::kernel_for<ECAH_DTYPE_F16>(D, e4m3, many)
                                                         : append::kernel_for<ECAH_DTYPE_BF16>(D, e4m3, many);
  return launch_kernel(fn, dim3(static_cast<unsigned>(blocks)), append::kT, 0, reinterpret_cast<cudaStream_t>(stream), P)
             ? ECAH_OK : ECAH_ERR_LAUNCH;
}
