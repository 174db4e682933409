// Token log probabilities, entropy and most likely alternatives of logits
// rows: ecah_token_logprobs (contract in include/ecah_sampler.h).

#include "common.cuh"
#include "host_util.h"

namespace ecah {
namespace lp {

constexpr int kT = 256;
constexpr int kW = kT / 32;

struct Params {
  const void* logits;
  long long row_stride;
  const int* row_index;
  int logit_rows, R, V, K, N;
  const int* token_ids;
  const float* temperature;
  float* logprobs;
  float* entropy;
  int* top_ids;
  float* top_logprobs;
};

// Order of the alternatives: value descending, then index ascending, as one
// 64-bit key (larger is earlier).  -0 counts as +0, as a comparison would.
__device__ __forceinline__ unsigned long long order_key(float x, unsigned idx) {
  return (static_cast<unsigned long long>(key32(x == 0.0f ? 0.0f : x)) << 32) | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ float order_value(unsigned long long k) { return unkey32(static_cast<uint32_t>(k >> 32)); }
__device__ __forceinline__ int order_index(unsigned long long k) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(k)); }

__device__ __forceinline__ float block_sum(float v, float* s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int w = 0; w < kW; ++w) v += s[w];
  return v;
}

__device__ __forceinline__ unsigned long long block_max(unsigned long long v, unsigned long long* s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const unsigned long long u = __shfl_xor_sync(0xFFFFFFFFu, v, o);
    v = u > v ? u : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
  for (int w = 1; w < kW; ++w) v = s[w] > v ? s[w] : v;
  return v;
}

// One CTA per row: a pass for the maximum, one for the sums, one for each
// alternative.
template <int DT>
__global__ void __launch_bounds__(kT) token_logprobs_kernel(const Params P) {
  using D = DType<DT>;
  __shared__ float sf[kW];
  __shared__ unsigned long long su[kW];
  const int r = blockIdx.x, tid = threadIdx.x;
  long long row = r;
  if (P.row_index) row = min(max(P.row_index[r], 0), P.logit_rows - 1);
  const typename D::Raw* x = static_cast<const typename D::Raw*>(P.logits) + row * P.row_stride;
  const float T = P.temperature ? P.temperature[r] : 1.0f;

  unsigned long long best = 0;
  int bad = 0;
  for (int i = tid; i < P.V; i += kT) {
    const float v = D::to_f32(x[i]);
    if (!(v < INFINITY)) bad = 1;
    const unsigned long long k = order_key(v, i);
    best = k > best ? k : best;
  }
  bad = __syncthreads_or(bad);
  best = block_max(best, su);
  const float m = order_value(best);
  const int arg = order_index(best);
  const bool empty = !bad && m == -INFINITY, greedy = T <= 0.0f;

  float z = 0.0f, s = 0.0f;
  if (!bad && !empty) {
    const float c = kLog2e / T;
    for (int i = tid; i < P.V; i += kT) {
      const float v = D::to_f32(x[i]);
      if (v == -INFINITY) continue;
      const float t = (v - m) * c, e = ex2_approx(t);
      z += e;
      s = fmaf(e, fmaxf(t, -150.0f), s);
    }
  }
  z = block_sum(z, sf);
  s = block_sum(s, sf);
  const float lz = logf(z);
  auto logprob = [&](float v, int i) -> float {
    if (bad) return NAN;
    if (empty || v == -INFINITY) return -INFINITY;
    if (greedy) return i == arg ? 0.0f : -INFINITY;
    // halved, so that the difference of two values of opposite sign near the type's largest stays finite
    return (0.5f * v - 0.5f * m) / (0.5f * T) - lz;
  };
  if (tid == 0 && P.entropy)
    P.entropy[r] = bad ? NAN : (empty || greedy) ? 0.0f : lz - s / z * 0.6931471805599453f;
  for (int j = tid; j < P.K; j += kT) {
    const long long at = static_cast<long long>(r) * P.K + j;
    const int t = P.token_ids[at];
    P.logprobs[at] = (t < 0 || t >= P.V) ? NAN : logprob(D::to_f32(x[t]), t);
  }
  unsigned long long below = ~0ull;
  for (int n = 0; n < P.N; ++n) {
    unsigned long long k = 0;
    if (!bad)
      for (int i = tid; i < P.V; i += kT) {
        const float v = D::to_f32(x[i]);
        const unsigned long long u = order_key(v, i);
        if (v > -INFINITY && u < below && u > k) k = u;
      }
    k = block_max(k, su);
    if (tid == 0) {
      const long long at = static_cast<long long>(r) * P.N + n;
      P.top_ids[at] = k ? order_index(k) : -1;
      P.top_logprobs[at] = k ? logprob(order_value(k), order_index(k)) : bad ? NAN : -INFINITY;
    }
    below = k;
  }
}

}  // namespace lp
}  // namespace ecah

using namespace ecah;

extern "C" {

size_t ecah_token_logprobs_workspace_bytes(void) { return device_sms() > 0 ? 256 : 0; }

int ecah_token_logprobs(const ecah_logprob_args* a, void* stream) {
  if (!a) return ECAH_ERR_NULL;
  if (a->abi_version != ECAH_SAMPLER_ABI_VERSION) return ECAH_ERR_ABI;
  if (a->dtype < ECAH_DTYPE_F16 || a->dtype > ECAH_DTYPE_F32) return ECAH_ERR_DTYPE;
  if (a->rows < 0 || a->vocab < 1 || a->vocab > 0x7FFFFFFF - 65536 || a->row_stride < a->vocab || a->tokens_per_row < 0 ||
      a->top_n < 0 || a->top_n > ECAH_MAX_TOP_N || (a->row_index && a->logit_rows < 1))
    return ECAH_ERR_SHAPE;
  if (a->rows == 0) return ECAH_OK;
  if (!a->logits || (a->tokens_per_row && (!a->token_ids || !a->logprobs)) ||
      (a->top_n && (!a->top_ids || !a->top_logprobs)))
    return ECAH_ERR_NULL;
  if (!a->workspace || a->workspace_bytes < ecah_token_logprobs_workspace_bytes()) return ECAH_ERR_WORKSPACE;
  lp::Params P = {};
  P.logits = a->logits;
  P.row_stride = a->row_stride;
  P.row_index = a->row_index;
  P.logit_rows = a->logit_rows;
  P.R = a->rows;
  P.V = a->vocab;
  P.K = a->tokens_per_row;
  P.N = a->top_n;
  P.token_ids = a->token_ids;
  P.temperature = a->temperature;
  P.logprobs = a->logprobs;
  P.entropy = a->entropy;
  P.top_ids = a->top_ids;
  P.top_logprobs = a->top_logprobs;
  auto fn = a->dtype == ECAH_DTYPE_F16 ? lp::token_logprobs_kernel<ECAH_DTYPE_F16>
            : a->dtype == ECAH_DTYPE_BF16 ? lp::token_logprobs_kernel<ECAH_DTYPE_BF16>
                                          : lp::token_logprobs_kernel<ECAH_DTYPE_F32>;
  return launch_kernel(fn, dim3(P.R), lp::kT, 0, reinterpret_cast<cudaStream_t>(stream), P) ? ECAH_OK : ECAH_ERR_LAUNCH;
}

}  // extern "C"
