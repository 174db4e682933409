// Verification of drafted tokens: ecah_verify_drafts (contract in
// include/ecah_sampler.h).

#include <algorithm>

#include "host_util.h"
#include "common.cuh"

namespace ecah {
namespace drafts {

// The mathematics: the tests u q(x) < p(x) of a request's drafts name the row k where
// it stops; the token there is drawn by inverting the cumulative sum of
// r = max(p_k - q_k, 0) (or p_k) over the vocabulary at u_N.  Sums are float64: a
// float32 sum over 10^5 entries would move the drawn entry in about one draw in 10^3.
//
// Bound: HBM; only the rows at k are read, 4 to 8 bytes an entry, each once.
//
// Split: a request's row is divided over a row of blocks and each block's range over
// its warps; a warp's sum goes to the workspace.  Every block finds k by itself (a few
// dependent loads).  The block that arrives last takes the prefix sums of the warps'
// sums in vocabulary order, and reads the one range again in which the target lies.  No
// result depends on which block that is.
//
// Measured on one B200, passes through the Python entry point one after another: 64
// requests of 5 drafts over 151 936 float32 entries 19 us (4.1 TB/s; floor 11.9), 128
// requests of up to 8 looked-up drafts over 32 003 bf16 entries 10.0 (9.8 on the device), one
// request of 4 drafts 7.1 (6.0 on the device).  What bounds them: about 8 us of dependent reads
// (drafts, probabilities, the row, the sums, the range again), from cold rows.  With twice the
// blocks the batch took 2 us more, with half as many 6; without 4 loads a row in flight 10.

constexpr int kT = 256;
constexpr int kW = kT / 32;
constexpr int kMaxChunks = 128;              // blocks to a request
constexpr int kParts = kMaxChunks * kW;
constexpr int kRecord = 256 + kParts * 8;    // workspace of a request: its counter, its sums
constexpr int kRange = 256;                  // entries of a warp's range at the least
constexpr int kWave = 4;                     // blocks to an SM

struct Params {
  const void *target, *draft;
  long long t_batch, t_row, d_batch, d_row;
  const int *ids, *num;
  const float* u;
  int *tokens, *accepted;
  unsigned char* workspace;
  int N, V, chunks, range;                   // range: entries of a warp, a multiple of 8
};

template <int DT> struct Vec {               // 16 bytes of probabilities
  static constexpr int kN = DType<DT>::kVec;
  uint4 v;
  __device__ __forceinline__ void load(const void* p) { v = *static_cast<const uint4*>(p); }
  __device__ __forceinline__ float operator[](int i) const {
    const int at = kN == 4 ? i : i / 2;
    const uint32_t w = at == 0 ? v.x : at == 1 ? v.y : at == 2 ? v.z : v.w;
    return DType<DT>::to_f32(kN == 4 ? w : i & 1 ? w >> 16 : w & 0xFFFFu);
  }
};

template <int DT>
__device__ __forceinline__ float one(const void* row, long long i) {
  using Raw = typename DType<DT>::Raw;
  return DType<DT>::to_f32(static_cast<const Raw*>(row)[i]);
}

// The larger of a difference and zero; a NaN stays one.
__device__ __forceinline__ float positive(float a) {
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(a));
  return r;
}

// The row that a request's token is drawn from.
template <int DT>
struct Row {
  const void *p, *q;                         // q: subtracted, or NULL
  int out;                                   // entry left out (a certain draft that was refused), or -1
  static constexpr int kN = Vec<DT>::kN, kSize = 16 / kN;
  __device__ __forceinline__ float mass(long long i) const {
    const float x = one<DT>(p, i);
    const float m = positive(q ? x - one<DT>(q, i) : x);
    return i == out ? 0.0f : m;
  }
  // Sum of the warp's entries [lo, hi), in every lane: 16 bytes a load from the first
  // 16-byte boundary on, where both rows have theirs at the same entries.
  __device__ __forceinline__ double sum(long long lo, long long hi) const {
    const int lane = threadIdx.x & 31;
    double s = 0.0, t = 0.0;                 // two chains
    long long i = lo;
    const unsigned off = static_cast<unsigned>(reinterpret_cast<uintptr_t>(p) + lo * kSize) & 15u;
    if (!q || ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(q)) & 15) == 0) {
      const int head = static_cast<int>((16u - off) & 15u) / kSize;
      if (lane < head && lo + lane < hi) s = mass(lo + lane);
      i += head;
      const char *a = static_cast<const char*>(p), *b = static_cast<const char*>(q);
      auto add = [&](const Vec<DT>& x, const Vec<DT>& y, long long at) {
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          const float m = positive(q ? x[j] - y[j] : x[j]);
          (j & 1 ? t : s) += at + j == out ? 0.0f : m;
        }
      };
      constexpr int kFlight = 4;             // loads of a row in flight
      for (; i + 32 * kN * kFlight <= hi; i += 32 * kN * kFlight) {
        Vec<DT> x[kFlight], y[kFlight];
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
          const long long at = i + (u * 32 + lane) * kN;
          x[u].load(a + at * kSize);
          if (q) y[u].load(b + at * kSize);
        }
#pragma unroll
        for (int u = 0; u < kFlight; ++u) add(x[u], y[u], i + (u * 32 + lane) * kN);
      }
      Vec<DT> x[kFlight], y[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {    // the rest, ended lane by lane
        const long long at = i + (u * 32 + lane) * kN;
        if (at + kN <= hi) {
          x[u].load(a + at * kSize);
          if (q) y[u].load(b + at * kSize);
        }
      }
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        const long long at = i + (u * 32 + lane) * kN;
        if (at + kN <= hi) add(x[u], y[u], at);
      }
      i = max(i, hi - (hi - min(i, hi)) % kN);               // what is no whole vector
      if (i + lane < hi) t += mass(i + lane);
    } else {
#pragma unroll 8
      for (i += lane; i < hi; i += 32) s += mass(i);
    }
    s += t;
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    return s;
  }
};

// Inclusive sum of the block's doubles in thread order; `total` is everybody's.
__device__ __forceinline__ double scan(double v, double* total, double* s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double w = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += w;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  double before = 0.0, all = 0.0;
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    if (w < warp) before += s_warp[w];
    all += s_warp[w];
  }
  *total = all;
  return before + v;
}

struct Shared {
  double warp[kW];
  double base;                               // mass before the part that holds the target
  int part, last, found, flag;
};

// The entry whose cumulative mass first exceeds u times the whole, from the sums of
// `parts` ranges of `range` entries; -1 where the whole is not positive and finite.
template <int DT, typename Sums>
__device__ int pick(const Row<DT>& row, const Params& P, float u, Sums sum_of, int parts, long long range, Shared& S, double* whole) {
  const int tid = threadIdx.x;
  constexpr int kOwn = kParts / kT;
  if (tid == 0) { S.part = 0x7FFFFFFF; S.last = -1; S.found = 0x7FFFFFFF; }
  double own[kOwn], mine = 0.0, total;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    own[i] = tid * kOwn + i < parts ? sum_of(tid * kOwn + i) : 0.0;
    mine += own[i];
  }
  double at = scan(mine, &total, S.warp) - mine;
  *whole = total;
  if (!(total > 0.0) || total == INFINITY) return -1;
  const double target = static_cast<double>(u) * total;
  for (int i = 0; i < kOwn; ++i) {           // the first part that passes the target; without one the last with mass
    if (own[i] > 0.0) atomicMax(&S.last, tid * kOwn + i);
    if (at + own[i] > target) atomicMin(&S.part, tid * kOwn + i);
    at += own[i];
  }
  __syncthreads();
  const int part = S.part < parts ? S.part : S.last;
  at -= mine;
  for (int i = 0; i < kOwn; ++i) {
    if (tid * kOwn + i == part) S.base = at;
    at += own[i];
  }
  __syncthreads();
  if (tid == 0) S.last = -1;
  double base = S.base;
  __syncthreads();
  const long long lo = part * range, hi = min(lo + range, static_cast<long long>(P.V));
  constexpr int kEach = 4;
  for (long long b0 = lo; b0 < hi; b0 += kT * kEach) {
    float m[kEach];
    double sum = 0.0, all;
    int top = -1;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const long long i = b0 + tid * kEach + j;
      m[j] = i < hi ? row.mass(i) : 0.0f;
      sum += m[j];
      if (m[j] > 0.0f) top = static_cast<int>(i);
    }
    double c = scan(sum, &all, S.warp) - sum + base;
    if (top >= 0) atomicMax(&S.last, top);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      c += m[j];
      if (m[j] > 0.0f && c > target) atomicMin(&S.found, static_cast<int>(b0) + tid * kEach + j);
    }
    base += all;
    __syncthreads();
    if (S.found != 0x7FFFFFFF) break;
  }
  return S.found != 0x7FFFFFFF ? S.found : S.last;   // rounding may leave the target above the part's own sum
}

template <int DT>
__global__ void __launch_bounds__(kT, kWave) verify_kernel(const Params P) {
  grid_start();
  __shared__ Shared S;
  __shared__ int s_stop;
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = P.num ? min(P.num[b], P.N) : P.N;
  int* tokens = P.tokens + static_cast<long long>(b) * (P.N + 1);
  if (n < 0) {                                       // a padding row
    if (blockIdx.x == 0) {
      for (int j = tid; j <= P.N; j += kT) tokens[j] = -1;
      if (tid == 0) P.accepted[b] = 0;
    }
    return;
  }
  using Raw = typename DType<DT>::Raw;
  const Raw* target = static_cast<const Raw*>(P.target) + b * P.t_batch;
  const Raw* draft = P.draft ? static_cast<const Raw*>(P.draft) + b * P.d_batch : nullptr;
  const int* ids = P.ids + static_cast<long long>(b) * P.N;
  const float* u = P.u + static_cast<long long>(b) * (P.N + 1);
  if (warp == 0) {
    int stop = n;
    for (int j0 = 0; j0 < n; j0 += 32) {
      const int j = j0 + lane;
      bool kept = true;
      if (j < n) {
        const int x = ids[j];
        kept = x >= 0 && x < P.V;
        if (kept) {
          const float p = one<DT>(target + j * P.t_row, x), q = draft ? one<DT>(draft + j * P.d_row, x) : 1.0f;
          kept = static_cast<double>(u[j]) * static_cast<double>(q) < static_cast<double>(p);   // exact products
        }
      }
      const unsigned refused = __ballot_sync(0xFFFFFFFFu, !kept);
      if (refused) { stop = j0 + __ffs(refused) - 1; break; }
    }
    if (lane == 0) s_stop = stop;
  }
  __syncthreads();
  const int k = s_stop;
  Row<DT> row;
  row.p = target + k * P.t_row;
  row.q = k < n && draft ? draft + k * P.d_row : nullptr;
  row.out = k < n && !draft ? ids[k] : -1;

  unsigned char* record = P.workspace + static_cast<long long>(b) * kRecord;
  double* sums = reinterpret_cast<double*>(record + 256);
  const int part = blockIdx.x * kW + warp;
  const long long lo = static_cast<long long>(part) * P.range;
  const double s = row.sum(lo, min(lo + P.range, static_cast<long long>(P.V)));
  if (lane == 0) {
    sums[part] = s;
    __threadfence();
  }
  __syncthreads();
  if (tid == 0) {
    unsigned arrived;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(arrived) : "l"(record) : "memory");
    S.flag = arrived + 1u == static_cast<unsigned>(P.chunks);
    if (S.flag) *reinterpret_cast<unsigned*>(record) = 0u;
  }
  __syncthreads();
  if (!S.flag) return;

  double whole;
  int token = pick<DT>(row, P, u[P.N], [&](int i) { return __ldcg(sums + i); }, P.chunks * kW, P.range, S, &whole);
  if (whole == 0.0 && (row.q || row.out >= 0)) {     // nothing left of the target: it is drawn from as it is
    __syncthreads();
    row.q = nullptr;
    row.out = -1;
    const long long range = (static_cast<long long>(P.V) + 8 * kW - 1) / (8 * kW) * 8;
    __shared__ double s_sum[kW];
    const double mine = row.sum(warp * range, min((warp + 1) * range, static_cast<long long>(P.V)));
    if (lane == 0) s_sum[warp] = mine;
    __syncthreads();
    token = pick<DT>(row, P, u[P.N], [&](int i) { return s_sum[i]; }, kW, range, S, &whole);
  }
  for (int j = tid; j <= P.N; j += kT) tokens[j] = j < k ? ids[j] : j == k ? token : -1;
  if (tid == 0) P.accepted[b] = k;
}

}  // namespace drafts
}  // namespace ecah

using namespace ecah;

extern "C" {

size_t ecah_verify_drafts_workspace_bytes(int32_t batch) {
  return batch < 0 ? 0 : static_cast<size_t>(std::max(batch, 1)) * drafts::kRecord;
}

int ecah_verify_drafts(const ecah_verify_args* a, void* stream) {
  if (!a) return ECAH_ERR_NULL;
  if (a->abi_version != ECAH_SAMPLER_ABI_VERSION) return ECAH_ERR_ABI;
  if (a->dtype != ECAH_DTYPE_F16 && a->dtype != ECAH_DTYPE_BF16 && a->dtype != ECAH_DTYPE_F32) return ECAH_ERR_DTYPE;
  if (a->batch < 0 || a->batch > 65535 || a->drafts < 0 || a->drafts == 0x7FFFFFFF || a->vocab < 1 || a->vocab > 0x7FFFFFFF - 65536)
    return ECAH_ERR_SHAPE;
  for (long long s : {a->target_batch_stride, a->target_row_stride, a->draft_batch_stride, a->draft_row_stride})
    if (s < 0) return ECAH_ERR_SHAPE;
  if (a->batch == 0) return ECAH_OK;
  if (!a->target || !a->uniforms || !a->tokens || !a->accepted || (a->drafts && !a->draft_ids)) return ECAH_ERR_NULL;
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < ecah_verify_drafts_workspace_bytes(a->batch))
    return ECAH_ERR_WORKSPACE;
  const int sms = device_sms();
  if (sms <= 0) return ECAH_ERR_LAUNCH;
  drafts::Params P = {};
  P.target = a->target; P.draft = a->drafts ? a->draft : nullptr;
  P.t_batch = a->target_batch_stride; P.t_row = a->target_row_stride;
  P.d_batch = a->draft_batch_stride; P.d_row = a->draft_row_stride;
  P.ids = a->draft_ids; P.num = a->num_drafts; P.u = a->uniforms;
  P.tokens = a->tokens; P.accepted = a->accepted;
  P.workspace = static_cast<unsigned char*>(a->workspace);
  P.N = a->drafts; P.V = a->vocab;
  // Blocks to a request: about a wave over the SMs, and ranges of kRange entries a warp at the least.
  const long long wave = std::max<long long>(1, drafts::kWave * static_cast<long long>(sms) / a->batch);
  const long long least = static_cast<long long>(drafts::kW) * drafts::kRange;
  long long chunks = std::min<long long>((a->vocab + least - 1) / least, wave);
  chunks = std::max<long long>(1, std::min<long long>(chunks, drafts::kMaxChunks));
  const long long warps = chunks * drafts::kW;
  P.range = static_cast<int>((a->vocab + warps * 8 - 1) / (warps * 8) * 8);
  P.chunks = static_cast<int>(chunks);
  const dim3 grid(P.chunks, a->batch);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool ok = a->dtype == ECAH_DTYPE_F16    ? launch_kernel(drafts::verify_kernel<ECAH_DTYPE_F16>, grid, drafts::kT, 0, s, P)
                  : a->dtype == ECAH_DTYPE_BF16 ? launch_kernel(drafts::verify_kernel<ECAH_DTYPE_BF16>, grid, drafts::kT, 0, s, P)
                                                : launch_kernel(drafts::verify_kernel<ECAH_DTYPE_F32>, grid, drafts::kT, 0, s, P);
  return ok ? ECAH_OK : ECAH_ERR_LAUNCH;
}

}  // extern "C"
