// Token log probabilities, entropy and most likely alternatives of logits
// rows: ecah_token_logprobs (contract in include/ecah_sampler.h).

#include <algorithm>

#include "common.cuh"
#include "host_util.h"

namespace ecah {
namespace lp {

// The mathematics, in one pass over the row: a thread keeps a reference m that is
// one of its own values, z = sum 2^((x - m) c) and s = sum 2^((x - m) c) (x - m) c with
// c = log2 e / T.  Triples over disjoint entries join exactly:
//   (m, z, s) as seen from M: (M, z f, f (s + d z)), d = (m - M) c, f = 2^d,
// and ln Z = ln z, entropy = ln z - ln 2 s / z.  The differences are taken before
// the multiplication, so a temperature of 1e-5 loses nothing.
//
// The alternatives need no second pass either: entries are kept while they may
// still be among the N largest.  Within a step (a contiguous piece of the row, so
// later steps have larger indices and lose ties) a floor below the N-th best is
// found from the threads' maxima; after that an entry is kept only above it.
//
// Bound: HBM for many rows (one read of the logits); 16-bit logits at 6.5 TB/s
// bring 11.6 entries a clock to an SM, whose 16 exponentials a clock are then 70 %
// busy.  Few rows are bound by latency: the row is cut into parts of at least one
// 16-byte vector a thread.
//
// Split: all rows' vectors, in order, are divided evenly over the blocks; a row
// that spans several blocks is joined by the block that arrives last, in the order
// of the parts.

constexpr int kT = 256;
constexpr int kW = kT / 32;
constexpr int kU = 4;                  // vectors of a thread and step
constexpr int kStep = kT * kU;         // vectors of a step
constexpr int kBlocks = 4;             // per SM
constexpr int kRing = 2 * kU;          // a step in flight behind the one at work
constexpr int kC = 2048;               // kept entries
constexpr int kMaxN = ECAH_MAX_TOP_N;
constexpr int kMaxParts = kC / kMaxN;  // parts of a row: all their alternatives fit the kept entries
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kSlack = 40.0f;        // the reference moves when an exponent would pass it
constexpr float kTiny = -150.0f;       // 2^kTiny is zero in float32

struct alignas(16) Part {
  float m, z, s;
  int flags;                           // alternatives | bad << 16
};

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
  long long nv;                        // vectors of a row, its edges included
  unsigned* counters;                  // [slots], zero between launches
  Part* parts;                         // [slots]
  unsigned long long* part_top;        // [slots][kMaxN]
};

struct Smem {
  uint4 ring[kRing][kT];
  unsigned long long kept[kC];
  unsigned long long top[kMaxN];
  float red[3][kW];
  int n, flag, count;
};

// Order of the alternatives: value descending, then index ascending, as one
// 64-bit key (larger is earlier).  -0 counts as +0, as a comparison would.
__device__ __forceinline__ uint32_t value_key(float x) { return key32(x == 0.0f ? 0.0f : x); }
__device__ __forceinline__ unsigned long long order_key(float x, unsigned idx) {
  return (static_cast<unsigned long long>(value_key(x)) << 32) | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ float order_value(unsigned long long k) { return unkey32(static_cast<uint32_t>(k >> 32)); }
__device__ __forceinline__ int order_index(unsigned long long k) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(k)); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

using f2 = unsigned long long;         // two float32 in a register pair
__device__ __forceinline__ f2 pack(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// A 16-byte vector of the row by type: its values two at a time, its maximum
// (a NaN if it holds one), and the word that stands for entries outside the row.
template <int DT> struct Vec {
  static constexpr int kN = DType<DT>::kVec;
  static constexpr uint32_t kOut = DT == ECAH_DTYPE_F16 ? 0xFC00FC00u : 0xFF80FF80u;   // -inf
  static __device__ __forceinline__ void pair(const uint4& v, int i, float& a, float& b) {
    const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
    if (DT == ECAH_DTYPE_F16) {
      asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, h; }" : "=f"(a), "=f"(b) : "r"(w));
    } else {
      a = __uint_as_float(w << 16);
      b = __uint_as_float(w & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    if (DT == ECAH_DTYPE_F16) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float biggest(const uint4 (&v)[kU]) {
    uint32_t m = v[0].x;
#pragma unroll
    for (int u = 0; u < kU; ++u) m = max2(max2(m, max2(v[u].x, v[u].y)), max2(v[u].z, v[u].w));
    return max_nan(DType<DT>::to_f32(m & 0xFFFFu), DType<DT>::to_f32(m >> 16));
  }
};
template <> struct Vec<ECAH_DTYPE_F32> {
  static constexpr int kN = 4;
  static constexpr uint32_t kOut = 0xFF800000u;
  static __device__ __forceinline__ void pair(const uint4& v, int i, float& a, float& b) {
    a = __uint_as_float(i == 0 ? v.x : v.z);
    b = __uint_as_float(i == 0 ? v.y : v.w);
  }
  static __device__ __forceinline__ float biggest(const uint4 (&v)[kU]) {
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < kU; ++u)
      m = max_nan(max_nan(max_nan(m, __uint_as_float(v[u].x)), max_nan(__uint_as_float(v[u].y), __uint_as_float(v[u].z))),
                  __uint_as_float(v[u].w));
    return m;
  }
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A row as vectors: vector v holds entries [v kN - mis, (v + 1) kN - mis).
template <int DT>
struct Row {
  const unsigned char* base;           // the 16-byte boundary at or before entry 0
  int mis;
  __device__ __forceinline__ void set(const Params& P, int r) {
    long long row = r;
    if (P.row_index) row = min(max(P.row_index[r], 0), P.logit_rows - 1);
    const auto* x = static_cast<const typename DType<DT>::Raw*>(P.logits) + row * P.row_stride;
    const unsigned long long p = reinterpret_cast<unsigned long long>(x);
    mis = static_cast<int>(p & 15u) / static_cast<int>(sizeof(*x));
    base = reinterpret_cast<const unsigned char*>(p & ~15ull);
  }
  __device__ __forceinline__ float at(int i) const {
    return DType<DT>::to_f32(reinterpret_cast<const typename DType<DT>::Raw*>(base)[i + mis]);
  }
};

// This block's walk over its vectors [pos, end): steps of at most kStep vectors
// within one row.
template <int DT>
struct Walk {
  long long pos, end, row_start;
  int r;
  Row<DT> row;
  __device__ __forceinline__ bool done() const { return pos >= end; }
  __device__ __forceinline__ int length(const Params& P) const {
    return static_cast<int>(min(static_cast<long long>(kStep), min(end, row_start + P.nv) - pos));
  }
  __device__ __forceinline__ void advance(const Params& P) {
    pos += length(P);
    if (pos >= row_start + P.nv && pos < end) {
      row_start += P.nv;
      row.set(P, ++r);
    }
  }
};

// Copies this thread's vectors of the step into its own ring slots.
template <int DT>
__device__ __forceinline__ void fetch(const Params& P, const Walk<DT>& w, Smem& S, int parity) {
  constexpr int kN = Vec<DT>::kN;
  if (!w.done()) {
    const int v0 = static_cast<int>(w.pos - w.row_start), len = w.length(P), tid = threadIdx.x;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = u * kT + tid, v = v0 + i;
      const long long first = static_cast<long long>(v) * kN - w.row.mis;
      uint4* slot = &S.ring[parity * kU + u][tid];
      if (i < len && first >= 0 && first + kN <= P.V) {
        cp16(static_cast<uint32_t>(__cvta_generic_to_shared(slot)), w.row.base + static_cast<long long>(v) * 16);
      } else {
        uint32_t q[4] = {Vec<DT>::kOut, Vec<DT>::kOut, Vec<DT>::kOut, Vec<DT>::kOut};
        if (i < len) {                  // the row's edge: entry by entry
          using Raw = typename DType<DT>::Raw;
          const Raw* x = reinterpret_cast<const Raw*>(w.row.base) + static_cast<long long>(v) * kN;
#pragma unroll
          for (int j = 0; j < kN; ++j)
            if (first + j >= 0 && first + j < P.V) {
              const uint32_t raw = x[j];
              if (kN == 4) q[j] = raw;
              else q[j / 2] = (j & 1) ? (q[j / 2] & 0xFFFFu) | (raw << 16) : (q[j / 2] & 0xFFFF0000u) | raw;
            }
        }
        *slot = make_uint4(q[0], q[1], q[2], q[3]);
      }
    }
  }
  cp_commit();
}

__device__ __forceinline__ int block_sum(int v, Smem& S) {
  __syncthreads();
  if (threadIdx.x == 0) S.count = 0;
  __syncthreads();
  v = __reduce_add_sync(0xFFFFFFFFu, v);
  if ((threadIdx.x & 31) == 0) atomicAdd(&S.count, v);
  __syncthreads();
  return S.count;
}

// The N largest of the n kept entries, in order, in S.top; returns their number.
// Called by the whole block; S.kept is then free to be written again.
__device__ __noinline__ int select_top(Smem& S, int n, int N) {
  const int tid = threadIdx.x;
  __syncthreads();
  if (n > kT) {
    // more than one each: the N-th largest by bits (the keys are distinct), then only those
    unsigned long long T = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const unsigned long long t = T | (1ull << bit);
      int c = 0;
      for (int i = tid; i < n; i += kT) c += S.kept[i] >= t;
      if (block_sum(c, S) >= N) T = t;
    }
    __syncthreads();
    if (tid == 0) S.count = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kT)
      if (S.kept[i] >= T) S.top[atomicAdd(&S.count, 1)] = S.kept[i];
    __syncthreads();
    n = N;
    if (tid < n) S.kept[tid] = S.top[tid];
    __syncthreads();
  }
  unsigned long long k = 0;
  int rank = N;
  if (tid < n) {
    k = S.kept[tid];
    rank = 0;
    for (int i = 0; i < n; ++i) rank += S.kept[i] > k;
  }
  __syncthreads();
  if (rank < N) S.top[rank] = k;
  __syncthreads();
  return min(n, N);
}

// A floor for this step when its candidates are too many to keep: at least N
// threads hold an entry at or above it, and no more than `most` threads do, by
// value (key) or, among equal values, by the index `last` of the latest kept one.
__device__ __noinline__ void find_floor(Smem& S, uint32_t mine, int first_of_mine, int N, int most, uint32_t* floor_key, int* last) {
  uint32_t T = 0;
  int cnt = kT;
  for (int bit = 31; bit >= 0 && cnt > most; --bit) {
    const uint32_t t = T | (1u << bit);
    const int c = __syncthreads_count(mine >= t);
    if (c >= N) { T = t; cnt = c; }
  }
  *floor_key = T;
  *last = 0x7FFFFFFF;
  if (cnt > most) {
    // ties at T: the N-th lowest first index among the threads at it
    const int above = __syncthreads_count(mine > T);
    int I = 0;
    for (int bit = 30; bit >= 0; --bit) {
      const int t = I | (1 << bit);
      if (above + __syncthreads_count(mine == T && first_of_mine < t) < N) I = t;
    }
    *last = I;
  }
}

// One row's (or part's) running state and the reading of it, by one block.
template <int DT>
__global__ void __launch_bounds__(kT, kBlocks) token_logprobs_kernel(const Params P) {
  constexpr int kN = Vec<DT>::kN;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Smem& S = *reinterpret_cast<Smem*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long total = P.nv * P.R, blocks = gridDim.x;

  Walk<DT> w;
  w.pos = blockIdx.x * total / blocks;
  w.end = (blockIdx.x + 1ll) * total / blocks;
  w.r = static_cast<int>(w.pos / P.nv);
  w.row_start = w.r * P.nv;
  w.row.set(P, w.r);
  Walk<DT> ahead = w;
  fetch(P, ahead, S, 0);
  ahead.advance(P);
  if (tid == 0) S.n = 0;
  int parity = 0;

  while (!w.done()) {
    const int r = w.r;
    const Row<DT> row = w.row;
    const long long row_start = w.row_start, row_end = min(w.end, row_start + P.nv);
    const float T = P.temperature ? P.temperature[r] : 1.0f;
    const bool greedy = T <= 0.0f;
    const float c = greedy ? 0.0f : fminf(kLog2e / T, 3e38f);
    const int N = max(P.N, greedy ? 1 : 0);
    // the row's tokens, read while the row streams
    int tok = -1;
    float tok_x = 0.0f;
    if (tid < P.K) {
      tok = P.token_ids[static_cast<long long>(r) * P.K + tid];
      if (tok >= 0 && tok < P.V) tok_x = row.at(tok);
    }

    float ref = -INFINITY, big = -INFINITY, floor_v = -INFINITY;
    f2 z2 = pack(0.0f, 0.0f), s2 = pack(0.0f, 0.0f);
    bool bad = false;
    int n = 0;
    for (; w.pos < row_end; w.advance(P), parity ^= 1) {
      fetch(P, ahead, S, parity ^ 1);
      if (!ahead.done()) ahead.advance(P);
      cp_wait<1>();
      uint4 v[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) v[u] = S.ring[parity * kU + u][tid];
      const float top = Vec<DT>::biggest(v);
      bad |= !(top < INFINITY);
      big = fmaxf(big, top);
      if ((top - ref) * c > kSlack || (ref == -INFINITY && top > ref)) {
        const float d = (ref - top) * c, f = ref == -INFINITY ? 0.0f : ex2_approx(d);
        float za, zb, sa, sb;
        unpack(z2, za, zb);
        unpack(s2, sa, sb);
        if (f > 0.0f) {
          s2 = pack(f * (sa + d * za), f * (sb + d * zb));
          z2 = pack(f * za, f * zb);
        } else {
          s2 = z2 = pack(0.0f, 0.0f);
        }
        ref = top;
      }
      if (ref > -INFINITY) {
        const f2 minus = pack(-ref, -ref), c2 = pack(c, c);
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
          for (int i = 0; i < kN / 2; ++i) {
            float a, b;
            Vec<DT>::pair(v[u], i, a, b);
            unpack(mul2(add2(pack(a, b), minus), c2), a, b);
            a = fmaxf(a, kTiny);       // an entry of -inf has no mass and no part in s
            b = fmaxf(b, kTiny);
            const f2 e = pack(ex2_approx(a), ex2_approx(b));
            z2 = add2(z2, e);
            s2 = fma2(e, pack(a, b), s2);
          }
      }
      if (N > 0) {
        const int cand = __syncthreads_count(top > floor_v);
        if (cand) {
          const int v0 = static_cast<int>(w.pos - row_start);
          uint32_t floor_key = 0;
          int last = 0x7FFFFFFF;
          bool keep = top > floor_v;
          const int most = (kC - n) / (kU * kN);
          if (cand > most) {
            const uint32_t mine = keep ? value_key(top) : 0u;
            int first = 0x7FFFFFFF;
#pragma unroll
            for (int u = kU - 1; u >= 0; --u)
#pragma unroll
              for (int i = kN / 2 - 1; i >= 0; --i) {
                float a, b;
                Vec<DT>::pair(v[u], i, a, b);
                const int at = (v0 + u * kT + tid) * kN - row.mis + 2 * i;
                if (b == top) first = at + 1;
                if (a == top) first = at;
              }
            find_floor(S, mine, first, N, most, &floor_key, &last);
            keep = mine > floor_key || (mine == floor_key && first <= last);
          }
          if (keep) {
#pragma unroll 1
            for (int u = 0; u < kU; ++u) {
              const uint4 q = S.ring[parity * kU + u][tid];
              const int at = (v0 + u * kT + tid) * kN - row.mis;
#pragma unroll
              for (int i = 0; i < kN; ++i) {
                float a, b;
                Vec<DT>::pair(q, i / 2, a, b);
                const float x = i & 1 ? b : a;
                const uint32_t k = value_key(x);
                if (x > floor_v && (k > floor_key || (k == floor_key && at + i <= last)))
                  S.kept[atomicAdd(&S.n, 1)] = order_key(x, at + i);
              }
            }
          }
          __syncthreads();
          n = S.n;
          if (floor_key) floor_v = fmaxf(floor_v, unkey32(floor_key));
          if (n > 3 * N + 16) {        // fewer candidates from here on
            n = select_top(S, n, N);
            if (tid < n) S.kept[tid] = S.top[tid];
            if (tid == 0) S.n = n;
            if (n == N) floor_v = order_value(S.top[N - 1]);
            __syncthreads();
          }
        }
      }
    }

    // ---- this block's triple
    float M = big, z, s, zb, sb;
    unpack(z2, z, zb);
    unpack(s2, s, sb);
    z += zb;
    s += sb;
    bad = __syncthreads_or(bad);
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, o));
    if (lane == 0) S.red[0][warp] = M;
    __syncthreads();
    M = S.red[0][0];
#pragma unroll
    for (int i = 1; i < kW; ++i) M = fmaxf(M, S.red[0][i]);
    auto seen_from = [&](float m, float& zz, float& ss) {
      const float d = (m - M) * c, f = m == -INFINITY ? 0.0f : m == M ? 1.0f : ex2_approx(d);
      ss = f > 0.0f ? f * (ss + (m == M ? 0.0f : d) * zz) : 0.0f;
      zz *= f;
    };
    seen_from(ref, z, s);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      z += __shfl_xor_sync(0xFFFFFFFFu, z, o);
      s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    }
    if (lane == 0) { S.red[1][warp] = z; S.red[2][warp] = s; }
    int have = 0;
    if (N > 0) have = select_top(S, n, N);
    else __syncthreads();
    z = s = 0.0f;
#pragma unroll
    for (int i = 0; i < kW; ++i) { z += S.red[1][i]; s += S.red[2][i]; }

    // ---- the row's parts: the blocks whose shares overlap it
    const long long a = ((row_start + 1) * blocks - 1) / total, b = ((row_start + P.nv) * blocks - 1) / total;
    const int parts = static_cast<int>(b - a) + 1;
    bool finish = parts == 1;
    if (parts > 1) {
      auto slot_of = [&](int p) -> long long { return p == 0 ? 2 * a + 1 : 2 * (a + p); };
      const long long slot = slot_of(static_cast<int>(blockIdx.x - a));
      if (tid < have) P.part_top[slot * kMaxN + tid] = S.top[tid];
      if (tid == 0) P.parts[slot] = Part{M, z, s, have | (bad ? 1 << 16 : 0)};
      __syncthreads();
      if (tid == 0) {
        unsigned got;
        unsigned* counter = P.counters + slot_of(0);
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(got) : "l"(counter) : "memory");
        S.flag = got + 1u == static_cast<unsigned>(parts);
        if (S.flag) *counter = 0u;
        S.n = 0;
      }
      __syncthreads();
      finish = S.flag != 0;
      if (finish) {
        // parts <= kMaxParts < kT: one each
        Part q = {-INFINITY, 0.0f, 0.0f, 0};
        unsigned long long low = 0;
        if (tid < parts) {
          const float4 u = __ldcg(reinterpret_cast<const float4*>(P.parts + slot_of(tid)));
          q = Part{u.x, u.y, u.z, __float_as_int(u.w)};
          // a part with N alternatives bounds the row's N-th from below
          if (N > 0 && (q.flags & 0xFFFF) == N) low = __ldcg(P.part_top + slot_of(tid) * kMaxN + N - 1);
        }
        bad = __syncthreads_or(q.flags >> 16);
        M = q.m;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, o));
          const unsigned long long other = __shfl_xor_sync(0xFFFFFFFFu, low, o);
          low = other > low ? other : low;
        }
        if (lane == 0) { S.red[0][warp] = M; S.top[warp] = low; }
        __syncthreads();
        M = S.red[0][0];
        low = S.top[0];
#pragma unroll
        for (int i = 1; i < kW; ++i) {
          M = fmaxf(M, S.red[0][i]);
          low = S.top[i] > low ? S.top[i] : low;
        }
        z = q.z;
        s = q.s;
        seen_from(q.m, z, s);
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          z += __shfl_xor_sync(0xFFFFFFFFu, z, o);
          s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        }
        if (lane == 0) { S.red[1][warp] = z; S.red[2][warp] = s; }
        if (N > 0) {
          for (int i = tid; i < parts * N; i += kT) {
            const long long from = slot_of(i / N);
            if (i % N < (__ldcg(&P.parts[from].flags) & 0xFFFF)) {
              const unsigned long long k = __ldcg(P.part_top + from * kMaxN + i % N);
              if (k >= low) S.kept[atomicAdd(&S.n, 1)] = k;
            }
          }
          __syncthreads();
          have = select_top(S, S.n, N);
        } else {
          __syncthreads();
        }
        z = s = 0.0f;
#pragma unroll
        for (int i = 0; i < kW; ++i) { z += S.red[1][i]; s += S.red[2][i]; }
      }
    }

    // ---- the row's results
    if (finish) {
      const bool empty = !bad && M == -INFINITY;
      const float lz = logf(z);
      const int arg = greedy && have > 0 ? order_index(S.top[0]) : -1;
      auto logprob = [&](float x, int i) -> float {
        if (bad) return NAN;
        if (empty || x == -INFINITY) return -INFINITY;
        if (greedy) return i == arg ? 0.0f : -INFINITY;
        // halved, so that the difference of two values of opposite sign near the type's largest stays finite
        return (0.5f * x - 0.5f * M) / (0.5f * T) - lz;
      };
      if (tid == 0 && P.entropy) P.entropy[r] = bad ? NAN : (empty || greedy) ? 0.0f : lz - s / z * kLn2;
      for (int j = tid; j < P.K; j += kT) {
        const long long at = static_cast<long long>(r) * P.K + j;
        if (j >= kT) {
          tok = P.token_ids[at];
          tok_x = tok >= 0 && tok < P.V ? row.at(tok) : 0.0f;
        }
        P.logprobs[at] = (tok < 0 || tok >= P.V) ? NAN : logprob(tok_x, tok);
      }
      if (tid < P.N) {
        const long long at = static_cast<long long>(r) * P.N + tid;
        const bool is = !bad && tid < have;
        P.top_ids[at] = is ? order_index(S.top[tid]) : -1;
        P.top_logprobs[at] = is ? logprob(order_value(S.top[tid]), order_index(S.top[tid])) : bad ? NAN : -INFINITY;
      }
    }
    __syncthreads();
    if (tid == 0) S.n = 0;
    __syncthreads();
  }
  cp_wait<0>();
}

// Workspace: one slot for a part a block shares with the one before it, one for
// a part it shares with the one after it.
struct Layout {
  size_t parts, top, total;
};

static Layout layout(int sms) {
  const size_t slots = 2 * static_cast<size_t>(sms) * kBlocks + 2;
  Layout L;
  L.parts = (slots * sizeof(unsigned) + 255) / 256 * 256;
  L.top = L.parts + slots * sizeof(Part);
  L.total = L.top + slots * kMaxN * sizeof(unsigned long long);
  return L;
}

}  // namespace lp
}  // namespace ecah

using namespace ecah;

extern "C" {

size_t ecah_token_logprobs_workspace_bytes(void) {
  const int sms = device_sms();
  return sms > 0 ? lp::layout(sms).total : 0;
}

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
  const int sms = device_sms();
  if (sms <= 0) return ECAH_ERR_LAUNCH;
  const lp::Layout L = lp::layout(sms);
  unsigned char* ws = static_cast<unsigned char*>(a->workspace);
  P.counters = reinterpret_cast<unsigned*>(ws);
  P.parts = reinterpret_cast<lp::Part*>(ws + L.parts);
  P.part_top = reinterpret_cast<unsigned long long*>(ws + L.top);
  const int vec = a->dtype == ECAH_DTYPE_F32 ? 4 : 8;
  P.nv = (static_cast<long long>(P.V) + 2 * (vec - 1)) / vec;
  // a vector a thread at least; a row overlaps at most blocks / R + 2 of them, and its
  // alternatives are joined of at most kMaxParts
  long long blocks = std::min<long long>(static_cast<long long>(sms) * lp::kBlocks, (P.nv * P.R + lp::kT - 1) / lp::kT);
  blocks = std::min<long long>(blocks, (lp::kMaxParts - 2ll) * P.R);
  auto fn = a->dtype == ECAH_DTYPE_F16 ? lp::token_logprobs_kernel<ECAH_DTYPE_F16>
            : a->dtype == ECAH_DTYPE_BF16 ? lp::token_logprobs_kernel<ECAH_DTYPE_BF16>
                                          : lp::token_logprobs_kernel<ECAH_DTYPE_F32>;
  return launch_kernel(fn, dim3(static_cast<unsigned>(blocks)), lp::kT, static_cast<int>(sizeof(lp::Smem)),
                       reinterpret_cast<cudaStream_t>(stream), P) ? ECAH_OK : ECAH_ERR_LAUNCH;
}

}  // extern "C"
