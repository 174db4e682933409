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
// The alternatives: a thread leaves the largest value of each of its steps (40 or
// 20 entries) as a record in shared memory, nothing more while the row streams.
// Afterwards the N-th largest of the threads' maxima is a floor that N entries
// reach; only the steps whose record reaches it, about N of them, are read again
// (from L2) for the entries at or above it.
//
// Bound: HBM for many rows (one read of the logits); 16-bit logits at 6.5 TB/s
// bring 11.6 entries a clock to an SM, whose 16 exponentials a clock are then 70 %
// busy.  Few rows are bound by latency: the row is cut into parts of at least one
// 16-byte vector a thread.
//
// Split: all rows' vectors, in order, are divided evenly over the blocks; a row
// that spans several blocks is joined by the block that arrives last, in the order
// of the parts.
//
// Measured on one B200, device time of graph replays: 2048 rows of 128256 bf16 with
// one alternative 109 us (4.8 TB/s; 95 us without alternatives, 112 with 5, 127 with
// 20), 512 rows of 151936 f32 with 5 alternatives 63 us (4.9 TB/s), 128 rows of 151936
// f16 with 20 alternatives at a temperature 19.8 us (13.4 without), one row with 5
// alternatives 9.2 us, 37 masked rows of 32003 f32 with 8 alternatives 10.5 us.
// What bounds them: 7.6 instructions an entry and the row's end (a row every 3 us in
// each block) for many rows; start, row end and join, in turn, for few.

constexpr int kT = 128;
constexpr int kW = kT / 32;
constexpr int kU = 5;                  // vectors of a thread and step
constexpr int kStep = kT * kU;         // vectors of a step
// per SM, 96 registers a thread, 50 KB in flight.  Small blocks leave others streaming
// while one ends a row: 2048 rows took 117 us in 256-thread blocks, 107 us in these.
constexpr int kBlocks = 5;
constexpr int kRing = 2 * kU;          // a step in flight behind the one at work
constexpr int kC = 512;                // entries of one selection
constexpr int kMaxSteps = 32;          // steps with a record: 163840 16-bit logits
constexpr int kMaxN = ECAH_MAX_TOP_N;
constexpr int kList = 128;             // steps read again at once
constexpr int kMaxParts = 32;          // parts of a row
constexpr int kJoin = (kC - kMaxN) / kMaxN;   // parts whose alternatives are joined at once
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kSlack = 40.0f;        // the reference moves when an exponent would pass it
constexpr float kTiny = -150.0f;       // 2^kTiny is zero in float32

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
  long long share;                     // vectors of a block: share, and one more in the first `more`
  int more;
  unsigned* counters;                  // [slots], zero between launches
  float4* parts;                       // [slots] m (NaN: the row has no distribution), z, s
  unsigned long long* part_top;        // [slots][kMaxN]
};

struct Smem {
  uint4 ring[kRing][kT];
  unsigned long long kept[kC];
  uint16_t records[kMaxSteps][kT];
  int chunks[kList];
  unsigned long long top[kMaxN];
  float red[3][kW];
  uint32_t best[32];
  int n, flag, list;
  long long begin, end;                // this block's share
};

static_assert((sizeof(Smem) + 1024) * kBlocks <= 227 * 1024, "the blocks of an SM fit its shared memory");

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
  // a value's record, in the order of the values (f32: rounded down to 16 bits)
  static __device__ __forceinline__ uint32_t rec(float x) { return key16(DType<DT>::to_raw(x == 0.0f ? 0.0f : x)); }
  static __device__ __forceinline__ float value(uint32_t rec) { return DType<DT>::to_f32(unkey16(rec)); }
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
  template <int U>
  static __device__ __forceinline__ float biggest(const uint4 (&v)[U]) {
    uint32_t m = v[0].x;
#pragma unroll
    for (int u = 0; u < U; ++u) m = max2(max2(m, max2(v[u].x, v[u].y)), max2(v[u].z, v[u].w));
    return max_nan(DType<DT>::to_f32(m & 0xFFFFu), DType<DT>::to_f32(m >> 16));
  }
};
template <> struct Vec<ECAH_DTYPE_F32> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ uint32_t rec(float x) { return value_key(x) >> 16; }
  static __device__ __forceinline__ float value(uint32_t rec) { return unkey32(rec << 16); }
  static constexpr uint32_t kOut = 0xFF800000u;
  static __device__ __forceinline__ void pair(const uint4& v, int i, float& a, float& b) {
    a = __uint_as_float(i == 0 ? v.x : v.z);
    b = __uint_as_float(i == 0 ? v.y : v.w);
  }
  template <int U>
  static __device__ __forceinline__ float biggest(const uint4 (&v)[U]) {
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
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

// This block's piece of one row: vectors [v, v_end).
template <int DT>
struct Piece {
  Row<DT> row;
  int v, v_end;
};

// A vector at the row's edge, entry by entry: -inf outside the row.
template <int DT>
__device__ __noinline__ uint4 edge_vector(const unsigned char* base, int mis, int v, int V) {
  constexpr int kN = Vec<DT>::kN;
  using Raw = typename DType<DT>::Raw;
  uint32_t q[4] = {Vec<DT>::kOut, Vec<DT>::kOut, Vec<DT>::kOut, Vec<DT>::kOut};
  const long long first = static_cast<long long>(v) * kN - mis;
  const Raw* x = reinterpret_cast<const Raw*>(base) + static_cast<long long>(v) * kN;
#pragma unroll
  for (int j = 0; j < kN; ++j)
    if (first + j >= 0 && first + j < V) {
      const uint32_t raw = x[j];
      if (kN == 4) q[j] = raw;
      else q[j / 2] = (j & 1) ? (q[j / 2] & 0xFFFFu) | (raw << 16) : (q[j / 2] & 0xFFFF0000u) | raw;
    }
  return make_uint4(q[0], q[1], q[2], q[3]);
}

// Copies this thread's vectors of the step at v0 into its own ring slots, where
// the step is not wholly inside the row and the piece.
template <int DT>
__device__ __noinline__ void fetch_edge(const unsigned char* base, int mis, int v0, int v_end, int V, uint4* slot) {
  const int whole0 = mis ? 1 : 0, whole1 = (V + mis) / Vec<DT>::kN;     // vectors wholly inside the row
  for (int u = 0; u < kU; ++u) {
    const int v = v0 + u * kT + threadIdx.x;
    if (v >= whole0 && v < whole1 && v < v_end)
      cp16(static_cast<uint32_t>(__cvta_generic_to_shared(slot + u * kT)), base + static_cast<long long>(v) * 16);
    else
      slot[u * kT] = v < v_end ? edge_vector<DT>(base, mis, v, V) : make_uint4(Vec<DT>::kOut, Vec<DT>::kOut, Vec<DT>::kOut, Vec<DT>::kOut);
  }
}

// Steps that begin at [first, last] are wholly inside: copied without a look.
template <int DT>
__device__ __forceinline__ void fetch(const Piece<DT>& p, int first, int last, int V, Smem& S, int parity) {
  uint4* slot = &S.ring[parity * kU][threadIdx.x];
  if (p.v >= first && p.v <= last) {
    const unsigned char* src = p.row.base + static_cast<long long>(p.v + static_cast<int>(threadIdx.x)) * 16;
    const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(slot));
#pragma unroll
    for (int u = 0; u < kU; ++u) cp16(dst + u * kT * 16, src + u * kT * 16);
  } else {
    fetch_edge<DT>(p.row.base, p.row.mis, p.v, p.v_end, V, slot);
  }
  cp_commit();
}
template <int DT>
__device__ __forceinline__ int first_whole(const Piece<DT>& p) { return p.row.mis ? 1 : 0; }
template <int DT>
__device__ __forceinline__ int last_whole(const Piece<DT>& p, int V) { return min((V + p.row.mis) / Vec<DT>::kN, p.v_end) - kStep; }

// A triple (m, z, s) as seen from M >= m.
__device__ __forceinline__ void seen_from(float M, float m, float c, float& z, float& s) {
  const float d = (m - M) * c, f = m == -INFINITY ? 0.0f : m == M ? 1.0f : ex2_approx(d);
  s = f > 0.0f ? f * (s + (m == M ? 0.0f : d) * z) : 0.0f;
  z *= f;
}

// The N largest of the n kept entries, in order, in S.top; returns their number.
// Called by the whole block after a barrier; ends with one.
__device__ __noinline__ int select_top(Smem& S, int n, int N) {
  const int tid = threadIdx.x;
  if (n <= kT) {                       // four, two or one threads a key
    const int shift = n <= kT / 4 ? 2 : n <= kT / 2 ? 1 : 0, i = tid >> shift, step = 1 << shift;
    unsigned long long k = 0;
    int rank = 0;
    if (i < n) {
      k = S.kept[i];
#pragma unroll 8
      for (int j = tid & (step - 1); j < n; j += step) rank += S.kept[j] > k;
    }
    if (shift >= 1) rank += __shfl_xor_sync(0xFFFFFFFFu, rank, 1);
    if (shift == 2) rank += __shfl_xor_sync(0xFFFFFFFFu, rank, 2);
    if (i < n && rank < N) S.top[rank] = k;      // the threads of a key agree
  } else {                             // up to kC / kT keys a thread
    unsigned long long key[kC / kT];
    int above[kC / kT];
#pragma unroll
    for (int i = 0; i < kC / kT; ++i) {
      key[i] = i * kT + tid < n ? S.kept[i * kT + tid] : 0ull;
      above[i] = 0;
    }
    for (int j = 0; j < n; ++j) {
      const unsigned long long q = S.kept[j];
#pragma unroll
      for (int i = 0; i < kC / kT; ++i) above[i] += q > key[i];
    }
#pragma unroll
    for (int i = 0; i < kC / kT; ++i)
      if (i * kT + tid < n && above[i] < N) S.top[above[i]] = key[i];
  }
  __syncthreads();
  return min(n, N);
}

// The N best of what this block has kept (`have` in S.top) and of the steps
// recorded since, vectors [v0, v_end) of the row in steps of kStep, in S.top; returns
// their number.  `best` is the largest record of this thread; a single step is
// still in the ring's half `parity`.
template <int DT>
__device__ __noinline__ int collect(Smem& S, Row<DT> row, int V, int v0, int v_end, int parity, uint32_t best, int have, int N) {
  constexpr int kN = Vec<DT>::kN, kEach = kU * kN, kGroup = (kC - kMaxN) / kEach;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t none = Vec<DT>::rec(-INFINITY);
  const int steps = (v_end - v0 + kStep - 1) / kStep;
  // A floor that N threads reach: the N-th largest of every warp's few best lanes.
  const int share = (N + kW - 1) / kW, few = min(share > 1 ? share + 2 : 1, 32 / kW), all = few * kW;
  uint32_t v = best;
  for (int i = 0; i < few; ++i) {
    const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, v);
    const bool mine = lane == __ffs(__ballot_sync(0xFFFFFFFFu, v == m)) - 1;
    if (mine) { S.best[warp * few + i] = m; v = 0; }
  }
  const unsigned long long carried = have == N ? S.top[N - 1] : 0ull;
  if (tid < have) S.kept[tid] = S.top[tid];
  if (tid == 0) { S.n = have; S.list = 0; }
  __syncthreads();
  v = lane < all ? S.best[lane] : 0u;
  int rank = 0;
  for (int i = 0; i < all; ++i) {
    const uint32_t k = S.best[i];
    rank += k > v || (k == v && i < lane);
  }
  uint32_t floor_r = __shfl_sync(0xFFFFFFFFu, v, __ffs(__ballot_sync(0xFFFFFFFFu, lane < all && rank == N - 1)) - 1);
  floor_r = max(floor_r, none + 1u);             // entries of -inf are none
  unsigned long long floor_k = carried;
  if (best >= floor_r)
    for (int i = 0; i < steps; ++i)
      if (S.records[i][tid] >= floor_r) {
        const int at = atomicAdd(&S.list, 1);
        if (at < kList) S.chunks[at] = i * kT + tid;
      }
  __syncthreads();

  // Read the listed steps again, a lane to a vector.  `low_v` is the smallest value of
  // the floor's record; an entry at or below the carried floor leaves an empty key.
  const float low_v = Vec<DT>::value(floor_r);
  const int whole0 = row.mis ? 1 : 0, whole1 = (V + row.mis) / kN;
  auto read_list = [&]() {
    const int vectors = S.list * kU;
    for (int e = tid; e < vectors; e += kT) {
      const int chunk = S.chunks[e / kU], u = e % kU, v = v0 + (chunk / kT) * kStep + u * kT + chunk % kT;
      uint4 q = make_uint4(Vec<DT>::kOut, Vec<DT>::kOut, Vec<DT>::kOut, Vec<DT>::kOut);
      if (steps == 1) q = S.ring[parity * kU + u][chunk % kT];
      else if (v >= whole0 && v < min(whole1, v_end)) q = __ldg(reinterpret_cast<const uint4*>(row.base) + v);
      else if (v < v_end) q = edge_vector<DT>(row.base, row.mis, v, V);
      const uint4 one[1] = {q};
      if (!(Vec<DT>::rec(Vec<DT>::biggest(one)) >= floor_r)) continue;
      const int at = v * kN - row.mis;
      float x[kN];
      unsigned in = 0;
#pragma unroll
      for (int i = 0; i < kN / 2; ++i) Vec<DT>::pair(q, i, x[2 * i], x[2 * i + 1]);
#pragma unroll
      for (int i = 0; i < kN; ++i) in |= (x[i] >= low_v ? 1u : 0u) << i;
      int to = atomicAdd(&S.n, __popc(in));
#pragma unroll
      for (int i = 0; i < kN; ++i)
        if (in >> i & 1u) {
          const unsigned long long k = order_key(x[i], static_cast<unsigned>(at + i));
          if (to < kC) S.kept[to] = k > floor_k ? k : 0ull;
          ++to;
        }
    }
    __syncthreads();
  };
  if (S.list <= kList) {
    read_list();
    if (S.n <= kC) return select_top(S, S.n, N);
  }
  __syncthreads();
  if (tid < have) S.kept[tid] = S.top[tid];
  if (tid == 0) S.n = have;
  // Many: ties, or one thread's entries large in many steps.  In the row's order and
  // in groups, the floor rising: equal values stop at the first group (where a
  // record is the value; an f32 record stands for a range of values, so every group is
  // read again: 128 rows of 151936 f32 with 5 entries above one finite value of all
  // others take 1.72 ms for 20 alternatives, 18.5 us where the others are -inf).
  int n = have;
  for (int i = 0; i < steps; ++i)
    for (int part = 0; part < kT; part += kGroup) {
      const int first = (v0 + i * kStep + tid) * kN - row.mis;      // the chunk's lowest index
      const uint32_t k = S.records[i][tid];
      const bool in = tid >= part && tid < part + kGroup && k >= floor_r &&
                      (floor_k == 0ull || k > Vec<DT>::rec(order_value(floor_k)) ||
                       (k == Vec<DT>::rec(order_value(floor_k)) && (kN == 4 || first <= order_index(floor_k))));
      if (!__syncthreads_or(in)) continue;
      if (tid == 0) S.list = 0;
      __syncthreads();
      if (in) S.chunks[atomicAdd(&S.list, 1)] = i * kT + tid;
      __syncthreads();
      read_list();
      n = select_top(S, S.n, N);
      if (tid < n) S.kept[tid] = S.top[tid];
      if (tid == 0) S.n = n;
      if (n == N) floor_k = S.top[N - 1];
      __syncthreads();
    }
  return n;
}

// One row's (or part's) running state and the reading of it, by one block.
template <int DT>
__global__ void __launch_bounds__(kT, kBlocks) token_logprobs_kernel(const Params P) {
  constexpr int kN = Vec<DT>::kN;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Smem& S = *reinterpret_cast<Smem*>(smem_raw);
  grid_start();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long begin = blockIdx.x * P.share + min(static_cast<int>(blockIdx.x), P.more);
  if (tid == 0) {
    S.begin = begin;
    S.end = begin + P.share + (static_cast<int>(blockIdx.x) < P.more);
  }
  __syncthreads();
  int r = static_cast<int>(begin / P.nv);
  Piece<DT> p;
  p.row.set(P, r);
  p.v = static_cast<int>(begin - r * P.nv);
  p.v_end = static_cast<int>(min(S.end - r * P.nv, P.nv));
  fetch(p, first_whole(p), last_whole(p, P.V), P.V, S, 0);
  int parity = 0;

  for (;;) {
    int N = P.N, have = 0;
    float c = kLog2e;
    if (P.temperature) {
      const float T = P.temperature[r];
      c = T <= 0.0f ? 0.0f : fminf(kLog2e / T, 3e38f);
      if (T <= 0.0f) N = max(N, 1);                // greedy: the maximum's index is the answer
    }

    const int fast = last_whole(p, P.V);
    int tok = -1;
    float tok_x = 0.0f;
    if (tid < P.K) {                   // the row's tokens, read while it streams
      tok = P.token_ids[static_cast<long long>(r) * P.K + tid];
      if (tok >= 0 && tok < P.V) tok_x = p.row.at(tok);
    }
    float ref = -INFINITY, big = -INFINITY;
    f2 z2 = pack(0.0f, 0.0f), s2 = pack(0.0f, 0.0f);
    while (p.v < p.v_end) {             // once, but for rows of more steps than there are records
    const int v0 = p.v;
    uint32_t best = 0;
    for (int step = 0; step < kMaxSteps && p.v < p.v_end; ++step, parity ^= 1) {
      p.v += kStep;
      if (p.v < p.v_end) fetch(p, 1, fast, P.V, S, parity ^ 1);
      else if ((r + 1) * P.nv < S.end) {
        Piece<DT> next;                // the next row begins while this one ends
        next.row.set(P, r + 1);
        next.v = 0;
        next.v_end = static_cast<int>(min(S.end - (r + 1) * P.nv, P.nv));
        fetch(next, first_whole(next), last_whole(next, P.V), P.V, S, parity ^ 1);
      } else cp_commit();
      cp_wait<1>();
      uint4 v[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) v[u] = S.ring[parity * kU + u][tid];
      const float top = Vec<DT>::biggest(v);
      big = max_nan(big, top);
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
        const uint32_t k = Vec<DT>::rec(top);
        S.records[step][tid] = static_cast<uint16_t>(k);
        best = max(best, k);
      }
    }
    if (p.v >= p.v_end) {
      // the warp's triple; a NaN or +inf stays in its maximum
      float m = big, z, s, zb, sb;
#pragma unroll
      for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
      unpack(z2, z, zb);
      unpack(s2, s, sb);
      z += zb;
      s += sb;
      seen_from(m, ref, c, z, s);
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        z += __shfl_xor_sync(0xFFFFFFFFu, z, o);
        s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
      }
      if (lane == 0) { S.red[0][warp] = m; S.red[1][warp] = z; S.red[2][warp] = s; }
      if (N == 0) __syncthreads();
    }
    if (N > 0) have = collect<DT>(S, p.row, P.V, v0, min(p.v, p.v_end), parity ^ 1, best, have, N);
    }

    // ---- this block's triple
    const Row<DT> row = p.row;
    const long long row_start = r * P.nv;
    float M = -INFINITY, z = 0.0f, s = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kW; ++i) {
      bad |= !(S.red[0][i] < INFINITY);
      M = fmaxf(M, S.red[0][i]);
    }
#pragma unroll
    for (int i = 0; i < kW; ++i) {
      float zi = S.red[1][i], si = S.red[2][i];
      seen_from(M, S.red[0][i], c, zi, si);
      z += zi;
      s += si;
    }

    // ---- the row's parts: the blocks whose shares overlap it
    bool finish = row_start >= S.begin && row_start + P.nv <= S.end;
    if (!finish) {
      // the block of a vector: the first `more` blocks have share + 1, the others share
      const long long head = P.more * (P.share + 1);
      auto block_of = [&](long long x) { return x < head ? x / (P.share + 1) : P.more + (x - head) / P.share; };
      const long long a = block_of(row_start);
      const int parts = static_cast<int>(block_of(row_start + P.nv - 1) - a) + 1;
      auto slot_of = [&](int p) -> long long { return p == 0 ? 2 * a + 1 : 2 * (a + p); };
      const long long slot = slot_of(static_cast<int>(blockIdx.x - a));
      if (tid < N) P.part_top[slot * kMaxN + tid] = tid < have ? S.top[tid] : 0ull;
      if (tid == 0) P.parts[slot] = make_float4(bad ? NAN : M, z, s, 0.0f);
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
        // parts <= 32: a lane each, in every warp; the alternatives in the same round of loads
        constexpr int kEach = kMaxParts / kW;
        unsigned long long key[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          const int i = j * kW + warp;
          key[j] = i < parts && lane < N ? __ldcg(P.part_top + slot_of(i) * kMaxN + lane) : 0ull;
        }
        float4 q = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        unsigned long long low = 0;    // a part's N-th bounds the row's from below
        if (lane < parts) {
          q = __ldcg(P.parts + slot_of(lane));
          if (N > 0) low = __ldcg(P.part_top + slot_of(lane) * kMaxN + N - 1);
        }
        bad = __any_sync(0xFFFFFFFFu, !(q.x < INFINITY));
        M = q.x;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, o));
          const unsigned long long other = __shfl_xor_sync(0xFFFFFFFFu, low, o);
          low = other > low ? other : low;
        }
        z = q.y;
        s = q.z;
        seen_from(M, q.x, c, z, s);
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          z += __shfl_xor_sync(0xFFFFFFFFu, z, o);
          s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        }
        have = 0;
        if (N > 0) {
          // the parts' entries that reach the bound
          low = max(low, 1ull);
          int mine = 0;
#pragma unroll
          for (int j = 0; j < kEach; ++j) mine += key[j] >= low;
          if (mine) {
            int to = atomicAdd(&S.n, mine);
#pragma unroll
            for (int j = 0; j < kEach; ++j)
              if (key[j] >= low) {
                if (to < kC) S.kept[to] = key[j];
                ++to;
              }
          }
          __syncthreads();
          if (S.n <= kC) {
            have = select_top(S, S.n, N);
          } else {
            // too many for one selection: in groups of parts
            for (int p0 = 0; p0 < parts; p0 += kJoin) {
              __syncthreads();
              if (tid < have) S.kept[tid] = S.top[tid];
              if (tid == 0) S.n = have;
              __syncthreads();
              for (int i = tid; i < min(kJoin, parts - p0) * N; i += kT) {
                const unsigned long long k = __ldcg(P.part_top + slot_of(p0 + i / N) * kMaxN + i % N);
                if (k >= low) S.kept[atomicAdd(&S.n, 1)] = k;
              }
              __syncthreads();
              have = select_top(S, S.n, N);
            }
          }
        }
      }
    }

    // ---- the row's results
    if (finish && warp * 32 < max(max(P.K, P.N), 1)) {
      const float T = P.temperature ? P.temperature[r] : 1.0f;
      const bool greedy = T <= 0.0f;
      bad |= T != T;
      const bool empty = !bad && M == -INFINITY;
      const float lz = logf(z);
      const int arg = greedy && have > 0 ? order_index(S.top[0]) : -1;
      auto logprob = [&](float x, int i) -> float {
        if (bad) return NAN;
        if (empty || x == -INFINITY) return -INFINITY;
        if (greedy) return i == arg ? 0.0f : -INFINITY;
        // halved, so that the difference of two values of opposite sign near the type's largest stays
        // finite; doubled afterwards, since half of the smallest T is zero
        return 2.0f * ((0.5f * x - 0.5f * M) / T) - lz;
      };
      if (tid == 0 && P.entropy) P.entropy[r] = bad ? NAN : (empty || greedy) ? 0.0f : lz - s / z * kLn2;
      for (int j = tid; j < P.K; j += kT) {
        const long long at = static_cast<long long>(r) * P.K + j;
        if (j >= kT) {
          tok = P.token_ids[at];
          if (tok >= 0 && tok < P.V) tok_x = row.at(tok);
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
    ++r;
    if (r * P.nv >= S.end) break;
    p.row.set(P, r);
    p.v = 0;
    p.v_end = static_cast<int>(min(S.end - r * P.nv, P.nv));
    __syncthreads();
  }
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
  L.top = L.parts + slots * sizeof(float4);
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
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < ecah_token_logprobs_workspace_bytes())
    return ECAH_ERR_WORKSPACE;
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
  P.parts = reinterpret_cast<float4*>(ws + L.parts);
  P.part_top = reinterpret_cast<unsigned long long*>(ws + L.top);
  const int vec = a->dtype == ECAH_DTYPE_F32 ? 4 : 8;
  P.nv = (static_cast<long long>(P.V) + 2 * (vec - 1)) / vec;
  // a vector a thread at least; a row overlaps at most blocks / R + 2 of them, and its
  // alternatives are joined of at most kMaxParts
  long long blocks = std::min<long long>(static_cast<long long>(sms) * lp::kBlocks, (P.nv * P.R + lp::kT - 1) / lp::kT);
  blocks = std::min<long long>(blocks, (lp::kMaxParts - 2ll) * P.R);
  // Few rows: whole blocks to a row, so that no block ends one and begins another (128
  // rows with 20 alternatives: 26.5 us divided evenly, 21.3 us so).
  if (blocks >= 2ll * P.R) {
    const long long k = blocks / P.R;
    blocks = k * P.R;
    P.nv = (P.nv + k - 1) / k * k;
  }
  P.share = P.nv * P.R / blocks;
  P.more = static_cast<int>(P.nv * P.R % blocks);
  auto fn = a->dtype == ECAH_DTYPE_F16 ? lp::token_logprobs_kernel<ECAH_DTYPE_F16>
            : a->dtype == ECAH_DTYPE_BF16 ? lp::token_logprobs_kernel<ECAH_DTYPE_BF16>
                                          : lp::token_logprobs_kernel<ECAH_DTYPE_F32>;
  return launch_kernel(fn, dim3(static_cast<unsigned>(blocks)), lp::kT, static_cast<int>(sizeof(lp::Smem)),
                       reinterpret_cast<cudaStream_t>(stream), P) ? ECAH_OK : ECAH_ERR_LAUNCH;
}

}  // extern "C"
