// Attention of one new token per request over the paged key-value cache:
// ecah_paged_decode (contract in include/ecah_sampler.h).

#include <algorithm>

#include "host_util.h"
#include "paged.cuh"

namespace ecah {
namespace decode {

// The mathematics: softmax over a request's keys as one pass with a running
// reference m, o = sum_j 2^(s_j - m) v_j and l = sum_j 2^(s_j - m), s in units of
// log2; two such triples over disjoint keys join exactly, (m, l, o) + (m', l', o')
// = (M, l 2^(m-M) + l' 2^(m'-M), ...).
//
// Bound: HBM, every cached byte is used once by 4 G flops a value (G query heads
// to a KV head).  Up to 16 query heads of a KV head form the 16 rows of an
// m16n8k16 tensor-core product, so a KV row is read once for all of them: at
// 6.5 TB/s and head_dim 128 that is about 104 TFLOP/s of padded 16-bit products.
// tcgen05 wants 64 or 128 rows and would pad 8 to 16 times over; plain FMAs would
// need 26 Tfma/s for G = 8 beside the conversions.
//
// Split: a work unit is a tile of 64 keys of one (request, KV head, head tile).
// All units, in order, are divided evenly over the blocks by the lengths the
// device holds (no host read, so a captured launch serves any lengths); a
// (request, head) that spans several blocks is joined by the block that arrives
// last, in the order of the parts, so results do not depend on which that is.
//
// Inside a block each warp streams 16-key slices of its own through its own
// cp.async ring (no block barrier while streaming).

constexpr int kW = 4;                 // warps
constexpr int kT = kW * 32;
constexpr int kSlice = 16;            // keys per warp and step
constexpr int kTile = kW * kSlice;    // keys per work unit
constexpr int kRows = 16;             // query heads per head tile
constexpr int kMaxGroup = 32;         // parts joined at once
constexpr int kItemCost = 4;          // tiles of streaming that starting and joining an item takes
constexpr float kLazy = 8.0f;         // the reference moves when a score is 2^8 above it
constexpr float kLn2 = 0.6931471805599453f;

struct Params {
  const void* q;
  void* out;
  float* lse;
  const int* last_page_len;
  long long q_tok, q_head, o_tok, o_head;
  int hq, group, tiles_h;    // query heads, per KV head, head tiles per KV head
  float scale;               // sm_scale * log2 e
  unsigned* counters;        // [2 slots][2]: group and item arrivals, zero between launches
  float* part_ml;            // [slots][kRows][2]
  float* part_o;             // [slots][kRows][D]
  kv::Cache cache;
};

template <int D, bool E4M3>
struct Shape {
  static constexpr int kElem = E4M3 ? 1 : 2;
  static constexpr int kRowBytes = D * kElem;
  static constexpr int kChunks = kRowBytes / 16;          // 16-byte chunks of a row
  // Row strides in shared memory.  16-bit rows are read by ldmatrix: a stride of
  // an odd number of 16-byte units puts its 8 rows on different banks.  8-bit key
  // rows are read 8 bytes a lane, 4 rows to a half warp: stride 32 or 96 mod 128.
  static constexpr int kKStride = !E4M3 ? kRowBytes + 16
                                  : D % 128 == 32 || D % 128 == 96 ? D : D + 32;
  static constexpr int kVStride = kRowBytes + 16;
  static constexpr int kScaleBytes = E4M3 ? 2 * kSlice * 4 : 0;
  static constexpr int kStage = kSlice * (kKStride + kVStride) + kScaleBytes;
  // 2 blocks of 4 warps (3 for small rows) must hold about 100 KB in flight on an SM
  static constexpr int kStages = E4M3 ? (D <= 128 ? 4 : 3) : (D <= 64 ? 4 : D <= 128 ? 3 : 2);
  static constexpr int kWarpBytes = kStages * kStage;
  static constexpr int kSmem = kW * kWarpBytes;
  static constexpr int kBlocks = kSmem * 2 <= 220 * 1024 ? 2 : 1;   // per SM
  static_assert(kWarpBytes >= kRows * D * 4 + kRows * 8, "a warp's result fits its ring");
  static_assert(kStage % 16 == 0, "");
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// c += a b, 16 x 8 x 16; HT: the operands' 16-bit type
template <int HT>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (HT == ECAH_DTYPE_F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// two floats to packed 16-bit operands, lo in the low half
template <int HT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (HT == ECAH_DTYPE_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// two e4m3 codes (low and high byte) to f16, exactly
__device__ __forceinline__ uint32_t e4m3x2(uint32_t codes) {
  uint32_t r;
  asm("{ .reg .b16 t; cvt.u16.u32 t, %1; cvt.rn.f16x2.e4m3x2 %0, t; }" : "=r"(r) : "r"(codes));
  return r;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float lg2(float x) {
  float r;
  asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ long long request_len(const Params& P, int b, long long* first) {
  long long count;
  kv::page_range(P.cache, b, first, &count);
  if (count <= 0 || P.cache.num_pages <= 0) return 0;
  const long long len = (count - 1) * P.cache.page_size + min(max(P.last_page_len[b], 0), P.cache.page_size);
  return min(len, 0x7FFFFFFFll - kTile);
}

// Reads of a joined triple: from this block's shared memory, or of another
// block's part through L2.
struct FromShared {
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ float4 four(const float* p) { return *reinterpret_cast<const float4*>(p); }
};
struct FromParts {
  static __device__ __forceinline__ float one(const float* p) { return __ldcg(p); }
  static __device__ __forceinline__ float4 four(const float* p) { return __ldcg(reinterpret_cast<const float4*>(p)); }
};

// Arrival of this block on a counter; true for the last of `expect`, which
// leaves the counter at zero and sees the others' writes.
__device__ __forceinline__ bool arrive(unsigned* counter, int expect, int* flag) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    const unsigned n = atomicAdd(counter, 1u) + 1u;
    const bool last = n == static_cast<unsigned>(expect);
    if (last) *counter = 0u;
    *flag = last;
    __threadfence();
  }
  __syncthreads();
  return *flag != 0;
}

template <int DT, bool E4M3, int D>
__global__ void __launch_bounds__(kT, Shape<D, E4M3>::kBlocks) decode_kernel(const Params P) {
  using S = Shape<D, E4M3>;
  constexpr int HT = E4M3 ? static_cast<int>(ECAH_DTYPE_F16) : DT;   // operand type of the products
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long s_scan[kW];
  __shared__ long long s_start;          // prefix of tiles before s_req
  __shared__ int s_req, s_flag;
  __shared__ float s_f[kMaxGroup][kRows];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const kv::Cache& C = P.cache;
  const int per_req = C.heads * P.tiles_h;       // (head, head tile) pairs of a request

  // Total cost, then this block's share [begin, end) and its first request.  An
  // item (one head tile of one request) costs kItemCost units, then one a tile.
  auto tiles_of = [&](int b) -> long long {
    long long f;
    if (b >= C.batch) return 0;
    const long long len = request_len(P, b, &f);
    return len ? (len + kTile - 1) / kTile + kItemCost : 0;
  };
  long long sum = 0;
  for (int b = tid; b < C.batch; b += kT) sum += tiles_of(b);
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (lane == 0) s_scan[warp] = sum;
  __syncthreads();
  long long total = 0;
  for (int w = 0; w < kW; ++w) total += s_scan[w];
  total *= per_req;
  const long long blocks = min(static_cast<long long>(gridDim.x), total);
  const bool busy = blockIdx.x < blocks;
  const long long begin = busy ? blockIdx.x * total / blocks : 0, end = busy ? (blockIdx.x + 1ll) * total / blocks : 0;
  long long run = 0;
  for (int b0 = 0; busy && b0 < C.batch; b0 += kT) {
    const long long mine = tiles_of(b0 + tid);
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += v;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    long long before = run;
    for (int w = 0; w < kW; ++w) {
      if (w < warp) before += s_scan[w];
      run += s_scan[w];
    }
    const long long lo = (before + inc - mine) * per_req, hi = (before + inc) * per_req;
    if (begin >= lo && begin < hi) { s_req = b0 + tid; s_start = before + inc - mine; }
    if (begin < run * per_req) break;
  }
  __syncthreads();
  int req = busy ? s_req : 0;
  long long req_start = busy ? s_start * per_req : 0;       // first unit of the request
  long long at = begin;

  const uint32_t ring = smem_u32(smem) + warp * S::kWarpBytes;
  unsigned char* ring_p = smem + warp * S::kWarpBytes;

  while (at < end) {
    // the unit's request, head and head tile
    long long first;
    const long long len = request_len(P, req, &first);
    const long long nt = (len + kTile - 1) / kTile, cost = len ? nt + kItemCost : 0;
    if (at >= req_start + cost * per_req) { req_start += cost * per_req; ++req; continue; }
    const int pair = static_cast<int>((at - req_start) / cost);
    const long long item_start = req_start + pair * cost;
    const long long tile0 = item_start + kItemCost;           // unit of the item's first tile
    const int h = pair / P.tiles_h, ht = pair % P.tiles_h;
    const long long seg_end = min(end, item_start + cost);
    const long long t0 = max(at, tile0) - tile0;
    const int n = static_cast<int>(seg_end - tile0 - t0);
    at = seg_end;
    if (n <= 0) continue;                                     // only the item's first units: no tile
    const int rows = min(P.group - ht * kRows, kRows);        // query heads of this tile
    const int head0 = h * P.group + ht * kRows;

    // ---- query fragments
    uint32_t qf[D / 16][4];
    float rs0 = P.scale, rs1 = P.scale;                       // score scale of rows g and g + 8
    {
      const uint16_t* q0 = static_cast<const uint16_t*>(P.q) + req * P.q_tok + (head0 + g) * P.q_head;
      const uint16_t* q1 = q0 + 8 * P.q_head;
      const bool v0 = g < rows, v1 = g + 8 < rows;
      if (!E4M3) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int d = 16 * k + 2 * t;
          qf[k][0] = v0 ? *reinterpret_cast<const uint32_t*>(q0 + d) : 0u;
          qf[k][1] = v1 ? *reinterpret_cast<const uint32_t*>(q1 + d) : 0u;
          qf[k][2] = v0 ? *reinterpret_cast<const uint32_t*>(q0 + d + 8) : 0u;
          qf[k][3] = v1 ? *reinterpret_cast<const uint32_t*>(q1 + d + 8) : 0u;
        }
      } else {
        // The products run in f16 (e4m3 codes are exact there).  Each query head is
        // scaled by a power of two to a largest magnitude in [1, 2), so that bf16
        // queries fit its range; the power goes into the row's score scale.
        // Dimensions are dealt so that a lane's 8 consecutive codes of a key feed
        // its operands of two products: k index 2t, 2t+1, 2t+8, 2t+9 of product 2i
        // are dimensions 32 i + 8 t + 0..3, of product 2i + 1 + 4..7.
        uint4 w0[D / 32], w1[D / 32];
        float m0 = 0.0f, m1 = 0.0f;
        auto biggest = [](const uint4& w, float m) {
          const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            m = fmaxf(m, fmaxf(fabsf(DType<DT>::to_f32(u[i] & 0xFFFFu)), fabsf(DType<DT>::to_f32(u[i] >> 16))));
          return m;
        };
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          const int d = 32 * k + 8 * t;
          w0[k] = v0 ? *reinterpret_cast<const uint4*>(q0 + d) : uint4{0, 0, 0, 0};
          w1[k] = v1 ? *reinterpret_cast<const uint4*>(q1 + d) : uint4{0, 0, 0, 0};
          m0 = biggest(w0[k], m0);
          m1 = biggest(w1[k], m1);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          m0 = fmaxf(m0, __shfl_xor_sync(0xFFFFFFFFu, m0, o));
          m1 = fmaxf(m1, __shfl_xor_sync(0xFFFFFFFFu, m1, o));
        }
        // 2^-e and 2^e from the exponent field, kept within [2^-100, 2^100]
        const int e0 = min(max(static_cast<int>(__float_as_uint(m0) >> 23) - 127, -100), 100);
        const int e1 = min(max(static_cast<int>(__float_as_uint(m1) >> 23) - 127, -100), 100);
        const float d0 = __uint_as_float((127 - e0) << 23), d1 = __uint_as_float((127 - e1) << 23);
        rs0 *= __uint_as_float((127 + e0) << 23);
        rs1 *= __uint_as_float((127 + e1) << 23);
        auto half2of = [](uint32_t w, float f) {
          return pack2<ECAH_DTYPE_F16>(DType<DT>::to_f32(w & 0xFFFFu) * f, DType<DT>::to_f32(w >> 16) * f);
        };
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          qf[2 * k][0] = half2of(w0[k].x, d0);
          qf[2 * k][1] = half2of(w1[k].x, d1);
          qf[2 * k][2] = half2of(w0[k].y, d0);
          qf[2 * k][3] = half2of(w1[k].y, d1);
          qf[2 * k + 1][0] = half2of(w0[k].z, d0);
          qf[2 * k + 1][1] = half2of(w1[k].z, d1);
          qf[2 * k + 1][2] = half2of(w0[k].w, d0);
          qf[2 * k + 1][3] = half2of(w1[k].w, d1);
        }
      }
    }

    // ---- stream
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;

    // Lane l < 16 finds the key row of key l of a slice, lane 16 + l the value row.
    const kv::Side& side = lane < kSlice ? C.k : C.v;
    const long long key0 = t0 * kTile + warp * kSlice + (lane & 15);
    auto page_of = [&](int i) -> int {
      const long long j = key0 + static_cast<long long>(i) * kTile;
      return i < n && j < len
                 ? min(max(C.indices[first + static_cast<unsigned>(j) / static_cast<unsigned>(C.page_size)], 0), C.num_pages - 1) : -1;
    };
    int page = page_of(0);
    auto issue = [&](int i) {
      if (i < n) {
        const unsigned j = static_cast<unsigned>(key0 + static_cast<long long>(i) * kTile);
        const int pg = page, slot = static_cast<int>(j % static_cast<unsigned>(C.page_size));
        page = page_of(i + 1);
        const unsigned char* row = static_cast<const unsigned char*>(side.base);
        if (pg >= 0) row += (pg * side.page + slot * side.slot + h * side.head) * S::kElem;
        const unsigned live = __ballot_sync(0xFFFFFFFFu, pg >= 0);
        const uint32_t st = ring + (i % S::kStages) * S::kStage;
        const unsigned long long rp = reinterpret_cast<unsigned long long>(row);
#pragma unroll
        for (int c0 = 0; c0 < kSlice * S::kChunks; c0 += 32) {
          const int c = c0 + lane, r = c / S::kChunks, col = c % S::kChunks;
          const unsigned long long kr = __shfl_sync(0xFFFFFFFFu, rp, r), vr = __shfl_sync(0xFFFFFFFFu, rp, r + kSlice);
          const int bytes = (live >> r) & 1u ? 16 : 0;       // past the length: zeros
          cp16(st + r * S::kKStride + col * 16, reinterpret_cast<const void*>(kr + col * 16), bytes);
          cp16(st + kSlice * S::kKStride + r * S::kVStride + col * 16, reinterpret_cast<const void*>(vr + col * 16), bytes);
        }
        if (E4M3) {
          const float* sc = side.scale;
          if (pg >= 0) sc += (static_cast<long long>(pg) * C.heads + h) * C.page_size + slot;
          cp4(st + kSlice * (S::kKStride + S::kVStride) + lane * 4, sc, pg >= 0 ? 4 : 0);
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) issue(i);

    for (int i = 0; i < n; ++i) {
      issue(i + S::kStages - 1);
      cp_wait<S::kStages - 1>();
      __syncwarp();
      const long long base = (t0 + i) * kTile + warp * kSlice;
      if (base < len) {
        const uint32_t ks = ring + (i % S::kStages) * S::kStage, vs = ks + kSlice * S::kKStride;
        float s[2][4] = {};                                   // keys 0-7 and 8-15
        if (!E4M3) {
          float s2[2][4] = {};                                // second chain: half the latency
          const uint32_t a = ks + ((lane & 7) + (lane >> 4) * 8) * S::kKStride + ((lane >> 3) & 1) * 16;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t b[4];
            ldsm4(b, a + k * 32);
            mma<HT>(k & 1 ? s2[0] : s[0], qf[k], b[0], b[1]);
            mma<HT>(k & 1 ? s2[1] : s[1], qf[k], b[2], b[3]);
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) { s[0][x] += s2[0][x]; s[1][x] += s2[1][x]; }
        } else {
          float s2[2][4] = {};
          const unsigned char* kp = ring_p + (i % S::kStages) * S::kStage + g * S::kKStride + 8 * t;
#pragma unroll
          for (int k = 0; k < D / 32; ++k) {
            const uint2 a = *reinterpret_cast<const uint2*>(kp + 32 * k);
            const uint2 b = *reinterpret_cast<const uint2*>(kp + 8 * S::kKStride + 32 * k);
            mma<HT>(s[0], qf[2 * k], e4m3x2(a.x), e4m3x2(a.x >> 16));
            mma<HT>(s[1], qf[2 * k], e4m3x2(b.x), e4m3x2(b.x >> 16));
            mma<HT>(s2[0], qf[2 * k + 1], e4m3x2(a.y), e4m3x2(a.y >> 16));
            mma<HT>(s2[1], qf[2 * k + 1], e4m3x2(b.y), e4m3x2(b.y >> 16));
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) { s[0][x] += s2[0][x]; s[1][x] += s2[1][x]; }
        }
        // scores in log2 units; w: the exponent of the value's weight.  An e4m3
        // value's scale goes into its weight through the exponent, which keeps the
        // f16 weights at or below 2^8 whatever the scales are.
        float w[2][4];
        float2 vsc[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          s[x][0] *= rs0; s[x][1] *= rs0; s[x][2] *= rs1; s[x][3] *= rs1;
          if (E4M3) {
            const float* sc = reinterpret_cast<const float*>(ring_p + (i % S::kStages) * S::kStage + kSlice * (S::kKStride + S::kVStride));
            const float2 kx = *reinterpret_cast<const float2*>(sc + 8 * x + 2 * t);
            vsc[x] = *reinterpret_cast<const float2*>(sc + kSlice + 8 * x + 2 * t);
            s[x][0] *= kx.x; s[x][1] *= kx.y; s[x][2] *= kx.x; s[x][3] *= kx.y;
            const float a = max_nan(lg2(vsc[x].x), -90.0f), b = max_nan(lg2(vsc[x].y), -90.0f);
            w[x][0] = s[x][0] + a; w[x][1] = s[x][1] + b; w[x][2] = s[x][2] + a; w[x][3] = s[x][3] + b;
          } else {
#pragma unroll
            for (int y = 0; y < 4; ++y) w[x][y] = s[x][y];
          }
        }
        if (base + kSlice > len) {
          const int live = static_cast<int>(len - base);
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 4; ++y)
              if (8 * x + 2 * t + (y & 1) >= live) s[x][y] = w[x][y] = -INFINITY;
        }
        float n0 = fmaxf(fmaxf(w[0][0], w[0][1]), fmaxf(w[1][0], w[1][1]));
        float n1 = fmaxf(fmaxf(w[0][2], w[0][3]), fmaxf(w[1][2], w[1][3]));
        if (__any_sync(0xFFFFFFFFu, n0 > m0 + kLazy || n1 > m1 + kLazy)) {
#pragma unroll
          for (int x = 1; x < 4; x <<= 1) {
            n0 = fmaxf(n0, __shfl_xor_sync(0xFFFFFFFFu, n0, x));
            n1 = fmaxf(n1, __shfl_xor_sync(0xFFFFFFFFu, n1, x));
          }
          n0 = fmaxf(n0, m0);
          n1 = fmaxf(n1, m1);
          const float f0 = m0 == n0 ? 1.0f : ex2_approx(m0 - n0), f1 = m1 == n1 ? 1.0f : ex2_approx(m1 - n1);
          l0 *= f0;
          l1 *= f1;
#pragma unroll
          for (int x = 0; x < D / 8; ++x) { o[x][0] *= f0; o[x][1] *= f0; o[x][2] *= f1; o[x][3] *= f1; }
          m0 = n0;
          m1 = n1;
        }
        const float r0 = m0 == -INFINITY ? 0.0f : m0, r1 = m1 == -INFINITY ? 0.0f : m1;
        float p[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          p[x][0] = ex2_approx(w[x][0] - r0);
          p[x][1] = ex2_approx(w[x][1] - r0);
          p[x][2] = ex2_approx(w[x][2] - r1);
          p[x][3] = ex2_approx(w[x][3] - r1);
          if (E4M3) {
            l0 += ex2_approx(s[x][0] - r0) + ex2_approx(s[x][1] - r0);
            l1 += ex2_approx(s[x][2] - r1) + ex2_approx(s[x][3] - r1);
            if (vsc[x].x == 0.0f) p[x][0] = p[x][2] = 0.0f;
            if (vsc[x].y == 0.0f) p[x][1] = p[x][3] = 0.0f;
          } else {
            l0 += p[x][0] + p[x][1];
            l1 += p[x][2] + p[x][3];
          }
        }
        const uint32_t pf[4] = {pack2<HT>(p[0][0], p[0][1]), pack2<HT>(p[0][2], p[0][3]),
                                pack2<HT>(p[1][0], p[1][1]), pack2<HT>(p[1][2], p[1][3])};
        const uint32_t va = vs + ((lane & 7) + ((lane >> 3) & 1) * 8) * S::kVStride + (lane >> 4) * 16;
        if (!E4M3) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t b[4];
            ldsm4_t(b, va + k * 32);
            mma<HT>(o[2 * k], pf, b[0], b[1]);
            mma<HT>(o[2 * k + 1], pf, b[2], b[3]);
          }
        } else {
          // 16-bit units of the transposed load hold two dimensions' codes: of two keys'
          // units, bytes 0 and 2 are the even dimension's, 1 and 3 the odd one's
#pragma unroll
          for (int k = 0; k < D / 32; ++k) {
            uint32_t b[4];
            ldsm4_t(b, va + k * 32);
#pragma unroll
            for (int x = 0; x < 4; ++x) b[x] = __byte_perm(b[x], 0u, 0x3120);
            mma<HT>(o[4 * k], pf, e4m3x2(b[0]), e4m3x2(b[1]));
            mma<HT>(o[4 * k + 1], pf, e4m3x2(b[0] >> 16), e4m3x2(b[1] >> 16));
            mma<HT>(o[4 * k + 2], pf, e4m3x2(b[2]), e4m3x2(b[3]));
            mma<HT>(o[4 * k + 3], pf, e4m3x2(b[2] >> 16), e4m3x2(b[3] >> 16));
          }
        }
      }
      __syncwarp();
    }
    cp_wait<0>();
    __syncwarp();

    // ---- join the warps: each leaves (m, l, o) in its ring
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, x);
      l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, x);
    }
    float* ro = reinterpret_cast<float*>(ring_p);
    float* rml = ro + kRows * D;
    if (t == 0) {
      rml[2 * g] = m0; rml[2 * g + 1] = l0;
      rml[2 * (g + 8)] = m1; rml[2 * (g + 8) + 1] = l1;
    }
#pragma unroll
    for (int k = 0; k < D / 8; ++k) {
      if (!E4M3) {
        *reinterpret_cast<float2*>(ro + g * D + 8 * k + 2 * t) = make_float2(o[k][0], o[k][1]);
        *reinterpret_cast<float2*>(ro + (g + 8) * D + 8 * k + 2 * t) = make_float2(o[k][2], o[k][3]);
      } else if ((k & 1) == 0) {     // tiles k (even dimensions) and k + 1 (odd ones) of 16 dimensions
        *reinterpret_cast<float4*>(ro + g * D + 8 * k + 4 * t) = make_float4(o[k][0], o[k + 1][0], o[k][1], o[k + 1][1]);
        *reinterpret_cast<float4*>(ro + (g + 8) * D + 8 * k + 4 * t) = make_float4(o[k][2], o[k + 1][2], o[k][3], o[k + 1][3]);
      }
    }
    __syncthreads();

    // parts of this item: the blocks whose shares overlap its tiles
    const long long a = ((tile0 + 1) * blocks - 1) / total, z = ((tile0 + nt) * blocks - 1) / total;
    const int parts = static_cast<int>(z - a) + 1, part = static_cast<int>(blockIdx.x - a);
    auto slot_of = [&](int p) -> long long { return p == 0 ? 2 * a + 1 : 2 * (a + p); };

    // combine `count` (m, l, o) triples into the output or a part's slot
    auto combine = [&](auto from, int count, auto ml_of, auto o_of, long long to) {
      using From = decltype(from);
      if (tid < rows) {
        float m = -INFINITY, l = 0.0f;
        for (int p = 0; p < count; ++p) m = fmaxf(m, From::one(ml_of(p) + 2 * tid));
        for (int p = 0; p < count; ++p) {
          const float mp = From::one(ml_of(p) + 2 * tid);
          const float f = mp == -INFINITY ? 0.0f : ex2_approx(mp - m);
          l = fmaf(From::one(ml_of(p) + 2 * tid + 1), f, l);
          s_f[p][tid] = f;
        }
        if (to >= 0) {
          P.part_ml[(to * kRows + tid) * 2] = m;
          P.part_ml[(to * kRows + tid) * 2 + 1] = l;
        } else {
          // a sum of zero (no key has mass) gives zeros
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
          for (int p = 0; p < count; ++p) s_f[p][tid] *= inv;
          if (P.lse) P.lse[static_cast<long long>(req) * P.hq + head0 + tid] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
        }
      }
      __syncthreads();
      for (int e = tid * 4; e < rows * D; e += kT * 4) {
        const int r = e / D, d = e % D;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int p = 0; p < count; ++p) {
          const float4 x = From::four(o_of(p) + e);
          const float f = s_f[p][r];
          v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w);
        }
        if (to >= 0) {
          *reinterpret_cast<float4*>(P.part_o + to * kRows * D + e) = v;
        } else {
          const uint2 w = make_uint2(pack2<DT>(v.x, v.y), pack2<DT>(v.z, v.w));
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(P.out) + req * P.o_tok + (head0 + r) * P.o_head + d) = w;
        }
      }
    };
    auto warp_ml = [&](int w) -> const float* { return reinterpret_cast<const float*>(smem + w * S::kWarpBytes) + kRows * D; };
    auto warp_o = [&](int w) -> const float* { return reinterpret_cast<const float*>(smem + w * S::kWarpBytes); };
    combine(FromShared(), kW, warp_ml, warp_o, parts == 1 ? -1 : slot_of(part));

    if (parts > 1) {
      // joined in one step, or in groups of about sqrt(parts) first
      int gs = parts;
      if (parts > kMaxGroup) { gs = 1; while (gs * gs < parts) ++gs; }
      const int groups = (parts + gs - 1) / gs, grp = part / gs, p0 = grp * gs, in_grp = min(gs, parts - p0);
      bool last = arrive(P.counters + 2 * slot_of(p0), in_grp, &s_flag);
      if (last) {
        combine(FromParts(), in_grp, [&](int p) { return P.part_ml + slot_of(p0 + p) * kRows * 2; },
                [&](int p) { return P.part_o + slot_of(p0 + p) * kRows * D; }, groups == 1 ? -1 : slot_of(p0));
        if (groups > 1 && arrive(P.counters + 2 * slot_of(0) + 1, groups, &s_flag))
          combine(FromParts(), groups, [&](int p) { return P.part_ml + slot_of(p * gs) * kRows * 2; },
                  [&](int p) { return P.part_o + slot_of(p * gs) * kRows * D; }, -1);
      }
    }
    __syncthreads();       // the rings are free again
  }

  // requests without tokens: zeros, spread over the blocks
  for (int b = blockIdx.x; b < C.batch; b += gridDim.x) {
    long long f;
    if (request_len(P, b, &f) != 0) continue;
    for (int i = tid; i < P.hq * D; i += kT)
      static_cast<uint16_t*>(P.out)[b * P.o_tok + (i / D) * P.o_head + i % D] = 0;
    if (P.lse)
      for (int i = tid; i < P.hq; i += kT) P.lse[static_cast<long long>(b) * P.hq + i] = -INFINITY;
  }
}

struct Variant {
  void (*fn)(const Params);
  int smem, blocks;
};

template <int DT, bool E4M3>
static Variant variant_for(int D) {
  switch (D) {
#define ECAH_D(N) case N: return Variant{decode_kernel<DT, E4M3, N>, Shape<N, E4M3>::kSmem, Shape<N, E4M3>::kBlocks};
    ECAH_D(64) ECAH_D(96) ECAH_D(128) ECAH_D(192)
#undef ECAH_D
    default: return Variant{decode_kernel<DT, E4M3, 256>, Shape<256, E4M3>::kSmem, Shape<256, E4M3>::kBlocks};
  }
}

constexpr int kMaxBlocksPerSm = 2;

// Workspace: counters, then the parts' (m, l), then their sums.  A block has at
// most two parts of items it shares with others, whatever the batch is.
struct Layout {
  size_t ml, o, total;
};

static Layout layout(int sms, int D) {
  const size_t slots = 2 * static_cast<size_t>(sms) * kMaxBlocksPerSm + 2;
  Layout L;
  L.ml = (slots * 2 * sizeof(unsigned) + 255) / 256 * 256;
  L.o = L.ml + slots * kRows * 2 * sizeof(float);
  L.total = L.o + slots * kRows * D * sizeof(float);
  return L;
}

}  // namespace decode
}  // namespace ecah

using namespace ecah;

extern "C" {

size_t ecah_paged_decode_workspace_bytes(int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim) {
  if (batch < 0 || num_kv_heads < 1 || num_qo_heads < 1 || num_qo_heads % num_kv_heads || !kv::head_dim_ok(head_dim) ||
      device_sms() <= 0)
    return 0;
  return decode::layout(device_sms(), head_dim).total;
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
  const int sms = device_sms();
  if (sms <= 0) return ECAH_ERR_LAUNCH;
  decode::Params P = {};
  P.q = a->q; P.out = a->out; P.lse = a->lse; P.last_page_len = a->kv_last_page_len;
  P.q_tok = a->q_token_stride; P.q_head = a->q_head_stride;
  P.o_tok = a->out_token_stride; P.o_head = a->out_head_stride;
  P.hq = a->num_qo_heads; P.group = a->num_qo_heads / c.num_kv_heads;
  P.tiles_h = (P.group + decode::kRows - 1) / decode::kRows;
  P.scale = a->sm_scale * kLog2e;
  P.cache = kv::make_cache(c);
  const decode::Layout L = decode::layout(sms, c.head_dim);
  unsigned char* ws = static_cast<unsigned char*>(a->workspace);
  P.counters = reinterpret_cast<unsigned*>(ws);
  P.part_ml = reinterpret_cast<float*>(ws + L.ml);
  P.part_o = reinterpret_cast<float*>(ws + L.o);
  const bool e4m3 = c.kv_dtype == ECAH_KV_E4M3, f16 = a->dtype == ECAH_DTYPE_F16;
  const decode::Variant v = f16 ? (e4m3 ? decode::variant_for<ECAH_DTYPE_F16, true>(c.head_dim) : decode::variant_for<ECAH_DTYPE_F16, false>(c.head_dim))
                                : (e4m3 ? decode::variant_for<ECAH_DTYPE_BF16, true>(c.head_dim) : decode::variant_for<ECAH_DTYPE_BF16, false>(c.head_dim));
  // no more blocks than tiles the listed pages can hold (and one for the empty requests)
  const double most = (static_cast<double>(c.num_indices) * c.page_size / decode::kTile + c.batch * (1.0 + decode::kItemCost)) * c.num_kv_heads * P.tiles_h + 1;
  const int blocks = static_cast<int>(std::min(most, static_cast<double>(sms * v.blocks)));
  return launch_kernel(v.fn, dim3(blocks), decode::kT, v.smem, reinterpret_cast<cudaStream_t>(stream), P) ? ECAH_OK : ECAH_ERR_LAUNCH;
}

}  // extern "C"
