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
// Bound: HBM; a cached byte is used once, by 2 G to 4 G flops (G query heads to a
// KV head).  The products run transposed on m16n8k16 tensor-core instructions, 16
// keys by 8 query heads, so a KV row is read once for up to 16 heads and nothing
// is padded beyond 8: S^T = K Q^T and O^T = V^T P^T.  At 6.5 TB/s and head_dim 128
// that is 52 TFLOP/s of 16-bit products for 8 heads.  tcgen05 would want its 128
// rows of keys staged as whole tiles and the softmax through TMEM for the same
// memory-bound rate; plain FMAs would need 26 Tfma/s beside the conversions.
//
// Split: a block's 4 warps take 4, 2 or 1 KV heads of a request, with 16-key slices
// of the same keys: an item is (request, group of KV heads, head tile), a work unit
// 64 rows of it (16 keys of 4 heads to 64 keys of one).  Neighbouring heads of a token
// lie side by side, so several of them make longer runs of DRAM.  All units, in order,
// are divided evenly over the blocks by the lengths the device holds (no host read, so
// a captured launch serves any lengths); an item that spans several blocks is joined by
// the block that arrives last, in the order of the parts, so results do not depend on
// which that is.
//
// Inside a block each warp streams 16-key slices of its own through its own ring in
// shared memory, filled by its threads' copies or by the copy engine (no block barrier
// while streaming).
//
// Measured on one B200, device time of graph replays: 4 requests of 100 001 to 131 072
// tokens, 32/8 heads of 128, bf16 302 us (6.5 TB/s), the same over an e4m3 cache 178 us
// (5.7 TB/s), with heads of 64 and 96 in bf16 174 and 258 us (5.6 TB/s); 64 requests of 1 to
// 16 384 tokens over an e4m3 cache 57 us (4.7 TB/s); 128 requests of 128 to 512 tokens,
// 16/2 heads, f16 13.7 us; one request of 512 9.2 us.
// What bounds the last three: finding the share (1.3 us), the first pages and rows (2
// us), and joining (1.5 us a block, 5 us where the item was divided).

constexpr int kW = 4;                 // warps
constexpr int kT = kW * 32;
constexpr int kSlice = 16;            // keys per warp and step
constexpr int kTile = kW * kSlice;    // rows (keys of a head) per work unit
constexpr int kMaxGroup = 25;         // parts joined at once: 25 * 25 blocks to an item at most
constexpr int kMaxRows = 32;          // query heads of an item
// Tiles of streaming that starting and joining an item takes (64 ragged requests over
// e4m3: 84 us with 2, 72 with 4, 77 with 8, and 139 without the term).
constexpr int kItemCost = 4;
constexpr int kWhole = 8;             // items of up to so many tiles are not divided, ...
constexpr int kWholeAlone = 4;        // ... or so many where there is a block for every tile (one
                                      // request of 512: 8.8 us divided, 10.4 whole; 128: 18.0, 13.2)
constexpr int kTries = 1 << 20;       // of a wait for copies: more than one in flight can need
// The reference moves when a score passes its last place by 2^kLazy.  Where the weights
// are f16 operands it then lies 2^kLift below the largest: weights reach 2^15, and one is
// lost to f16's smallest only at 2^-32 of the largest (2^-25 without the lift: a long tail
// of such weights is in the denominator, so it has to be in the sum).
constexpr float kLazy = 8.0f;
constexpr float kLift = 7.0f;
constexpr float kLn2 = 0.6931471805599453f;

// One side of the cache in 16-byte units from its base.
struct Side16 {
  const unsigned char* base;
  unsigned page, slot, head;
  const float* scale;
};

struct Params {
  const void* q;
  void* out;
  float* lse;
  const int* last_page_len;
  long long q_tok, q_head, o_tok, o_head;
  int hq, group, tiles_h;    // query heads, per KV head, head tiles per KV head
  int wh;                    // KV heads of an item: 1, 2 or 4
  int page_shift;            // log2 page_size, or -1
  int tries;                 // of a wait for the copy engine
  float scale;               // sm_scale * log2 e
  unsigned* counters;        // [2 slots][2]: group and item arrivals, zero between launches
  float2* part_ml;           // [slots][wh rows]
  float* part_o;             // [slots][wh rows][D]
  Side16 k, v;
  kv::Cache cache;
};

template <int D, bool E4M3, int NT, bool BULK>
struct Shape {
  static constexpr int kRows = 8 * NT;                    // query heads per head tile
  static constexpr int kElem = E4M3 ? 1 : 2;
  static constexpr int kRowBytes = D * kElem;
  static constexpr int kChunks = kRowBytes / 16;          // 16-byte chunks of a row
  // Row strides in shared memory.  ldmatrix reads 8 rows at once: a stride of an
  // odd number of 16-byte units puts them on different banks.  8-bit key rows are
  // read 8 bytes a lane, 4 rows to a half warp: stride 32 or 96 mod 128.
  static constexpr int kKStride = !E4M3 ? kRowBytes + 16
                                  : D % 128 == 32 || D % 128 == 96 ? D : D + 32;
  static constexpr int kVStride = kRowBytes + 16;
  static constexpr int kScaleBytes = E4M3 ? 2 * kSlice * 4 : 0;
  static constexpr int kStage = kSlice * (kKStride + kVStride) + kScaleBytes;
  // Blocks of an SM and stages of a warp's ring: 65 to 130 KB in flight on an SM
  // (6.5 TB/s over 148 SMs at about 1 us wants 45 KB) and 8 to 16 warps.
  static constexpr int kStages = E4M3 ? (D <= 96 ? 4 : 3) : BULK || D == 256 ? 2 : 3;
  static constexpr int kOStride = D + 4;                  // of a warp's result: 8 heads on 8 bank quads
  static constexpr int kWarpBytes = kStages * kStage;
  static constexpr int kSmem = kW * kWarpBytes;
  static constexpr int kResult = kRows * kOStride * 4 + kRows * 8;   // a warp's (m, l, o)
  static constexpr int kStatic = 256 + kT * 8 + 1024;
  static constexpr int kFit = (227 * 1024) / (kSmem + kStatic);
  static constexpr int kRegs = 50 + D / 4 * NT + D / 8 * NT;   // about: results, queries and the rest
  static constexpr int kByRegs = kRegs <= 110 ? 4 : kRegs <= 160 ? 3 : kRegs <= 215 ? 2 : 1;
  static constexpr int kBlocks = kFit < kByRegs ? kFit : kByRegs;
  static_assert(kBlocks >= 1 && kBlocks <= 4, "");
  static_assert(kWarpBytes >= kResult + kMaxGroup * kMaxRows * 8, "a warp's result and the join's factors fit its ring");
  static_assert(kStage % 16 == 0, "");
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
// One row of the cache to shared memory by the copy engine, counted by a barrier.
__device__ __forceinline__ void copy_row(uint32_t dst, const void* src, int bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void bar_init(uint32_t bar) { asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Waits for a phase of the barrier; false after `most` tries (each may itself wait).
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, int most) {
  for (int tries = 0; tries < most; ++tries) {
    uint32_t done;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
  }
  return false;
}
// Orders this thread's ordinary accesses to shared memory before later copies into it.
__device__ __forceinline__ void fence_copies() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void cp4_or_zero(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
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
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
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

// four e4m3 codes to f16, exactly: bytes 0 and 1, bytes 2 and 3
__device__ __forceinline__ void e4m3x4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }"
      : "=r"(lo), "=r"(hi) : "r"(codes));
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
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Tokens of request b and its first entry in the page list (the launcher has seen
// that there are fewer than 2^31 entries and units of work).
__device__ __forceinline__ int request_len(const Params& P, int b, int* first) {
  const int most = static_cast<int>(P.cache.num_indices);
  const int lo = min(max(P.cache.indptr[b], 0), most), hi = min(max(P.cache.indptr[b + 1], lo), most);
  *first = lo;
  if (hi <= lo || P.cache.num_pages <= 0) return 0;
  const long long len = static_cast<long long>(hi - lo - 1) * P.cache.page_size + min(max(P.last_page_len[b], 0), P.cache.page_size);
  return static_cast<int>(min(len, 0x7FFFFFFFll - kTile));
}

// Reads of a joined triple: from this block's shared memory, or of another
// block's part through L2.
struct FromShared {
  static __device__ __forceinline__ float2 two(const float2* p) { return *p; }
  static __device__ __forceinline__ float4 four(const float* p) { return *reinterpret_cast<const float4*>(p); }
};
struct FromParts {
  static __device__ __forceinline__ float2 two(const float2* p) { return __ldcg(p); }
  static __device__ __forceinline__ float4 four(const float* p) { return __ldcg(reinterpret_cast<const float4*>(p)); }
};

// Arrival of this block on a counter; true for the last of `expect`, which
// leaves the counter at zero and sees the others' writes.
__device__ __forceinline__ bool arrive(unsigned* counter, int expect, int* flag) {
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned n;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(n) : "l"(counter) : "memory");
    const bool last = n + 1u == static_cast<unsigned>(expect);
    if (last) *counter = 0u;
    *flag = last;
  }
  __syncthreads();
  return *flag != 0;
}

template <int DT, bool E4M3, int D, int NT, bool BULK>
__global__ void __launch_bounds__(kT, Shape<D, E4M3, NT, BULK>::kBlocks) decode_kernel(const Params P) {
  using S = Shape<D, E4M3, NT, BULK>;
  constexpr int kRows = S::kRows;
  constexpr int HT = E4M3 ? static_cast<int>(ECAH_DTYPE_F16) : DT;   // operand type of the products
  constexpr float lift = HT == ECAH_DTYPE_F16 ? kLift : 0.0f;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ unsigned s_scan[kW];
  __shared__ unsigned s_start[2];        // first unit of s_req
  __shared__ int s_req[2], s_flag;       // requests of the share's edges
  __shared__ int s_len[kT], s_first[kT];
  __shared__ unsigned long long s_bar[kW][S::kStages];
  __shared__ int s_failed;               // a wait for copies ran out: this block's results are NaN from then on
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // the join's (m, l) and factors: behind the first warp's result in its ring
  float2(*s_ml)[kMaxRows] = reinterpret_cast<float2(*)[kMaxRows]>(smem + S::kResult);
  const int wh = P.wh, sub = warp & (wh - 1), tile = kTile / wh;   // KV heads, this warp's, keys of a unit
  const int slice0 = (warp / wh) * kSlice;                         // this warp's keys of a unit
  const int g = lane >> 2, t = lane & 3;
  const kv::Cache& C = P.cache;
  const int per_req = C.heads / wh * P.tiles_h;  // items of a request

  grid_start();

  // Total cost, then this block's share.  An item costs kItemCost units, then one a
  // tile; the first `more` blocks take share + 1 units, the others share.
  // A batch of up to kT requests leaves its lengths in shared memory.
  const bool kept = C.batch <= kT;
  auto look = [&](int b, int* first) -> int {
    if (!kept) return request_len(P, b, first);
    *first = s_first[b];
    return s_len[b];
  };
  auto cost_of = [&](int len) { return len ? (len + tile - 1) / tile + kItemCost : 0; };
  unsigned mine = 0, total = 0;                               // mine: of request tid, or of this thread's requests
  for (int b = tid; b < C.batch; b += kT) {
    int f;
    const int len = request_len(P, b, &f);
    if (kept) { s_len[b] = len; s_first[b] = f; }
    mine += cost_of(len);
  }
  unsigned inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) s_scan[warp] = inc;
  if (tid < 2) s_req[tid] = -1;
  if (BULK && tid == 0) s_failed = 0;
  __syncthreads();
  unsigned before = 0;
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  total *= per_req;
  const unsigned blocks = min(gridDim.x, total);
  const bool busy = blockIdx.x < blocks;
  const unsigned share = busy ? total / blocks : 1, more = total - share * blocks;
  const unsigned whole = share > 1 ? kWhole : kWholeAlone;
  unsigned edge[2] = {0, 0};
  if (busy) {
    edge[0] = blockIdx.x * share + min(blockIdx.x, more);
    edge[1] = edge[0] + share + (blockIdx.x < more);
  }
  // the requests of the share's edges
  unsigned run = 0;
  for (int b0 = 0; busy && b0 < C.batch; b0 += kT) {
    if (!kept) {                                              // the scan again, by requests in order
      int f;
      mine = b0 + tid < C.batch ? cost_of(request_len(P, b0 + tid, &f)) : 0;
      inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += v;
      }
      __syncthreads();
      if (lane == 31) s_scan[warp] = inc;
      __syncthreads();
      before = run;
      for (int w = 0; w < kW; ++w) {
        if (w < warp) before += s_scan[w];
        run += s_scan[w];
      }
    }
    const unsigned lo = (before + inc - mine) * per_req, hi = (before + inc) * per_req;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (edge[e] >= lo && edge[e] < hi) { s_req[e] = b0 + tid; s_start[e] = lo; }
    if (!kept && edge[1] < run * per_req) break;
  }
  __syncthreads();
  // A share's edge inside a short item moves to the item's nearer end: joining its
  // parts would take longer than streaming it.
  auto settle = [&](int e) -> unsigned {
    if (!busy || s_req[e] < 0) return edge[e];                // the end of all
    int f;
    const unsigned nt = (look(s_req[e], &f) + tile - 1) / tile, cost = nt + kItemCost;
    if (nt > whole) return edge[e];
    const unsigned into = (edge[e] - s_start[e]) % cost;
    return edge[e] - into + (2 * into < cost ? 0 : cost);
  };
  unsigned at = settle(0);
  const unsigned end = settle(1);
  int req = busy ? s_req[0] : 0;
  unsigned req_start = busy ? s_start[0] : 0;                 // first unit of the request

  const uint32_t ring = smem_u32(smem) + warp * S::kWarpBytes;
  unsigned char* ring_p = smem + warp * S::kWarpBytes;
  const uint32_t bars = smem_u32(s_bar[warp]);
  uint32_t phase = 0;                            // of each stage's barrier
  bool failed = false;                           // a wait ran out: the warp copies nothing more
  if (BULK && lane == 0) {
    for (int i = 0; i < S::kStages; ++i) bar_init(bars + 8 * i);
    fence_copies();
  }
  __syncwarp();

  while (at < end && req < C.batch) {
    // the unit's request, head and head tile
    int first;
    const int len = look(req, &first);
    const unsigned nt = (len + tile - 1) / tile, cost = len ? nt + kItemCost : 0;
    if (at >= req_start + cost * per_req) { req_start += cost * per_req; ++req; continue; }
    const unsigned pair = (at - req_start) / cost, item_start = req_start + pair * cost;
    const unsigned tile0 = item_start + kItemCost;            // unit of the item's first tile
    const int h0 = pair / P.tiles_h * wh, ht = pair % P.tiles_h, h = h0 + sub;
    const unsigned seg_end = min(end, item_start + cost);
    const int t0 = static_cast<int>(max(at, tile0) - tile0);
    const int n = static_cast<int>(seg_end) - static_cast<int>(tile0) - t0;
    at = seg_end;
    if (n <= 0) continue;                                     // only the item's first units: no tile
    const int steps = BULK && failed ? 0 : n;
    const int rows = min(P.group - ht * kRows, kRows);        // query heads of this tile
    const int head0 = h * P.group + ht * kRows;

    // ---- stream: the first slices
    // Lane l < 16 finds the key row of key l of a slice, lane 16 + l the value row.
    const Side16& side = lane < kSlice ? P.k : P.v;
    const unsigned head_off = h * side.head;
    const unsigned key0 = static_cast<unsigned>(t0) * tile + slice0 + (lane & 15);
    const int* pages = C.indices + first;
    auto nth_page = [&](unsigned j) { return P.page_shift >= 0 ? j >> P.page_shift : j / static_cast<unsigned>(C.page_size); };
    auto page_of = [&](int i) -> int {
      const unsigned j = key0 + static_cast<unsigned>(i) * tile;
      return i < steps && j < static_cast<unsigned>(len) ? min(max(pages[nth_page(j)], 0), C.num_pages - 1) : -1;
    };
    int page = page_of(0), page_after = page_of(1);           // two slices ahead: an L2 read away
    // ---- the queries, asked for while the pages come and before the stream fills the memory's queues: heads
    // 8 x + g, as the products' second operand takes them (e4m3: 8 dimensions a load)
    uint32_t qf[NT][D / 16][2];
    uint4 qw[NT][E4M3 ? D / 32 : 1];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const bool live = 8 * x + g < rows;
      const uint16_t* q = static_cast<const uint16_t*>(P.q) + req * P.q_tok + (head0 + 8 * x + g) * P.q_head;
      if (!E4M3) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          qf[x][k][0] = live ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 2 * t) : 0u;
          qf[x][k][1] = live ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 2 * t + 8) : 0u;
        }
      } else {
#pragma unroll
        for (int k = 0; k < D / 32; ++k)
          qw[x][k] = live ? *reinterpret_cast<const uint4*>(q + 32 * k + 8 * t) : uint4{0, 0, 0, 0};
      }
    }

    auto issue = [&](int i) {
      if (i < steps) {
        const unsigned j = key0 + static_cast<unsigned>(i) * tile;
        const int pg = page;
        const unsigned slot = j - nth_page(j) * static_cast<unsigned>(C.page_size);
        page = page_after;
        page_after = page_of(i + 2);
        const unsigned off = pg < 0 ? 0u : pg * side.page + slot * side.slot + head_off;
        const unsigned live = __ballot_sync(0xFFFFFFFFu, pg >= 0);
        const uint32_t st = ring + (i % S::kStages) * S::kStage, bar = bars + 8 * (i % S::kStages);
        if (BULK) {
          const uint32_t row = st + (lane < kSlice ? lane * S::kKStride : kSlice * S::kKStride + (lane - kSlice) * S::kVStride);
          if (lane == 0) bar_expect(bar, __popc(live) * S::kRowBytes);
          fence_copies();                                     // after the reads of the slice before
          if (pg >= 0) {
            copy_row(row, side.base + off * 16ull, S::kRowBytes, bar);
          } else {                                            // past the length: zeros
            for (int c = 0; c < S::kChunks; ++c)
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(row + c * 16), "r"(0) : "memory");
          }
        } else {
          constexpr int kCopies = kSlice * S::kChunks / 32;   // of a lane and side
          unsigned ko[kCopies], vo[kCopies];
#pragma unroll
          for (int x = 0; x < kCopies; ++x) {                 // all in flight before the first copy needs one
            const int r = (x * 32 + lane) / S::kChunks;
            ko[x] = __shfl_sync(0xFFFFFFFFu, off, r);
            vo[x] = __shfl_sync(0xFFFFFFFFu, off, r + kSlice);
          }
          if (live == 0xFFFFFFFFu) {
#pragma unroll
            for (int x = 0; x < kCopies; ++x) {
              const int c = x * 32 + lane, r = c / S::kChunks, col = c % S::kChunks;
              cp16(st + r * S::kKStride + col * 16, P.k.base + (ko[x] + col) * 16ull);
              cp16(st + kSlice * S::kKStride + r * S::kVStride + col * 16, P.v.base + (vo[x] + col) * 16ull);
            }
          } else {                                            // past the length: zeros
#pragma unroll
            for (int x = 0; x < kCopies; ++x) {
              const int c = x * 32 + lane, r = c / S::kChunks, col = c % S::kChunks;
              const bool ok = (live >> r) & 1u;
              cp16_or_zero(st + r * S::kKStride + col * 16, P.k.base + (ok ? ko[x] + col : 0u) * 16ull, ok);
              cp16_or_zero(st + kSlice * S::kKStride + r * S::kVStride + col * 16, P.v.base + (ok ? vo[x] + col : 0u) * 16ull, ok);
            }
          }
        }
        if (E4M3) {
          const float* sc = side.scale;
          if (pg >= 0) sc += (static_cast<long long>(pg) * C.heads + h) * C.page_size + slot;
          cp4_or_zero(st + kSlice * (S::kKStride + S::kVStride) + lane * 4, sc, pg >= 0);
        }
      }
      if (E4M3 || !BULK) cp_commit();
    };
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) issue(i);

    // ---- score scales of heads 8 x + 2 t and + 1
    float rs[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      rs[x][0] = rs[x][1] = P.scale;
      if (E4M3) {
        // The products run in f16 (e4m3 codes are exact there).  Each query head is
        // scaled by a power of two to a largest magnitude in [1, 2), so that bf16
        // queries fit its range; the power goes into the head's score scale.
        // Dimensions are dealt so that a lane's 8 consecutive codes of a key feed
        // its operands of two products: k index 2t, 2t+1, 2t+8, 2t+9 of product 2i
        // are dimensions 32 i + 8 t + 0..3, of product 2i + 1 + 4..7.
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          const uint32_t u[4] = {qw[x][k].x, qw[x][k].y, qw[x][k].z, qw[x][k].w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            m = fmaxf(m, fmaxf(fabsf(DType<DT>::to_f32(u[i] & 0xFFFFu)), fabsf(DType<DT>::to_f32(u[i] >> 16))));
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        // 2^-e and 2^e from the exponent field, kept within [2^-100, 2^100]
        const int e = min(max(static_cast<int>(__float_as_uint(m) >> 23) - 127, -100), 100);
        const float down = __uint_as_float((127 - e) << 23), up = P.scale * __uint_as_float((127 + e) << 23);
        rs[x][0] = __shfl_sync(0xFFFFFFFFu, up, 8 * t);
        rs[x][1] = __shfl_sync(0xFFFFFFFFu, up, 8 * t + 4);
        auto half2of = [&](uint32_t v) {
          return pack2<ECAH_DTYPE_F16>(DType<DT>::to_f32(v & 0xFFFFu) * down, DType<DT>::to_f32(v >> 16) * down);
        };
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          qf[x][2 * k][0] = half2of(qw[x][k].x);
          qf[x][2 * k][1] = half2of(qw[x][k].y);
          qf[x][2 * k + 1][0] = half2of(qw[x][k].z);
          qf[x][2 * k + 1][1] = half2of(qw[x][k].w);
        }
      }
    }

    // o: 16 dimensions (rows) by 8 heads; m, l: heads 8 x + 2 t and + 1
    float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[x][i][0] = o[x][i][1] = o[x][i][2] = o[x][i][3] = 0.0f;
      m[x][0] = m[x][1] = -INFINITY;
      l[x][0] = l[x][1] = 0.0f;
    }

    bool stop = false;
    for (int i = 0; i < steps && !stop; ++i) {
      issue(i + S::kStages - 1);
      if (E4M3 || !BULK) cp_wait<S::kStages - 1>();
      if (BULK) {
        if (!bar_wait(bars + 8 * (i % S::kStages), phase >> (i % S::kStages) & 1u, P.tries)) {
          // Give up: wait again for the copies in flight, so that none lands in the
          // results or after the block has ended.
          for (int k = i; k < min(steps, i + S::kStages); ++k)
            bar_wait(bars + 8 * (k % S::kStages), phase >> (k % S::kStages) & 1u, kTries);
          failed = true;
          s_failed = 1;
        }
        phase ^= 1u << (i % S::kStages);
      }
      __syncwarp();
      const int base = (t0 + i) * tile + slice0;
      if (base < len) {
        const uint32_t ks = ring + (i % S::kStages) * S::kStage, vs = ks + kSlice * S::kKStride;
        const unsigned char* ks_p = ring_p + (i % S::kStages) * S::kStage;
        // scores: s[x][0..3] = (key g, head 8x + 2t), (g, + 1), (g + 8, 8x + 2t), (g + 8, + 1)
        float s[NT][4], s2[NT][4];                            // two chains: half the latency
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y) s[x][y] = s2[x][y] = 0.0f;
        if (!E4M3) {
          const uint32_t a0 = ks + ((lane & 7) + ((lane >> 3) & 1) * 8) * S::kKStride + (lane >> 4) * 16;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t a[4];
            ldsm4(a, a0 + k * 32);
#pragma unroll
            for (int x = 0; x < NT; ++x) mma<HT>(k & 1 ? s2[x] : s[x], a, qf[x][k][0], qf[x][k][1]);
          }
        } else {
          const unsigned char* kp = ks_p + g * S::kKStride + 8 * t;
#pragma unroll
          for (int k = 0; k < D / 32; ++k) {
            const uint2 u = *reinterpret_cast<const uint2*>(kp + 32 * k);
            const uint2 w = *reinterpret_cast<const uint2*>(kp + 8 * S::kKStride + 32 * k);
            uint32_t a[4], b[4];
            e4m3x4(u.x, a[0], a[2]);
            e4m3x4(w.x, a[1], a[3]);
            e4m3x4(u.y, b[0], b[2]);
            e4m3x4(w.y, b[1], b[3]);
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              mma<HT>(s[x], a, qf[x][2 * k][0], qf[x][2 * k][1]);
              mma<HT>(s2[x], b, qf[x][2 * k + 1][0], qf[x][2 * k + 1][1]);
            }
          }
        }
        // Scores in log2 units.  An e4m3 value's scale goes into its weight through
        // the exponent, so that the f16 weights stay at or below 2^15 whatever the
        // scales are: weight 2^(s + log2 scale - m), and the sum takes it back out.
        float inv[2] = {1.0f, 1.0f};
        const bool tail = base + kSlice > len;
        const int left = len - base;
        if (E4M3) {
          const float* sc = reinterpret_cast<const float*>(ks_p + kSlice * (S::kKStride + S::kVStride));
          const float kx0 = sc[g], kx1 = sc[g + 8];
          const float v0 = max_nan(sc[kSlice + g], 8e-28f), v1 = max_nan(sc[kSlice + g + 8], 8e-28f);   // 2^-90
          const float lv0 = lg2(v0), lv1 = lg2(v1);
          inv[0] = rcp(v0);
          inv[1] = rcp(v1);
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            s[x][0] = fmaf((s[x][0] + s2[x][0]) * kx0, rs[x][0], lv0);
            s[x][1] = fmaf((s[x][1] + s2[x][1]) * kx0, rs[x][1], lv0);
            s[x][2] = fmaf((s[x][2] + s2[x][2]) * kx1, rs[x][0], lv1);
            s[x][3] = fmaf((s[x][3] + s2[x][3]) * kx1, rs[x][1], lv1);
          }
        } else {
#pragma unroll
          for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int y = 0; y < 4; ++y) s[x][y] = (s[x][y] + s2[x][y]) * P.scale;
        }
        if (tail) {
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            if (g >= left) s[x][0] = s[x][1] = -INFINITY;
            if (g + 8 >= left) s[x][2] = s[x][3] = -INFINITY;
          }
        }
        float top[NT][2];
        bool above = BULK && failed;                          // of one lane: told to all by the vote below
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          top[x][0] = fmaxf(s[x][0], s[x][2]);
          top[x][1] = fmaxf(s[x][1], s[x][3]);
          above |= top[x][0] > m[x][0] + (kLazy + lift) || top[x][1] > m[x][1] + (kLazy + lift);
        }
        if (__any_sync(0xFFFFFFFFu, above)) {
          if (BULK) stop = __any_sync(0xFFFFFFFFu, failed);
#pragma unroll
          for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float v = top[x][y];
#pragma unroll
              for (int z = 4; z < 32; z <<= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, z));
              v = fmaxf(v - lift, m[x][y]);
              const float f = m[x][y] == v ? 1.0f : ex2_approx(m[x][y] - v);
              m[x][y] = v;
              l[x][y] *= f;
#pragma unroll
              for (int k = 0; k < D / 16; ++k) { o[x][k][y] *= f; o[x][k][y + 2] *= f; }
            }
        }
        uint32_t pf[NT][2];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          const float r0 = m[x][0] == -INFINITY ? 0.0f : m[x][0], r1 = m[x][1] == -INFINITY ? 0.0f : m[x][1];
          const float p0 = ex2_approx(s[x][0] - r0), p1 = ex2_approx(s[x][1] - r1);
          const float p2 = ex2_approx(s[x][2] - r0), p3 = ex2_approx(s[x][3] - r1);
          if (E4M3) {
            l[x][0] = fmaf(p0, inv[0], fmaf(p2, inv[1], l[x][0]));
            l[x][1] = fmaf(p1, inv[0], fmaf(p3, inv[1], l[x][1]));
          } else {
            l[x][0] += p0 + p2;
            l[x][1] += p1 + p3;
          }
          // Keys by heads to heads by keys: the products' second operand, in its 16 bits.  A
          // weight is off by at most 2^-9 of itself in bf16 (2^-12 in f16), at random over the
          // keys: in bf16 about 0.8 of the output's own rounding.
          pf[x][0] = transpose8x8(pack2<HT>(p0, p1));
          pf[x][1] = transpose8x8(pack2<HT>(p2, p3));
        }
        if (!E4M3) {
          const uint32_t a0 = vs + ((lane & 7) + (lane >> 4) * 8) * S::kVStride + ((lane >> 3) & 1) * 16;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t a[4];
            ldsm4_t(a, a0 + k * 32);
#pragma unroll
            for (int x = 0; x < NT; ++x) mma<HT>(o[x][k], a, pf[x][0], pf[x][1]);
          }
        } else {
          // 16-bit units of the transposed load hold two dimensions' codes: of two keys'
          // units, bytes 0 and 2 are the even dimension's (row g), 1 and 3 the odd one's
          // (row g + 8)
          const uint32_t a0 = vs + ((lane & 7) + ((lane >> 3) & 1) * 8) * S::kVStride + (lane >> 4) * 16;
#pragma unroll
          for (int k = 0; k < D / 32; ++k) {
            uint32_t b[4], a[4];
            ldsm4_t(b, a0 + k * 32);
            e4m3x4(__byte_perm(b[0], 0u, 0x3120), a[0], a[1]);
            e4m3x4(__byte_perm(b[1], 0u, 0x3120), a[2], a[3]);
#pragma unroll
            for (int x = 0; x < NT; ++x) mma<HT>(o[x][2 * k], a, pf[x][0], pf[x][1]);
            e4m3x4(__byte_perm(b[2], 0u, 0x3120), a[0], a[1]);
            e4m3x4(__byte_perm(b[3], 0u, 0x3120), a[2], a[3]);
#pragma unroll
            for (int x = 0; x < NT; ++x) mma<HT>(o[x][2 * k + 1], a, pf[x][0], pf[x][1]);
          }
        }
      }
      __syncwarp();
    }
    if (E4M3 || !BULK) cp_wait<0>();
    if (BULK) failed = __any_sync(0xFFFFFFFFu, failed);       // also where the last slice had no key
    __syncwarp();

    // ---- join the warps: each leaves (m, l, o) in its ring
    float* ro = reinterpret_cast<float*>(ring_p);
    float2* rml = reinterpret_cast<float2*>(ro + kRows * S::kOStride);
#pragma unroll
    for (int x = 0; x < NT; ++x) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int z = 4; z < 32; z <<= 1) l[x][y] += __shfl_xor_sync(0xFFFFFFFFu, l[x][y], z);
        if (g == 0) rml[8 * x + 2 * t + y] = make_float2(m[x][y], l[x][y]);
      }
      float* r0 = ro + (8 * x + 2 * t) * S::kOStride;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        if (!E4M3) {
          r0[16 * k + g] = o[x][k][0];
          r0[16 * k + g + 8] = o[x][k][2];
          r0[S::kOStride + 16 * k + g] = o[x][k][1];
          r0[S::kOStride + 16 * k + g + 8] = o[x][k][3];
        } else {
          *reinterpret_cast<float2*>(r0 + 16 * k + 2 * g) = make_float2(o[x][k][0], o[x][k][2]);
          *reinterpret_cast<float2*>(r0 + S::kOStride + 16 * k + 2 * g) = make_float2(o[x][k][1], o[x][k][3]);
        }
      }
    }
    __syncthreads();

    // parts of this item: the blocks whose shares overlap its tiles
    int a = blockIdx.x, parts = 1;
    if (nt > whole) {
      auto block_of = [&](unsigned x) { return x < more * (share + 1) ? x / (share + 1) : more + (x - more * (share + 1)) / share; };
      a = block_of(tile0);
      parts = block_of(tile0 + nt - 1) - a + 1;
    }
    const int part = blockIdx.x - a;
    auto slot_of = [&](int p) { return p == 0 ? 2 * a + 1 : 2 * (a + p); };

    // Combine `count` triples (m, l, o) of each of the item's rows (head h0 + j, query
    // head r of its tile; row j kRows + r) into the output or a part's slot.
    const int item_rows = wh * kRows;
    const bool bad = BULK && s_failed;
    auto combine = [&](auto from, int count, auto ml_of, auto o_of, int o_stride, int to) {
      using From = decltype(from);
      for (int i = tid; i < count * item_rows; i += kT) {
        const int p = i / item_rows, r = i % item_rows;
        s_ml[p][r] = From::two(ml_of(p, r / kRows) + r);
      }
      __syncthreads();
      if (tid < item_rows && tid % kRows < rows) {
        float mm = -INFINITY, ll = 0.0f;
        for (int p = 0; p < count; ++p) mm = fmaxf(mm, s_ml[p][tid].x);
        for (int p = 0; p < count; ++p) {
          const float2 v = s_ml[p][tid];
          const float f = v.x == -INFINITY ? 0.0f : ex2_approx(v.x - mm);
          ll = fmaf(v.y, f, ll);
          s_ml[p][tid].x = f;
        }
        if (bad) ll = NAN;
        if (to >= 0) {
          P.part_ml[static_cast<long long>(to) * item_rows + tid] = make_float2(mm, ll);
        } else {
          // a sum of zero (no key has mass) gives zeros
          const float r = ll == 0.0f ? 0.0f : 1.0f / ll;
          for (int p = 0; p < count; ++p) s_ml[p][tid].x *= r;
          if (P.lse)
            P.lse[static_cast<long long>(req) * P.hq + (h0 + tid / kRows) * P.group + ht * kRows + tid % kRows] =
                ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * kLn2;
        }
      }
      __syncthreads();
      for (int e = tid * 4; e < item_rows * D; e += kT * 4) {
        const int r = e / D, d = e % D, j = r / kRows;
        if (r % kRows >= rows) continue;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int p = 0; p < count; ++p) {
          const float4 w = From::four(o_of(p, j) + r * o_stride + d);
          const float f = s_ml[p][r].x;
          v.x = fmaf(w.x, f, v.x); v.y = fmaf(w.y, f, v.y); v.z = fmaf(w.z, f, v.z); v.w = fmaf(w.w, f, v.w);
        }
        if (bad) v = make_float4(NAN, NAN, NAN, NAN);
        if (to >= 0) {
          *reinterpret_cast<float4*>(P.part_o + static_cast<long long>(to) * item_rows * D + e) = v;
        } else {
          const uint2 w = make_uint2(pack2<DT>(v.x, v.y), pack2<DT>(v.z, v.w));
          const int head = (h0 + j) * P.group + ht * kRows + r % kRows;
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(P.out) + req * P.o_tok + head * P.o_head + d) = w;
        }
      }
    };
    // the warps of head j: j, j + wh, ...; their rows start at theirs
    auto warp_o = [&](int p, int j) -> const float* {
      return reinterpret_cast<const float*>(smem + (p * wh + j) * S::kWarpBytes) - j * kRows * S::kOStride;
    };
    auto warp_ml = [&](int p, int j) -> const float2* {
      return reinterpret_cast<const float2*>(smem + (p * wh + j) * S::kWarpBytes + kRows * S::kOStride * 4) - j * kRows;
    };
    combine(FromShared(), kW / wh, warp_ml, warp_o, S::kOStride, parts == 1 ? -1 : slot_of(part));

    if (parts > 1) {
      // joined in one step, or in groups of about sqrt(parts) first
      int gs = parts;
      if (parts > kMaxGroup) { gs = 1; while (gs * gs < parts) ++gs; }
      const int groups = (parts + gs - 1) / gs, grp = part / gs, p0 = grp * gs, in_grp = min(gs, parts - p0);
      auto ml_at = [&](int slot) { return P.part_ml + static_cast<long long>(slot) * item_rows; };
      auto o_at = [&](int slot) { return P.part_o + static_cast<long long>(slot) * item_rows * D; };
      if (arrive(P.counters + 2 * slot_of(p0), in_grp, &s_flag)) {
        combine(FromParts(), in_grp, [&](int p, int) { return ml_at(slot_of(p0 + p)); },
                [&](int p, int) { return o_at(slot_of(p0 + p)); }, D, groups == 1 ? -1 : slot_of(p0));
        if (groups > 1 && arrive(P.counters + 2 * slot_of(0) + 1, groups, &s_flag))
          combine(FromParts(), groups, [&](int p, int) { return ml_at(slot_of(p * gs)); },
                  [&](int p, int) { return o_at(slot_of(p * gs)); }, D, -1);
      }
    }
    if (BULK) fence_copies();
    __syncthreads();       // the rings are free again
  }

  // requests without tokens: zeros, spread over the blocks
  for (int b = blockIdx.x; b < C.batch; b += gridDim.x) {
    int f;
    if (look(b, &f) != 0) continue;
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

// The kernel of a head layout: one head tile of 8 query heads where a KV head has
// at most 8, else tiles of 16 (a KV row is then read once per 16 heads).
//
// BULK: rows by the copy engine, for 16-bit heads of 128 and 192 where there is much
// to stream.  It starts a copy about every 10 clocks an SM, at 256 bytes more than HBM
// brings, and leaves the threads free.  4 requests of 100 001 to 131 072 tokens, 32/8
// heads: 302 us against 321 with heads of 128, 454 against 495 with 192.  Elsewhere
// the threads' copies are better: shorter rows starve (128 bytes: 3.4 TB/s), rows of 256
// in 8 bits with their conversions take 430 us against 339, heads of 256 leave room for
// one block (711 against 638), and a block with little to do waits longer for its 128
// copies (128 requests of up to 512 tokens: 18.6 us against 13.7).  The rule goes by the
// pages listed, which is all that the host knows: a list with room for much more than the
// requests hold, as a captured step keeps one, takes the copy engine for short requests too.
template <int DT, bool E4M3, int D, int NT>
static Variant variant_of(bool bulk) {
  constexpr bool kCan = !E4M3 && (D == 128 || D == 192);
  using Bulk = Shape<D, E4M3, NT, kCan>;
  using Threads = Shape<D, E4M3, NT, false>;
  if (kCan && bulk) return Variant{decode_kernel<DT, E4M3, D, NT, kCan>, Bulk::kSmem, Bulk::kBlocks};
  return Variant{decode_kernel<DT, E4M3, D, NT, false>, Threads::kSmem, Threads::kBlocks};
}

template <int DT, bool E4M3, int NT>
static Variant variant_for(int D, bool bulk) {
  switch (D) {
    case 64: return variant_of<DT, E4M3, 64, NT>(bulk);
    case 96: return variant_of<DT, E4M3, 96, NT>(bulk);
    case 128: return variant_of<DT, E4M3, 128, NT>(bulk);
    case 192: return variant_of<DT, E4M3, 192, NT>(bulk);
    default: return variant_of<DT, E4M3, 256, NT>(bulk);
  }
}

template <int DT, bool E4M3>
static Variant variant_for(int D, int group, bool bulk) {
  return group <= 8 ? variant_for<DT, E4M3, 1>(D, bulk) : variant_for<DT, E4M3, 2>(D, bulk);
}

constexpr int kMaxBlocksPerSm = 4;

// Workspace: counters, then the parts' (m, l), then their sums.  A block has at
// most two parts of items it shares with others, whatever the batch is.
struct Layout {
  size_t ml, o, total;
};

static Layout layout(int sms, int D) {
  const size_t slots = 2 * static_cast<size_t>(sms) * kMaxBlocksPerSm + 2;
  Layout L;
  L.ml = (slots * 2 * sizeof(unsigned) + 255) / 256 * 256;
  L.o = L.ml + slots * kMaxRows * sizeof(float2);
  L.total = L.o + slots * kMaxRows * D * sizeof(float);
  return L;
}

// A side of the cache in 16-byte units; false where a row lies past 2^32 of them
// (64 GB from the base).
static bool side16(const kv::Side& s, int pages, int page_size, int heads, int elem, Side16* r) {
  const long long unit = 16 / elem;
  const long long most = (std::max(pages, 1) - 1ll) * (s.page / unit) + (page_size - 1ll) * (s.slot / unit) + (heads - 1ll) * (s.head / unit);
  if (s.page / unit > 0xFFFFFFFFll || s.slot / unit > 0xFFFFFFFFll || s.head / unit > 0xFFFFFFFFll || most + 64 > 0xFFFFFFFFll) return false;
  *r = Side16{static_cast<const unsigned char*>(s.base), static_cast<unsigned>(s.page / unit), static_cast<unsigned>(s.slot / unit),
              static_cast<unsigned>(s.head / unit), s.scale};
  return true;
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

int ecah_paged_decode(const ecah_decode_args* a, void* stream) { return ecah_paged_decode_bounded(a, decode::kTries, stream); }

int ecah_paged_decode_bounded(const ecah_decode_args* a, int32_t tries, void* stream) {
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
  if (!aligned16(a->q) || !aligned16(a->out)) return ECAH_ERR_SHAPE;
  if (!a->workspace || !aligned16(a->workspace) ||
      a->workspace_bytes < ecah_paged_decode_workspace_bytes(c.batch, a->num_qo_heads, c.num_kv_heads, c.head_dim))
    return ECAH_ERR_WORKSPACE;
  const int sms = device_sms();
  if (sms <= 0) return ECAH_ERR_LAUNCH;
  decode::Params P = {};
  P.q = a->q; P.out = a->out; P.lse = a->lse; P.last_page_len = a->kv_last_page_len;
  P.q_tok = a->q_token_stride; P.q_head = a->q_head_stride;
  P.o_tok = a->out_token_stride; P.o_head = a->out_head_stride;
  P.hq = a->num_qo_heads; P.group = a->num_qo_heads / c.num_kv_heads;
  const int rows = P.group <= 8 ? 8 : 16;
  P.tiles_h = (P.group + rows - 1) / rows;
  P.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (c.page_size == 1 << i) P.page_shift = i;
  P.tries = tries;
  P.scale = a->sm_scale * kLog2e;
  P.cache = kv::make_cache(c);
  const decode::Layout L = decode::layout(sms, c.head_dim);
  unsigned char* ws = static_cast<unsigned char*>(a->workspace);
  P.counters = reinterpret_cast<unsigned*>(ws);
  P.part_ml = reinterpret_cast<float2*>(ws + L.ml);
  P.part_o = reinterpret_cast<float*>(ws + L.o);
  const bool e4m3 = c.kv_dtype == ECAH_KV_E4M3, f16 = a->dtype == ECAH_DTYPE_F16;
  if (!decode::side16(P.cache.k, c.num_pages, c.page_size, c.num_kv_heads, e4m3 ? 1 : 2, &P.k) ||
      !decode::side16(P.cache.v, c.num_pages, c.page_size, c.num_kv_heads, e4m3 ? 1 : 2, &P.v))
    return ECAH_ERR_SHAPE;
  // Units that the listed pages can hold with one KV head an item; `much`: 64 of them to
  // an SM, where streaming outweighs starting and joining.
  const double units = static_cast<double>(c.num_indices) * c.page_size / decode::kTile * c.num_kv_heads * P.tiles_h;
  const bool much = units > 64.0 * sms;
  const decode::Variant v =
      f16 ? (e4m3 ? decode::variant_for<ECAH_DTYPE_F16, true>(c.head_dim, P.group, much)
                  : decode::variant_for<ECAH_DTYPE_F16, false>(c.head_dim, P.group, much))
          : (e4m3 ? decode::variant_for<ECAH_DTYPE_BF16, true>(c.head_dim, P.group, much)
                  : decode::variant_for<ECAH_DTYPE_BF16, false>(c.head_dim, P.group, much));
  P.wh = 1;
  // Runs of 256 bytes of a token where there is much to stream (the long requests over
  // an e4m3 cache of 128-byte rows: 172 us with two heads a block, 197 with one, 186
  // with four).
  const int row_bytes = c.head_dim * (e4m3 ? 1 : 2);
  if (much)
    while (P.wh < 4 && P.wh * row_bytes < 256 && P.wh * 2 * rows <= decode::kMaxRows && c.num_kv_heads % (P.wh * 2) == 0) P.wh *= 2;
  const double items = static_cast<double>(c.batch) * (c.num_kv_heads / P.wh) * P.tiles_h;
  const double most = units + items * (1.0 + decode::kItemCost) + 1;
  if (most >= 2147483648.0 || c.num_indices > 0x7FFFFFFF) return ECAH_ERR_SHAPE;   // units are counted in 32 bits
  // no more blocks than units (and one for the empty requests)
  const double grid = std::min(sms * v.blocks, decode::kMaxGroup * decode::kMaxGroup);
  const int blocks = static_cast<int>(std::min(most, grid));
  return launch_kernel(v.fn, dim3(blocks), decode::kT, v.smem, reinterpret_cast<cudaStream_t>(stream), P) ? ECAH_OK : ECAH_ERR_LAUNCH;
}

}  // extern "C"
