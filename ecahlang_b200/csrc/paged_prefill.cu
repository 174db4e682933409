// Attention of several new tokens per request over the paged key-value cache:
// ecah_paged_prefill (contract in include/ecah_sampler.h).

#include <cuda.h>

#include <algorithm>
#include <cstring>

#include "host_util.h"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace ecah {
namespace prefill {

// The mathematics: as in decode attention, softmax over a row's keys as one pass with
// a running reference m, o = sum_j 2^(s_j - m) v_j and l = sum_j 2^(s_j - m), s in
// units of log2, joined over disjoint runs of keys by their references.
//
// Bound: the tensor cores (4 D flops a visible key and query head) for prompts, HBM
// for few tokens over long contexts.  Both products run on tcgen05: S = Q K^T with
// both operands in shared memory, O += P V with P in tensor memory over S's columns.
//
// Rows: the G query heads of a KV head and the tokens of a request are packed into one
// axis, row = token G + head, so that any G fills the 128 rows of a product and a cached
// byte is used by as many rows as there are.  An item is (request, KV head, tile of
// rows); its keys come in tiles of kKeys.
//
// Two products' rows are in flight ("slots"), so that one slot's softmax runs beside the
// other's products: slots are the two halves of a tile of 256 rows over the same keys;
// or, where an item has at most 128 rows, alternating key tiles of the same rows, each
// slot with a sum of its own; heads of 192 and 256 leave tensor memory for one sum, and
// alternating key tiles share it.
//
// Warps: 4 of softmax to a slot (a thread to a row: no shuffles; it also rescales its
// row of O, which the lazily moved reference makes rare, and writes it out), 4 that
// bring keys and values (pages are lists of rows anywhere, so by threads' 16-byte
// copies into the swizzled tiles; e4m3 codes are converted on the way), 1 that
// issues the products.
//
// Split: one block to an SM; all iterations of all items, in order, are divided evenly
// over the blocks by the lengths the device holds (a captured launch serves any
// lengths).  An item that spans several blocks is joined by the block that arrives
// last, in the order of the parts, so results do not depend on which that is.

constexpr int kT = 512;
constexpr int kLoaders = 8;            // first warp of those that bring keys and values
constexpr int kIssuer = 12;            // the warp that issues the products
constexpr int kItemCost = 3;           // iterations that starting and finishing an item takes
constexpr int kWhole = 6;              // items of up to so many iterations are not divided
constexpr int kLeast = 4;              // iterations to a block at the least
constexpr int kKeep = 128;             // requests looked at together
constexpr int kTries = 1 << 20;        // of a wait: more than one between warps of a block can need
constexpr float kLazy = 8.0f;          // as in decode attention: a reference moves when a score passes it by 2^kLazy;
constexpr float kLift = 7.0f;          // f16 weights reach 2^15, so that small ones are not lost
constexpr float kLn2 = 0.6931471805599453f;

struct alignas(64) Params {
  CUtensorMap k_map, v_map;            // [pages][heads][slots][head_dim], boxes of 64 elements by the slots of a page in a tile
  int boxes;                           // whether the copy engine brings whole tiles
  const void* q;
  void* out;
  float* lse;
  const int *qo_indptr, *last_page_len;
  long long q_tok, q_head, o_tok, o_head;
  int tokens, hq, group, causal;
  int page_shift, tries;
  float scale;                         // sm_scale * log2 e
  unsigned* counters;                  // [blocks] arrivals, zero between launches
  float2* part_ml;                     // [2 blocks][256]
  float* part_o;                       // [2 blocks][256][D] (rows of 128 with one slot)
  kv::Side16 k, v;
  kv::Cache cache;
};

template <int D, bool E4M3>
struct Shape {
  static constexpr int kSlots = D <= 128 ? 2 : 1;
  static constexpr int kRows = 128 * kSlots;               // of an item
  static constexpr int kKeys = D <= 128 ? 128 : 64;        // of a tile
  static constexpr int kBlocks = (D + 63) / 64;            // of 64 elements
  static constexpr int kQ = 128 * kBlocks * 128;           // bytes of a slot's queries
  static constexpr int kTile = kKeys * kBlocks * 128;      // bytes of a tile
  static constexpr int kScales = E4M3 ? kKeys * 12 : 0;    // of a tile: key scale, log2 and reciprocal of the value scale
  static constexpr int kRoom = 227 * 1024 - 1024 - 512;    // alignment, barriers
  static constexpr int ring(int n) { return kSlots * kQ + n * kTile + (n / 2 + 2) * kScales <= kRoom ? n : ring(n - 1); }
  static constexpr int kRing = ring(8);
  static constexpr int kScaleRing = kRing / 2 + 2;
  static constexpr int kSmem = kSlots * kQ + kRing * kTile + kScaleRing * kScales + 1024;
  static constexpr int kBuffer = kKeys;                    // tensor-memory columns of one of the two score buffers
  static constexpr int kSum = 2 * kKeys;                   // first column of the sums
  static constexpr int kColumns = 512;
  static_assert(kRing >= 4 && kSum + kSlots * D <= kColumns, "");
};

// Device-wide facts of a request.
struct Request {
  int q0, n, off, len, first;          // first token, tokens; keys before the first token; keys; first entry of the page list
};

template <int KEYS>
__device__ __forceinline__ Request request(const Params& P, int b) {
  Request r;
  r.q0 = min(max(P.qo_indptr[b], 0), P.tokens);
  r.n = min(max(P.qo_indptr[b + 1], r.q0), P.tokens) - r.q0;
  long long at, count, len = 0;
  kv::page_range(P.cache, b, &at, &count);
  if (count > 0 && P.cache.num_pages > 0)
    len = (count - 1) * P.cache.page_size + min(max(P.last_page_len[b], 0), P.cache.page_size);
  r.len = static_cast<int>(min(len, 0x7FFFFFFFll - 2 * KEYS));
  r.off = r.len - r.n;
  r.first = static_cast<int>(at);
  return r;
}

// Keys that token i of a request sees.
__device__ __forceinline__ int sees(const Params& P, const Request& r, int i) {
  return P.causal ? min(max(r.off + i + 1, 0), r.len) : r.len;
}

template <int D, bool E4M3>
struct Tile {                          // a tile of rows of a request
  int row0, rows, keys, tiles, iters;  // tiles: of keys, for its last row
  bool few;
  __device__ __forceinline__ Tile(const Params& P, const Request& r, int t) {
    using S = Shape<D, E4M3>;
    row0 = t * S::kRows;
    rows = min(r.n * P.group - row0, S::kRows);
    keys = sees(P, r, (row0 + rows - 1) / P.group);
    tiles = (keys + S::kKeys - 1) / S::kKeys;
    few = S::kSlots == 2 && rows <= 128;
    iters = few ? (tiles + 1) / 2 : tiles;
  }
};

template <int D, bool E4M3>
__device__ __forceinline__ int tiles_of(const Params& P, const Request& r) {
  return (r.n * P.group + Shape<D, E4M3>::kRows - 1) / Shape<D, E4M3>::kRows;
}

struct Edge { int req, head, tile; long long start; int iters; };

// The items of this block's share, in order.  Every warp that works on them walks them
// alike, with its own walk in shared memory: only what a loop uses is held in registers.
template <int D, bool E4M3>
struct Walk {
  using S = Shape<D, E4M3>;
  long long lo, hi, at, share, more;
  Request r;
  int req, head, tile, tiles, iters;
  // the present item's part
  int row0, rows, keys, jb, je, je0;   // key tiles [jb, je); of the first slot of two halves [jb, je0)
  int first_block, parts;
  bool fresh, few, whole;

  __device__ __forceinline__ void begin(const Params& P, const Edge& edge, const long long* bounds) {
    if ((threadIdx.x & 31) == 0) {
      lo = bounds[0]; hi = bounds[1]; share = bounds[2]; more = bounds[3];
      req = edge.req; head = edge.head; tile = edge.tile; at = edge.start;
      fresh = true;
      if (req < P.cache.batch) {
        r = request<S::kKeys>(P, req);
        tiles = tiles_of<D, E4M3>(P, r);
      }
    }
    __syncwarp();
  }
  // The next item with work for this block; false behind the last.  Called by whole warps.
  __device__ __forceinline__ bool next(const Params& P) {
    __syncwarp();
    bool found = false;
    if ((threadIdx.x & 31) == 0) found = advance(P);
    return __shfl_sync(0xFFFFFFFFu, found, 0);               // and orders what lane 0 wrote
  }

 private:
  __device__ __forceinline__ int block_of(long long x) const {
    return static_cast<int>(x < more * (share + 1) ? x / (share + 1) : more + (x - more * (share + 1)) / share);
  }
  __device__ __forceinline__ bool advance(const Params& P) {
    while (true) {
      if (!fresh) {
        at += iters + kItemCost;
        if (++tile >= tiles) {
          tile = 0;
          if (++head >= P.cache.heads) {
            head = 0;
            do {
              if (++req >= P.cache.batch) return false;
              r = request<S::kKeys>(P, req);
              tiles = tiles_of<D, E4M3>(P, r);
            } while (tiles == 0);
          }
        }
      }
      fresh = false;
      if (req >= P.cache.batch || at >= hi) {
        fresh = true;                                         // stays behind the last
        return false;
      }
      const Tile<D, E4M3> t(P, r, tile);
      iters = t.iters;
      const long long begin = at + kItemCost;
      int i0 = 0, i1 = t.iters;
      whole = t.iters <= kWhole;
      first_block = blockIdx.x;
      parts = 1;
      if (whole) {
        if (at < lo) continue;
      } else {
        i0 = static_cast<int>(min(max(lo - begin, 0ll), static_cast<long long>(t.iters)));
        i1 = static_cast<int>(min(max(hi - begin, 0ll), static_cast<long long>(t.iters)));
        if (i0 >= i1) continue;
        first_block = block_of(begin);
        parts = block_of(begin + t.iters - 1) - first_block + 1;
        whole = parts == 1;
      }
      row0 = t.row0; rows = t.rows; keys = t.keys; few = t.few;
      jb = few ? 2 * i0 : i0;
      je = few ? min(2 * i1, t.tiles) : i1;
      je0 = je;
      if (S::kSlots == 2 && !few)      // the first half's last row sees fewer keys
        je0 = max(jb, min(je, (sees(P, r, (row0 + 127) / P.group) + S::kKeys - 1) / S::kKeys));
      return true;
    }
  }
};

template <int HT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (HT == ECAH_DTYPE_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void st16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void e4m3x4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }"
      : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
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
__device__ __forceinline__ void sync_some(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// The block's barriers.
template <int D, bool E4M3>
struct Bars {
  unsigned long long q_full, q_empty, done;
  unsigned long long kv_full[Shape<D, E4M3>::kRing], kv_empty[Shape<D, E4M3>::kRing];
  unsigned long long s_full[2], p_full[2], pv_done[2];
};

template <int DT, bool E4M3, int D>
__global__ void __launch_bounds__(kT, 1) prefill_kernel(const __grid_constant__ Params P) {
  using S = Shape<D, E4M3>;
  constexpr int HT = E4M3 ? static_cast<int>(ECAH_DTYPE_F16) : DT;   // operand type of the products
  constexpr float lift = HT == ECAH_DTYPE_F16 ? kLift : 0.0f;
  constexpr int kKeys = S::kKeys, kRing = S::kRing, kSlots = S::kSlots;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Bars<D, E4M3> s_bars;
  __shared__ Edge s_edge[2];
  __shared__ long long s_bounds[4];
  __shared__ uint32_t s_tmem;
  __shared__ int s_failed, s_flag;
  __shared__ Walk<D, E4M3> s_walk[kIssuer + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* base_p = smem_raw + (base - tc::smem_u32(smem_raw));
  const uint32_t s_q = base, s_ring = base + kSlots * S::kQ, s_scales = s_ring + kRing * S::kTile;
  const kv::Cache& C = P.cache;

  grid_start();

  // ---- barriers, tensor memory
  if (tid == 0) {
    auto init = [&](unsigned long long* b, int n) { tc::bar_init(tc::smem_u32(b), n); };
    init(&s_bars.q_full, E4M3 ? 4 * kSlots : 4);
    init(&s_bars.q_empty, 1);
    init(&s_bars.done, 1);
    for (int i = 0; i < kRing; ++i) { init(&s_bars.kv_full[i], 4); init(&s_bars.kv_empty[i], 1); }
    for (int i = 0; i < 2; ++i) { init(&s_bars.s_full[i], 1); init(&s_bars.p_full[i], 4); init(&s_bars.pv_done[i], 1); }
    tc::fence_smem();
    s_failed = 0;
    s_edge[0].req = s_edge[1].req = C.batch;
    s_edge[0].start = s_edge[1].start = 0;
  }
  if (warp == kIssuer) tc::tmem_alloc(tc::smem_u32(&s_tmem), S::kColumns);

  // ---- this block's share.  An item costs kItemCost units, then one an iteration; the
  // first `more` blocks take share + 1 units, the others share.
  {
    Request* s_req = reinterpret_cast<Request*>(base_p + kSlots * S::kQ);            // the ring is not in use yet
    long long* s_cost = reinterpret_cast<long long*>(base_p + kSlots * S::kQ + kKeep * 32);
    auto look = [&](int b0) {          // cost of a head of each of kKeep requests
      __syncthreads();
      if (tid < kKeep) {
        if (b0 + tid < C.batch) s_req[tid] = request<kKeys>(P, b0 + tid);
        else s_req[tid].n = 0;
      }
      __syncthreads();
      for (int i = warp; i < kKeep; i += kT / 32) {
        const Request r = s_req[i];
        long long sum = 0;
        for (int t = lane; t < tiles_of<D, E4M3>(P, r); t += 32) sum += Tile<D, E4M3>(P, r, t).iters + kItemCost;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (lane == 0) s_cost[i] = sum;
      }
      __syncthreads();
    };
    auto chunk_sum = [&]() {
      long long sum = 0;
      for (int i = lane; i < kKeep; i += 32) sum += s_cost[i];
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
      return sum * C.heads;
    };
    long long total = 0;
    for (int b0 = 0; b0 < C.batch; b0 += kKeep) {
      look(b0);
      total += chunk_sum();
    }
    const long long blocks = min(static_cast<long long>(gridDim.x), max(1ll, total / kLeast));
    const bool busy = blockIdx.x < blocks && total > 0;
    const long long share = max(1ll, total / blocks), more = total - share * blocks;
    long long edge[2] = {0, 0};
    if (busy) {
      edge[0] = blockIdx.x * share + min(static_cast<long long>(blockIdx.x), more);
      edge[1] = edge[0] + share + (blockIdx.x < more);
    }
    long long run = 0;
    for (int b0 = 0; busy && b0 < C.batch; b0 += kKeep) {
      if (C.batch > kKeep) look(b0);
      const long long sum = chunk_sum();
      if (warp < 2) {
        const long long x = edge[warp];
        if (x >= run && x < run + sum) {
          long long p = run;
          int i = 0;                                          // the request
          for (int i0 = 0;; i0 += 32) {
            const long long c = s_cost[i0 + lane] * C.heads;
            long long inc = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const long long v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
              if (lane >= o) inc += v;
            }
            const unsigned past = __ballot_sync(0xFFFFFFFFu, p + inc > x);
            if (past) {
              const int l = __ffs(past) - 1;
              p += __shfl_sync(0xFFFFFFFFu, inc - c, l);
              i = i0 + l;
              break;
            }
            p += __shfl_sync(0xFFFFFFFFu, inc, 31);
          }
          const long long one = s_cost[i];
          const int head = static_cast<int>((x - p) / one);
          p += head * one;
          const Request r = s_req[i];
          const int tiles = tiles_of<D, E4M3>(P, r);
          for (int t0 = 0;; t0 += 32) {                       // the tile
            int iters = 0;
            long long c = 0;
            if (t0 + lane < tiles) { iters = Tile<D, E4M3>(P, r, t0 + lane).iters; c = iters + kItemCost; }
            long long inc = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const long long v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
              if (lane >= o) inc += v;
            }
            const unsigned past = __ballot_sync(0xFFFFFFFFu, p + inc > x);
            if (past) {
              const int l = __ffs(past) - 1;
              p += __shfl_sync(0xFFFFFFFFu, inc - c, l);
              iters = __shfl_sync(0xFFFFFFFFu, iters, l);
              if (lane == 0) s_edge[warp] = Edge{b0 + i, head, t0 + l, p, iters};
              break;
            }
            p += __shfl_sync(0xFFFFFFFFu, inc, 31);
          }
        }
      }
      run += sum;
      if (edge[1] < run) break;
    }
    __syncthreads();
    if (tid == 0) {
      // an edge inside an item that is not divided moves to the item's nearer end
      for (int e = 0; e < 2; ++e) {
        const Edge& g = s_edge[e];
        if (busy && g.req < C.batch && g.iters <= kWhole) {
          const long long cost = g.iters + kItemCost, into = edge[e] - g.start;
          edge[e] = g.start + (2 * into < cost ? 0 : cost);
        }
        s_bounds[e] = edge[e];
      }
      s_bounds[2] = share;
      s_bounds[3] = more;
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
  }
  const uint32_t tmem = s_tmem;

  // Waits for a phase of a barrier; false when it ran out, here or in another warp: the
  // block then ends as fast as it can, and its results are NaN.
  auto wait = [&](unsigned long long* b, uint32_t parity) -> bool {
    const uint32_t bar = tc::smem_u32(b);
    bool ok = false;
    for (int i = 0; i < P.tries && !ok; ++i) {
      ok = tc::bar_test(bar, parity);
      if (!ok && *static_cast<volatile int*>(&s_failed)) break;
    }
    ok = __all_sync(0xFFFFFFFFu, ok);
    if (!ok) *static_cast<volatile int*>(&s_failed) = 1;
    return ok;
  };

  Walk<D, E4M3>& w = s_walk[min(warp, kIssuer)];
  if (warp <= kIssuer) w.begin(P, s_edge[0], s_bounds);

  if (warp < 4 * kSlots) {
    // =============================================================== softmax
    const int slot = warp >> 2, row = tid & 127;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);
    const uint32_t sum_at = lanes + S::kSum + slot * D;
    uint32_t s_phase = 0, q_phase = 0;                        // a bit a buffer
    int before = 0;                                           // key tiles of the items before
    unsigned pv = 0;                                          // products O += P V of this slot so far
    bool ok = true;
    // The last product so far.  A slot's scores come after its product before, so at most
    // one is outstanding on a barrier; with one slot two are, on barriers in turn.
    auto wait_sum = [&]() {
      const unsigned x = pv - 1;
      const bool there = kSlots == 2 ? wait(&s_bars.pv_done[slot], x & 1) : wait(&s_bars.pv_done[x & 1], x >> 1 & 1);
      tc::fence_after();
      return there;
    };
    while (w.next(P)) {
      const bool own_rows = kSlots == 2 && !w.few;            // slots are halves of the rows
      const int my = (own_rows ? slot * 128 : 0) + row;       // row of the item
      const bool live = my < w.rows;
      const int packed = w.row0 + my;
      const int token = live ? packed / P.group : 0, head = w.head * P.group + packed - token * P.group;
      const int lim = live ? sees(P, w.r, token) : w.keys;   // other rows' scores are zeros, and not used
      const int least = __reduce_min_sync(0xFFFFFFFFu, lim);
      float scale = P.scale;

      if (E4M3 && w.jb < w.je && ok) {
        // This thread's row of queries, scaled by a power of two to a largest magnitude in
        // [1, 2) so that bf16 queries fit f16's range; the power goes into the score scale.
        if (ok) ok = wait(&s_bars.q_empty, q_phase ^ 1);
        q_phase ^= 1;
        if (ok) {
          const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(P.q) + (w.r.q0 + token) * P.q_tok + head * P.q_head);
          float big = 0.0f;
          if (live) {
#pragma unroll 8
            for (int c = 0; c < D / 8; ++c) {
              const uint4 v = src[c];
              const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int i = 0; i < 4; ++i)
                big = fmaxf(big, fmaxf(fabsf(DType<DT>::to_f32(u[i] & 0xFFFFu)), fabsf(DType<DT>::to_f32(u[i] >> 16))));
            }
          }
          const int e = min(max(static_cast<int>(__float_as_uint(big) >> 23) - 127, -100), 100);
          const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
          scale = P.scale * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
          if (own_rows || slot == 0) {
            const uint32_t dst = s_q + (own_rows ? slot : 0) * S::kQ + row * 128;
#pragma unroll 8
            for (int c = 0; c < D / 8; ++c) {
              const uint4 v = live ? src[c] : make_uint4(0, 0, 0, 0);
              const uint32_t u[4] = {v.x, v.y, v.z, v.w};
              uint32_t h[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) h[i] = pack2<HT>(DType<DT>::to_f32(u[i] & 0xFFFFu) * down, DType<DT>::to_f32(u[i] >> 16) * down);
              st16(dst + (c / 8) * (128 * 128) + ((c % 8) ^ (row & 7)) * 16, h[0], h[1], h[2], h[3]);
            }
          }
          tc::fence_smem();
          __syncwarp();
          if (lane == 0) tc::bar_arrive(tc::smem_u32(&s_bars.q_full));
        }
      }

      float m = -INFINITY, l = 0.0f;
      bool any = false;                                       // the sum holds something
      const int step = own_rows || kSlots == 1 ? 1 : 2, jb = w.jb, je = own_rows && slot == 0 ? w.je0 : w.je;
      int buf = kSlots == 2 ? slot : 0;
      for (int j = jb + (own_rows || kSlots == 1 ? 0 : slot); j < je && ok; j += step) {
        ok = wait(&s_bars.s_full[buf], s_phase >> buf & 1);
        if (!ok) break;
        s_phase ^= 1u << buf;
        tc::fence_after();
        const uint32_t s_at = lanes + buf * S::kBuffer;
        // Scores in log2 units; an e4m3 value's scale goes into its weight through the
        // exponent (weight 2^(s + log2 scale - m)), and the sum takes it back out.  They are
        // read twice, 32 at a time: a row's 128 do not fit beside the rest in the registers.
        const float* sc = reinterpret_cast<const float*>(base_p + (s_scales - base) + ((before + j - jb) % S::kScaleRing) * S::kScales);
        const bool masked = (j + 1) * kKeys > least;
        const int left = lim - j * kKeys;
        auto ready = [&](uint32_t (&r)[32], int i) {
          if (E4M3) {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const float4 kx = *reinterpret_cast<const float4*>(sc + 32 * i + c), lv = *reinterpret_cast<const float4*>(sc + kKeys + 32 * i + c);
              const float x[4] = {kx.x, kx.y, kx.z, kx.w}, y[4] = {lv.x, lv.y, lv.z, lv.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) r[c + e] = __float_as_uint(fmaf(__uint_as_float(r[c + e]) * x[e], scale, y[e]));
            }
          }
          if (masked) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (32 * i + c >= left) r[c] = 0xFF800000u;
          }
        };
        uint32_t ra[32], rb[32];
        float t0 = -INFINITY, t1 = -INFINITY, t2 = -INFINITY, t3 = -INFINITY;
#pragma unroll
        for (int i = 0; i < kKeys / 32; i += 2) {
          tc::load32(ra, s_at + 32 * i);
          tc::load32(rb, s_at + 32 * i + 32);
          tc::load_wait();
          tc::pin32(ra);
          tc::pin32(rb);
          ready(ra, i);
          ready(rb, i + 1);
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            t0 = max3(t0, __uint_as_float(ra[c]), __uint_as_float(rb[c]));
            t1 = max3(t1, __uint_as_float(ra[c + 1]), __uint_as_float(rb[c + 1]));
            t2 = max3(t2, __uint_as_float(ra[c + 2]), __uint_as_float(rb[c + 2]));
            t3 = max3(t3, __uint_as_float(ra[c + 3]), __uint_as_float(rb[c + 3]));
          }
        }
        float top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
        if (!E4M3) top *= P.scale;
        if (__any_sync(0xFFFFFFFFu, top > m + (kLazy + lift))) {
          const float v = fmaxf(top - lift, m), f = m == v ? 1.0f : ex2_approx(m - v);
          m = v;
          l *= f;
          if (any) {                                          // the row of O, once the product before is in it
            ok = wait_sum();
            if (!ok) break;
#pragma unroll 1
            for (int d = 0; d < D; d += 32) {
              uint32_t o[32];
              tc::load32(o, sum_at + d);
              tc::load_wait();
              tc::pin32(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tc::store32(sum_at + d, o);
            }
          }
        }
        tc::load32(ra, s_at);
        const float ref = m == -INFINITY ? 0.0f : m;
        const uint64_t scale2 = tc::two(P.scale, P.scale), ref2 = tc::two(-ref, -ref);
        uint64_t sum0 = 0, sum1 = 0;                          // four chains
#pragma unroll
        for (int i = 0; i < kKeys / 32; ++i) {
          uint32_t (&r)[32] = i & 1 ? rb : ra;
          tc::load_wait();
          tc::pin32(r);
          if (i + 1 < kKeys / 32) tc::load32(i & 1 ? ra : rb, s_at + 32 * i + 32);
          ready(r, i);
          // A weight is off by at most 2^-9 of itself in bf16 (2^-12 in f16), at random over the
          // keys; the sum takes it as it was.
          uint32_t w16[16];
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const uint64_t a = tc::two(__uint_as_float(r[c]), __uint_as_float(r[c + 1]));
            const uint64_t b = tc::two(__uint_as_float(r[c + 2]), __uint_as_float(r[c + 3]));
            float p[4];
            tc::apart(E4M3 ? tc::add2(a, ref2) : tc::fma2(a, scale2, ref2), p[0], p[1]);
            tc::apart(E4M3 ? tc::add2(b, ref2) : tc::fma2(b, scale2, ref2), p[2], p[3]);
#pragma unroll
            for (int x = 0; x < 4; ++x) p[x] = ex2_approx(p[x]);
            if (E4M3) {
              const float4 inv = *reinterpret_cast<const float4*>(sc + 2 * kKeys + 32 * i + c);
              sum0 = tc::fma2(tc::two(p[0], p[1]), tc::two(inv.x, inv.y), sum0);
              sum1 = tc::fma2(tc::two(p[2], p[3]), tc::two(inv.z, inv.w), sum1);
            } else {
              sum0 = tc::add2(tc::two(p[0], p[1]), sum0);
              sum1 = tc::add2(tc::two(p[2], p[3]), sum1);
            }
            w16[c / 2] = pack2<HT>(p[0], p[1]);
            w16[c / 2 + 1] = pack2<HT>(p[2], p[3]);
          }
          tc::store16(s_at + 16 * i, w16);
        }
        {
          float l0, l1;
          tc::apart(tc::add2(sum0, sum1), l0, l1);
          l += l0 + l1;
        }
        tc::store_wait();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::bar_arrive(tc::smem_u32(&s_bars.p_full[buf]));
        any = true;
        ++pv;
        if (kSlots == 1) buf ^= 1;
      }
      before += max(w.je - jb, 0);
      if (any && ok) ok = wait_sum();
      if (!ok) l = NAN;

      // ---- the item's rows, or this part of them
      const bool joined = !w.whole || w.few;                  // more than one sum to a row
      const int first_block = w.first_block, part = static_cast<int>(blockIdx.x) - first_block;
      auto part_slot = [&](int p) { return p == 0 ? 2 * first_block + 1 : 2 * (first_block + p); };
      if (!joined) {
        // a sum of zero (no key has mass) gives zeros
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* o = static_cast<uint16_t*>(P.out) + (w.r.q0 + token) * P.o_tok + head * P.o_head;
        if (live && P.lse) P.lse[static_cast<long long>(w.r.q0 + token) * P.hq + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
#pragma unroll 1
        for (int d = 0; d < D; d += 32) {
          uint32_t x[32];
          if (any && ok) {
            tc::load32(x, sum_at + d);
            tc::load_wait();
            tc::pin32(x);
          }
          const bool none = !any || l == 0.0f;
          uint32_t h[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            h[i] = !ok ? pack2<DT>(NAN, NAN) : none ? 0u : pack2<DT>(__uint_as_float(x[2 * i]) * inv, __uint_as_float(x[2 * i + 1]) * inv);
          if (live) {
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(o + d + 8 * i) = make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
          }
        }
        tc::fence_before();
      } else {
        const long long at = static_cast<long long>(part_slot(part)) * S::kRows + slot * 128 + row;
        if (live) P.part_ml[at] = make_float2(any || !ok ? m : -INFINITY, l);
        float* o = P.part_o + at * D;
#pragma unroll 1
        for (int d = 0; d < D && any && ok; d += 32) {
          uint32_t x[32];
          tc::load32(x, sum_at + d);
          tc::load_wait();
          tc::pin32(x);
          if (live) {
#pragma unroll
            for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(o + d + 4 * i) = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
          }
        }
        tc::fence_before();
        // the last part's block joins them all; a whole item's two sums are joined here
        const int parts = w.parts;
        sync_some(1, 128 * kSlots);
        if (tid == 0) {
          bool last = true;
          if (parts > 1) {
            unsigned* counter = P.counters + first_block;
            unsigned n;
            asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(n) : "l"(counter) : "memory");
            last = n + 1u == static_cast<unsigned>(parts);
            if (last) *counter = 0u;
          }
          s_flag = last;
        }
        sync_some(1, 128 * kSlots);
        const bool mine = *static_cast<volatile int*>(&s_flag) != 0;
        if (mine) {
          // A warp to a row; triple x of a row is part x, or of few rows part x / 2, slot x % 2.
          const int sums = w.few ? 2 * parts : parts;
          for (int rr = warp; rr < w.rows; rr += 4 * kSlots) {
            auto where = [&](int x) {
              const int p = w.few ? x >> 1 : x;
              return static_cast<long long>(part_slot(p)) * S::kRows + (w.few ? (x & 1) * 128 : 0) + rr;
            };
            float mm = -INFINITY, ll = 0.0f, acc[D / 32];
            bool bad = false;
            for (int x = lane; x < sums; x += 32) {
              const float2 v = __ldcg(P.part_ml + where(x));
              mm = fmaxf(mm, v.x);
              bad |= v.y != v.y;
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xFFFFFFFFu, mm, o));
            bad = __any_sync(0xFFFFFFFFu, bad);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;
            for (int x0 = 0; x0 < sums; x0 += 32) {
              float f = 0.0f;
              if (x0 + lane < sums) {
                const float2 v = __ldcg(P.part_ml + where(x0 + lane));
                f = v.x == -INFINITY ? 0.0f : ex2_approx(v.x - mm);
                ll = fmaf(v.y, f, ll);
              }
              const int n = min(32, sums - x0);
#pragma unroll 4
              for (int x = 0; x < n; ++x) {
                const float g = __shfl_sync(0xFFFFFFFFu, f, x);
                if (g != 0.0f) {                              // a sum of nothing was not written
                  const float* src = P.part_o + where(x0 + x) * D + lane;
#pragma unroll
                  for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(g, __ldcg(src + 32 * i), acc[i]);
                }
              }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) ll += __shfl_xor_sync(0xFFFFFFFFu, ll, o);
            if (bad) ll = NAN;
            const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
            const int packed_r = w.row0 + rr, tok = packed_r / P.group, hd = w.head * P.group + packed_r - tok * P.group;
            uint16_t* dst = static_cast<uint16_t*>(P.out) + (w.r.q0 + tok) * P.o_tok + hd * P.o_head + lane;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) dst[32 * i] = static_cast<uint16_t>(DType<DT>::to_raw(acc[i] * inv));
            if (P.lse && lane == 0) P.lse[static_cast<long long>(w.r.q0 + tok) * P.hq + hd] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * kLn2;
          }
        }
        sync_some(1, 128 * kSlots);                           // the flag and the part's room are free again
      }
    }
  } else if (warp >= kLoaders && warp < kLoaders + 4) {
    // ================================================ keys and values to the ring
    constexpr int kMine = kKeys / 4;                          // rows of a warp
    const int wl = warp - kLoaders;
    unsigned n = 0, tiles = 0;                                // loads, key tiles so far
    uint32_t q_phase = 0;
    bool ok = true;
    constexpr unsigned kLag = 2;
    unsigned long long waiting = 0;                           // ring slots filled by threads' copies that the products do not
    unsigned told_late = 0;                                   // know of yet, oldest in the low byte; how many
    auto tell = [&](unsigned at) {
      tc::fence_smem();
      __syncwarp();
      if (lane == 0) tc::bar_arrive(tc::smem_u32(&s_bars.kv_full[at]));
    };
    auto tell_oldest = [&]() {
      tell(static_cast<unsigned>(waiting & 255));
      waiting >>= 8;
      --told_late;
    };
    auto free_slot = [&]() { return wait(&s_bars.kv_empty[n % kRing], ((n / kRing) & 1) ^ 1); };

    while (ok && w.next(P)) {
      if (w.jb >= w.je) continue;
      const bool shared = kSlots == 2 && !w.few;
      if (!E4M3) {                                            // the item's queries
        cp_wait<0>();
        while (told_late) tell_oldest();
        ok = wait(&s_bars.q_empty, q_phase ^ 1);
        q_phase ^= 1;
        if (!ok) break;
        for (int g = wl; g < (shared ? 8 : 4); g += 4) {      // 32 rows at a time
          const int my = 32 * g + lane;
          long long off = -1;
          if (my < w.rows) {
            const int packed = w.row0 + my, token = packed / P.group;
            off = (w.r.q0 + token) * P.q_tok + (w.head * P.group + packed - token * P.group) * P.q_head;
          }
          const uint32_t dst = s_q + (g >> 2) * S::kQ + (g & 3) * 32 * 128;
          constexpr int kChunks = D / 8;
#pragma unroll 8
          for (int x = 0; x < kChunks; ++x) {
            const int c = x * 32 + lane, r = c / kChunks, col = c % kChunks;
            const long long o = __shfl_sync(0xFFFFFFFFu, off, r);
            cp16(dst + (col / 8) * (128 * 128) + r * 128 + ((col % 8) ^ (r & 7)) * 16,
                 static_cast<const uint16_t*>(P.q) + (o < 0 ? 0 : o + col * 8), o >= 0);
          }
        }
        cp_commit();
        cp_wait<0>();
        tc::fence_smem();
        __syncwarp();
        if (lane == 0) tc::bar_arrive(tc::smem_u32(&s_bars.q_full));
      }

      const int* pages = C.indices + w.r.first;
      const int len = w.r.len, head = w.head, je = w.je;
      auto nth_page = [&](int key) { return P.page_shift >= 0 ? key >> P.page_shift : key / C.page_size; };
      const int ahead = shared ? 1 : 2;
      int page_next = 0;
      auto page_of = [&](int j) -> int {
        const int key = j * kKeys + wl * kMine + lane;
        return lane < kMine && j < je && key < len ? min(max(pages[nth_page(key)], 0), C.num_pages - 1) : -1;
      };
      // the next loads in order: K jb .. (ahead of them), then V j, K j + ahead
      int jk = w.jb, jv = w.jb;
      page_next = page_of(jk);
      auto next_load = [&](bool* is_v, int* j, int* page) {
        *is_v = jk >= je || jk - jv >= ahead;
        *j = *is_v ? jv++ : jk++;
        if (*is_v) {
          *page = page_of(*j);                                // read a while ago: in L1
        } else {
          *page = page_next;
          page_next = page_of(jk);
        }
      };
      const int loads = 2 * (je - w.jb);
      if (!E4M3) {
        // pages of a tile that the copy engine brings, a lane to a page
        const int in_tile = P.boxes ? max(1, kKeys >> P.page_shift) : 0, slots = kKeys / max(1, in_tile);
        auto listed = [&](int j) { return lane < in_tile && (j + 1) * kKeys <= len ? pages[((j * kKeys) >> P.page_shift) + lane] : 0; };
        int box_next = listed(jk);
        for (int i = 0; i < loads; ++i) {
          bool is_v;
          int j, page;
          const bool v_next = jk >= je || jk - jv >= ahead;
          if (P.boxes && ((v_next ? jv : jk) + 1) * kKeys <= len) {
            // a whole tile: boxes of 64 elements by a page's slots, dealt to the warps
            is_v = v_next;
            j = is_v ? jv++ : jk++;
            int at = is_v ? listed(j) : box_next;             // values' pages were read a while ago: in L1
            if (!is_v) {
              box_next = listed(jk);
              if (jk < je && (jk + 1) * kKeys > len) page_next = page_of(jk);
            }
            at = min(max(at, 0), C.num_pages - 1);
            ok = free_slot();
            if (!ok) break;
            const uint32_t dst = s_ring + (n % kRing) * S::kTile, bar = tc::smem_u32(&s_bars.kv_full[n % kRing]);
            const void* map = is_v ? &P.v_map : &P.k_map;
            const int boxes = in_tile * S::kBlocks, mine = (boxes - wl + 3) / 4;
            const int slot = (j * kKeys) & (C.page_size - 1);
            if (tc::elect()) tc::bar_expect(bar, mine * slots * 128);
            for (int x = wl; x < boxes; x += 4) {
              const int nth = x / S::kBlocks, block = x - nth * S::kBlocks;
              const int pg = __shfl_sync(0xFFFFFFFFu, at, nth);
              if (tc::elect()) tc::copy_box(dst + block * (kKeys * 128) + nth * slots * 128, map, block * 64, slot, head, pg, bar);
            }
            ++n;
            continue;
          }
          next_load(&is_v, &j, &page);
          const kv::Side16& side = is_v ? P.v : P.k;
          const int key = j * kKeys + wl * kMine + lane;
          unsigned off = 0;
          if (page >= 0) off = page * side.page + static_cast<unsigned>(key - nth_page(key) * C.page_size) * side.slot + head * side.head;
          const unsigned live = __ballot_sync(0xFFFFFFFFu, page >= 0);
          ok = free_slot();
          if (!ok) break;
          const uint32_t dst = s_ring + (n % kRing) * S::kTile + wl * kMine * 128;
          constexpr int kChunks = D / 8;
#pragma unroll
          for (int x = 0; x < kMine * kChunks / 32; ++x) {
            const int c = x * 32 + lane, r = c / kChunks, col = c % kChunks;
            const unsigned o = __shfl_sync(0xFFFFFFFFu, off, r);
            const bool there = (live >> r) & 1u;              // past the length: zeros
            cp16(dst + (col / 8) * (kKeys * 128) + r * 128 + ((col % 8) ^ (r & 7)) * 16, side.base + (there ? o + col : 0u) * 16ull, there);
          }
          cp_commit();
          waiting |= static_cast<unsigned long long>(n % kRing) << (8 * told_late);
          ++told_late;
          ++n;
          if (told_late > kLag) {
            cp_wait<kLag>();
            tell_oldest();
          }
        }
      } else {
        constexpr int kChunks = D / 16, kEach = kMine * kChunks / 32;
        uint4 now[kEach], then[kEach];
        float ks = 0.0f, vs = 0.0f, ks_then = 0.0f, vs_then = 0.0f;
        bool is_v = false, is_v_then = false;
        int j_then = 0;
        bool on = false, on_then = false;
        auto fetch = [&]() {
          int page;
          next_load(&is_v_then, &j_then, &page);
          const kv::Side16& side = is_v_then ? P.v : P.k;
          const int key = j_then * kKeys + wl * kMine + lane;
          unsigned off = 0;
          on_then = page >= 0;
          ks_then = vs_then = 0.0f;
          if (on_then) {
            const int slot = key - nth_page(key) * C.page_size;
            off = page * side.page + static_cast<unsigned>(slot) * side.slot + head * side.head;
            if (!is_v_then) {
              const long long at = (static_cast<long long>(page) * C.heads + head) * C.page_size + slot;
              ks_then = P.k.scale[at];
              vs_then = P.v.scale[at];
            }
          }
          const unsigned live = __ballot_sync(0xFFFFFFFFu, on_then);
#pragma unroll
          for (int x = 0; x < kEach; ++x) {
            const int c = x * 32 + lane, r = c / kChunks, col = c % kChunks;
            const unsigned o = __shfl_sync(0xFFFFFFFFu, off, r);
            then[x] = make_uint4(0, 0, 0, 0);
            if ((live >> r) & 1u) then[x] = __ldcg(reinterpret_cast<const uint4*>(side.base + (static_cast<unsigned long long>(o) + col) * 16ull));
          }
        };
        fetch();
        for (int i = 0; i < loads; ++i) {
#pragma unroll
          for (int x = 0; x < kEach; ++x) now[x] = then[x];
          ks = ks_then; vs = vs_then; is_v = is_v_then; on = on_then;
          if (i + 1 < loads) fetch();
          ok = free_slot();
          if (!ok) break;
          const uint32_t dst = s_ring + (n % kRing) * S::kTile + wl * kMine * 128;
#pragma unroll
          for (int x = 0; x < kEach; ++x) {
            const int c = x * 32 + lane, r = c / kChunks, col = c % kChunks;
            uint32_t h[8];
            e4m3x4(now[x].x, h[0], h[1]);
            e4m3x4(now[x].y, h[2], h[3]);
            e4m3x4(now[x].z, h[4], h[5]);
            e4m3x4(now[x].w, h[6], h[7]);
            const uint32_t row = dst + (col / 4) * (kKeys * 128) + r * 128;
            const int c0 = (col % 4) * 2;
            st16(row + (c0 ^ (r & 7)) * 16, h[0], h[1], h[2], h[3]);
            st16(row + ((c0 + 1) ^ (r & 7)) * 16, h[4], h[5], h[6], h[7]);
          }
          if (!is_v && lane < kMine) {
            float* sc = reinterpret_cast<float*>(base_p + (s_scales - base) + (tiles % S::kScaleRing) * S::kScales) + wl * kMine + lane;
            const float v = max_nan(vs, 8e-28f);              // 2^-90
            sc[0] = on ? ks : 0.0f;
            sc[kKeys] = on ? lg2(v) : 0.0f;
            sc[2 * kKeys] = on ? rcp(v) : 0.0f;
          }
          if (!is_v) ++tiles;
          tell(n % kRing);
          ++n;
        }
      }
    }
    cp_wait<0>();
    while (ok && told_late) tell_oldest();
  } else if (warp == kIssuer) {
    // ================================================================ products
    unsigned n = 0, products = 0;                             // loads taken, products O += P V
    uint32_t q_phase = 0, p_phase = 0;                        // a bit a buffer
    bool ok = true;
    constexpr uint32_t score = tc::product(HT == ECAH_DTYPE_BF16, kKeys, false), sum = tc::product(HT == ECAH_DTYPE_BF16, D, true);
    auto scores = [&](int buf, int q_tile, unsigned at) {
      if (tc::elect()) {
        const uint64_t a = tc::tile_desc(s_q + q_tile * S::kQ, 0), b = tc::tile_desc(s_ring + (at % kRing) * S::kTile, 0);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc::mma(tmem + buf * S::kBuffer, a + (k / 4) * (128 * 128 >> 4) + (k % 4) * 2, b + (k / 4) * (kKeys * 128 >> 4) + (k % 4) * 2, score, k > 0);
        tc::commit(tc::smem_u32(&s_bars.s_full[buf]));
      }
      __syncwarp();
    };
    auto weigh = [&](int slot, int buf, unsigned at, bool add) {
      if (tc::elect()) {
        const uint64_t b = tc::tile_desc(s_ring + (at % kRing) * S::kTile, kKeys * 128);
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          tc::mma_ts(tmem + S::kSum + slot * D, tmem + buf * S::kBuffer + k * 8, b + k * (2048 >> 4), sum, add || k > 0);
        tc::commit(tc::smem_u32(&s_bars.pv_done[kSlots == 2 ? slot : products & 1]));
      }
      ++products;
      __syncwarp();
    };
    auto release = [&](unsigned at) {
      if (tc::elect()) tc::commit(tc::smem_u32(&s_bars.kv_empty[at % kRing]));
      __syncwarp();
    };
    auto arrived = [&](unsigned at) {
      const bool there = wait(&s_bars.kv_full[at % kRing], (at / kRing) & 1);
      tc::fence_after();
      return there;
    };
    auto weights = [&](int buf) {
      const bool there = wait(&s_bars.p_full[buf], p_phase >> buf & 1);
      p_phase ^= 1u << buf;
      tc::fence_after();
      return there;
    };
    while (ok && w.next(P)) {
      const int count = w.je - w.jb, first = w.je0 - w.jb;    // first: tiles of the first half
      if (count <= 0) continue;
      const bool few = w.few;
      ok = wait(&s_bars.q_full, q_phase);
      q_phase ^= 1;
      if (!ok) break;
      tc::fence_after();
      if (kSlots == 2 && !few) {
        if (!(ok = arrived(n))) break;
        if (first > 0) scores(0, 0, n);
        scores(1, 1, n);
        release(n);
        ++n;
        for (int x = 0; x < count && ok; ++x) {               // load n: V x; n + 1: K x + 1
          const bool again = x + 1 < count;
          if (!(ok = arrived(n))) break;
          if (x < first) {
            if (!(ok = weights(0))) break;
            weigh(0, 0, n, x > 0);
          }
          if (again && !(ok = arrived(n + 1))) break;
          if (x + 1 < first) scores(0, 0, n + 1);
          if (!(ok = weights(1))) break;
          weigh(1, 1, n, x > 0);
          release(n);
          if (again) {
            scores(1, 1, n + 1);
            release(n + 1);
          }
          n += again ? 2 : 1;
        }
      } else {
        const int lead = min(2, count);
        for (int x = 0; x < lead && ok; ++x) {
          if (!(ok = arrived(n))) break;
          scores(x, 0, n);
          release(n);
          ++n;
        }
        for (int x = 0; x < count && ok; ++x) {               // load n: V x; n + 1: K x + 2
          if (!(ok = arrived(n)) || !(ok = weights(x & 1))) break;
          weigh(kSlots == 2 ? x & 1 : 0, x & 1, n, x >= kSlots);
          release(n);
          ++n;
          if (x + 2 < count) {
            if (!(ok = arrived(n))) break;
            scores(x & 1, 0, n);
            release(n);
            ++n;
          }
        }
      }
      if (!ok) break;
      if (tc::elect()) tc::commit(tc::smem_u32(&s_bars.q_empty));
      __syncwarp();
    }
    // nothing is in flight when the tensor memory is given back
    if (tc::elect()) tc::commit(tc::smem_u32(&s_bars.done));
    __syncwarp();
    for (int i = 0; i < kTries && !tc::bar_test(tc::smem_u32(&s_bars.done), 0); ++i) {}
  }

  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == kIssuer) tc::tmem_free(tmem, S::kColumns);
}

using KernelFn = void (*)(const Params);
struct Variant {
  KernelFn fn;
  int smem;
};

template <int DT, bool E4M3>
static Variant variant_for(int D) {
  switch (D) {
    case 64: return {prefill_kernel<DT, E4M3, 64>, Shape<64, E4M3>::kSmem};
    case 96: return {prefill_kernel<DT, E4M3, 96>, Shape<96, E4M3>::kSmem};
    case 128: return {prefill_kernel<DT, E4M3, 128>, Shape<128, E4M3>::kSmem};
    case 192: return {prefill_kernel<DT, E4M3, 192>, Shape<192, E4M3>::kSmem};
    default: return {prefill_kernel<DT, E4M3, 256>, Shape<256, E4M3>::kSmem};
  }
}

// A side of the cache as the copy engine reads it; false where it cannot (a stride of
// zero, a driver that has no such call): threads copy the rows then.
static bool box_map(CUtensorMap* map, const kv::Side& s, const ecah_kv_cache& c, int slots) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<Encode>(f);
  }();
  if (!encode) return false;
  const cuuint64_t row = static_cast<cuuint64_t>(c.head_dim) * 2;
  const cuuint64_t sizes[4] = {static_cast<cuuint64_t>(c.head_dim), static_cast<cuuint64_t>(c.page_size), static_cast<cuuint64_t>(c.num_kv_heads),
                               static_cast<cuuint64_t>(c.num_pages)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(s.slot) * 2, static_cast<cuuint64_t>(s.head) * 2, static_cast<cuuint64_t>(s.page) * 2};
  for (int i = 0; i < 3; ++i) {
    if (sizes[i + 1] == 1) strides[i] = row;                  // of a dimension of one the stride may be anything
    if (strides[i] == 0 || strides[i] >= 1ull << 40) return false;
  }
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(slots), 1, 1}, steps[4] = {1, 1, 1, 1};
  return encode(map, c.kv_dtype == ECAH_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, s.base, sizes, strides,
                box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Workspace: counters, the parts' (m, l), their sums.  A block has at most two parts of
// items that it shares with others.
struct Layout {
  size_t ml, o, total;
};

static Layout layout(int sms, int D) {
  const size_t rows = (2 * static_cast<size_t>(sms) + 2) * (D <= 128 ? 256 : 128);
  Layout L;
  L.ml = (sms * sizeof(unsigned) + 255) / 256 * 256;
  L.o = L.ml + rows * sizeof(float2);
  L.total = L.o + rows * D * sizeof(float);
  return L;
}

}  // namespace prefill
}  // namespace ecah

using namespace ecah;

extern "C" {

size_t ecah_paged_prefill_workspace_bytes(int32_t head_dim) {
  if (!kv::head_dim_ok(head_dim) || device_sms() <= 0) return 0;
  return prefill::layout(device_sms(), head_dim).total;
}

int ecah_paged_prefill(const ecah_prefill_args* a, void* stream) { return ecah_paged_prefill_bounded(a, prefill::kTries, stream); }

int ecah_paged_prefill_bounded(const ecah_prefill_args* a, int32_t tries, void* stream) {
  if (!a) return ECAH_ERR_NULL;
  if (a->abi_version != ECAH_SAMPLER_ABI_VERSION) return ECAH_ERR_ABI;
  const int st = kv::check_cache(a->cache, a->dtype);
  if (st != ECAH_OK) return st;
  const ecah_kv_cache& c = a->cache;
  if (a->tokens < 0 || a->num_qo_heads < 1 || a->num_qo_heads % c.num_kv_heads || !(a->sm_scale > 0.0f)) return ECAH_ERR_SHAPE;
  for (long long s : {a->q_token_stride, a->q_head_stride, a->out_token_stride, a->out_head_stride})
    if (s < 0 || s % 8) return ECAH_ERR_SHAPE;
  const int group = a->num_qo_heads / c.num_kv_heads;
  // rows are counted in 32 bits, and so are the entries of the page list
  if (static_cast<long long>(a->tokens) * group > 0x7FFFFFFFll - 1024 || c.num_indices > 0x7FFFFFFF) return ECAH_ERR_SHAPE;
  if (c.batch == 0 || a->tokens == 0) return ECAH_OK;
  if (!a->q || !a->out || !a->qo_indptr || !a->kv_last_page_len) return ECAH_ERR_NULL;
  if (!aligned16(a->q) || !aligned16(a->out)) return ECAH_ERR_SHAPE;
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < ecah_paged_prefill_workspace_bytes(c.head_dim))
    return ECAH_ERR_WORKSPACE;
  const int sms = device_sms();
  if (sms <= 0) return ECAH_ERR_LAUNCH;
  prefill::Params P = {};
  P.q = a->q; P.out = a->out; P.lse = a->lse;
  P.qo_indptr = a->qo_indptr; P.last_page_len = a->kv_last_page_len;
  P.q_tok = a->q_token_stride; P.q_head = a->q_head_stride;
  P.o_tok = a->out_token_stride; P.o_head = a->out_head_stride;
  P.tokens = a->tokens; P.hq = a->num_qo_heads; P.group = group; P.causal = a->causal;
  P.page_shift = kv::page_shift(c.page_size);
  P.tries = tries;
  P.scale = a->sm_scale * kLog2e;
  P.cache = kv::make_cache(c);
  const bool e4m3 = c.kv_dtype == ECAH_KV_E4M3;
  if (!kv::side16(P.cache.k, c.num_pages, c.page_size, c.num_kv_heads, e4m3 ? 1 : 2, &P.k) ||
      !kv::side16(P.cache.v, c.num_pages, c.page_size, c.num_kv_heads, e4m3 ? 1 : 2, &P.v))
    return ECAH_ERR_SHAPE;
  const prefill::Layout L = prefill::layout(sms, c.head_dim);
  unsigned char* ws = static_cast<unsigned char*>(a->workspace);
  P.counters = reinterpret_cast<unsigned*>(ws);
  P.part_ml = reinterpret_cast<float2*>(ws + L.ml);
  P.part_o = reinterpret_cast<float*>(ws + L.o);
  const prefill::Variant v =
      a->dtype == ECAH_DTYPE_F16 ? (e4m3 ? prefill::variant_for<ECAH_DTYPE_F16, true>(c.head_dim) : prefill::variant_for<ECAH_DTYPE_F16, false>(c.head_dim))
                                 : (e4m3 ? prefill::variant_for<ECAH_DTYPE_BF16, true>(c.head_dim) : prefill::variant_for<ECAH_DTYPE_BF16, false>(c.head_dim));
  // Whole tiles by the copy engine where a page is a power of two of 8 slots or more (the
  // swizzle goes by 8 rows); smaller or odd pages and 8-bit rows go through threads.
  const int keys = c.head_dim <= 128 ? 128 : 64;
  P.boxes = !e4m3 && P.page_shift >= 3 && prefill::box_map(&P.k_map, P.cache.k, c, std::min(c.page_size, keys)) &&
            prefill::box_map(&P.v_map, P.cache.v, c, std::min(c.page_size, keys));
  return launch_kernel(v.fn, dim3(sms), prefill::kT, v.smem, reinterpret_cast<cudaStream_t>(stream), P) ? ECAH_OK : ECAH_ERR_LAUNCH;
}

}  // extern "C"
