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
// Warps: 8 of softmax to a slot, two threads to a row (a half of the columns each, so no
// shuffles; they also rescale their row of O, which a lazily moved reference makes rare,
// and write it out), 3 that bring keys and values, one thread that issues the products.
// The softmax warps ask for the next item's queries before they write out this one's rows.
// Whole tiles come by the copy engine, a box to a page; the last tile of a request (zeros
// past its length), pages that no box fits and e4m3 rows by threads' 16-byte copies into
// the swizzled tiles, e4m3 codes through a ring of their own and converted on the way.
//
// Split: one block to an SM; all iterations of all items, in order, are divided over the
// blocks by the lengths the device holds (a captured launch serves any lengths).  An item
// that spans several blocks is joined by the block that arrives last, in the order of the
// parts, so results do not depend on which that is.
//
// Measured on one B200, passes through the Python entry point one after another with
// changing inputs: a prompt of 8192 tokens, 32/8 heads of 128, bf16 566 us (972 TFLOP/s, 69 %
// of the sustained GEMM rate) under the power cap at 1.67 GHz, 490 in short runs at 1.97 GHz
// (1.1 PFLOP/s, 67 % of the burst rate); 16 packed prompts of 100 to 1024 tokens, 16/2 heads,
// f16 63; 64 drafts of 5 tokens over contexts up to 8000, 32/8 heads, bf16 97 (3.7 TB/s); 7
// chunks of up to 333 tokens behind up to 6001, bf16 110, e4m3 179; 2 prompts of heads of 256
// 70; a prompt of 37 tokens 15.
// What bounds the first: an iteration (256 rows by 128 keys) takes 4000 cycles, of which the
// products 2048 and the exponentials' unit 2048, since a slot's scores wait for its product
// and its softmax for the scores.  An item takes 6 to 9 us beside its iterations in a share of
// many small ones; the plan of the shares 1.5 (one request) to 4 us (64 requests).  Iterations
// of e4m3 caches take 6700 cycles (converting codes), of heads of 256 (128 rows by 64 keys)
// 3000 for products of 1024.
// Registers: 96 a thread.  16-bit caches of heads of 64 to 128 spill 40 bytes, e4m3 caches 16
// (heads of 256) to 80.

constexpr int kLoaders = 16;           // first of the warps that bring keys and values, and how many
constexpr int kLoadWarps = 3;
constexpr int kIssuer = 19;            // the warp that issues the products
constexpr int kT = 32 * (kIssuer + 1);
// Units of work: of an iteration (both halves of the rows against a key tile; few rows
// against two), and of starting and finishing an item.
constexpr unsigned kCost = 2, kFewCost = 4, kItemCost = 9, kFewItemCost = 4;
constexpr int kWhole = 6;              // items of up to so many iterations are not divided
constexpr unsigned kLeast = 8;         // units to a block at the least
constexpr int kWalks = 2 + kLoadWarps + 1;   // of the softmax slots, the loaders, the issuer
constexpr int kKeep = 128;             // requests looked at together
constexpr int kTries = 1 << 20;        // of a wait: more than one between warps of a block can need
constexpr float kLift = 7.0f;          // f16 weights begin at 2^7 and reach 2^15, so that small ones are not lost
constexpr float kLn2 = 0.6931471805599453f;

struct alignas(64) Params {
  CUtensorMap k_map, v_map;            // [pages][heads][slots][head_dim]; boxes of 64 elements (e4m3: rows) by the slots of a page in a tile
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
  float* part_o;                       // [2 blocks][slots][D / 4][128][4]
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
  static constexpr int kScales = E4M3 ? kKeys * 8 : 0;     // of a tile: key and value scales
  static constexpr int kRaw = E4M3 ? kKeys * (D + 8) : 0;  // of a tile as it is cached: codes, key and value scales
  static constexpr int kRaws = 3;                          // as many barriers in Bars
  static constexpr int kNotes = D == 64 || D == 192 || E4M3 ? 3584 : 3 * 1024;     // the block's Notes grow with its ring
  static constexpr int kRoom = 227 * 1024 - kNotes;
  static constexpr int bytes(int n) { return kSlots * kQ + n * kTile + (n / 2 + 2) * kScales + kRaws * kRaw; }
  static constexpr int ring(int n) { return n == 3 || bytes(n) <= kRoom ? n : ring(n - 1); }
  static constexpr int kRing = ring(8);
  static constexpr int kScaleRing = kRing / 2 + 2;
  static constexpr int kSmem = bytes(kRing) + kNotes;
  static constexpr int kHalf = kKeys / 2;                  // columns of a thread
  static constexpr int kBuffer = kKeys;                    // tensor-memory columns of one of the two score buffers
  static constexpr int kSum = 2 * kKeys;                   // first column of the sums
  static constexpr int kColumns = 512;
  static_assert(bytes(kRing) <= kRoom && kSum + kSlots * D <= kColumns, "");
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
  // Units of the order: an iteration's, and what starting and finishing the item takes.
  __device__ __forceinline__ unsigned unit() const { return few ? kFewCost : kCost; }
  __device__ __forceinline__ unsigned start() const { return few ? kFewItemCost : kItemCost; }
  __device__ __forceinline__ unsigned cost() const { return start() + iters * unit(); }
};

template <int D, bool E4M3>
__device__ __forceinline__ int tiles_of(const Params& P, const Request& r) {
  return (r.n * P.group + Shape<D, E4M3>::kRows - 1) / Shape<D, E4M3>::kRows;
}

// A block's share of the order, and everybody's.
struct Share {
  unsigned lo, hi, size, more;         // the first `more` blocks have size + 1, the others size
  __device__ __forceinline__ int block_of(unsigned x) const {
    return static_cast<int>(min(x < more * (size + 1) ? x / (size + 1) : more + (x - more * (size + 1)) / size, gridDim.x - 1));
  }
};

// The items of this block's share, in order.  Every role of warps walks them alike, with
// walks in shared memory: only what a loop uses is held in registers.
template <int D, bool E4M3>
struct Walk {
  using S = Shape<D, E4M3>;
  unsigned at, cost;                   // place of the item in the order, and its units
  Request r;
  int req, head, tile, tiles;
  // the present item's part
  int row0, rows, keys, jb, je, je0;   // key tiles [jb, je); of the first slot of two halves [jb, je0)
  int first_block, parts;
  bool fresh, few, whole, found;

  // The next item with work for this block; false behind the last.  For a warp with a walk
  // of its own.
  __device__ __forceinline__ bool next(const Params& P, const Share& share) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) found = advance(P, share);
    __syncwarp();
    return found;
  }
  // By one thread.
  __device__ __forceinline__ bool advance(const Params& P, const Share& share) {
    const unsigned lo = share.lo, hi = share.hi;
    while (true) {
      if (!fresh) {
        at += cost;
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
      cost = t.cost();
      const unsigned begin = at + t.start(), unit = t.unit();
      int i0 = 0, i1 = t.iters;
      whole = t.iters <= kWhole;
      first_block = blockIdx.x;
      parts = 1;
      if (whole) {
        if (at < lo) continue;
      } else {                         // iteration i is the block's that holds place begin + i unit
        i0 = lo <= begin ? 0 : min((lo - begin + unit - 1) / unit, static_cast<unsigned>(t.iters));
        i1 = hi <= begin ? 0 : min((hi - begin + unit - 1) / unit, static_cast<unsigned>(t.iters));
        if (i0 >= i1) continue;
        whole = i0 == 0 && i1 == t.iters;
        if (!whole) {
          first_block = share.block_of(begin);
          parts = max(1, share.block_of(begin + (t.iters - 1) * unit) - first_block + 1);
        }
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
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
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
// keeps a NaN
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float lg2(float x) {
  float r;
  asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// A barrier of `threads` threads that tells all of them whether one said so.
__device__ __forceinline__ bool any_of(int id, int threads, bool said) {
  uint32_t r;
  asm volatile("{ .reg .pred p, q; setp.ne.u32 q, %3, 0; barrier.cta.red.or.pred p, %1, %2, q; selp.u32 %0, 1, 0, p; }"
               : "=r"(r) : "r"(id), "r"(threads), "r"(static_cast<uint32_t>(said)) : "memory");
  return r != 0;
}
__device__ __forceinline__ void sync_some(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// The block's barriers.
template <int D, bool E4M3>
struct Bars {
  unsigned long long q_full, q_empty, done;
  unsigned long long kv_full[Shape<D, E4M3>::kRing], kv_empty[Shape<D, E4M3>::kRing];
  unsigned long long s_full[2], p_full[2], pv_done[2];
  unsigned long long raw_full[E4M3 ? 3 : 1], raw_empty[E4M3 ? 3 : 1];
};

// What the block keeps beside tiles.
template <int D, bool E4M3>
struct Notes {
  Bars<D, E4M3> bars;
  Share share;
  uint32_t tmem;
  int failed, flag;
  unsigned brought[kLoadWarps];        // tiles that a loader has announced on kv_full (e4m3: raw_full)
  Walk<D, E4M3> walk[kWalks + 4];      // the softmax slots have three each, in turn
  float other[2][2][128];                                     // between the threads of a row
};

template <int DT, bool E4M3, int D>
__global__ void __launch_bounds__(kT, 1) prefill_kernel(const __grid_constant__ Params P) {
  using S = Shape<D, E4M3>;
  constexpr int HT = E4M3 ? static_cast<int>(ECAH_DTYPE_F16) : DT;   // operand type of the products
  constexpr float lift = HT == ECAH_DTYPE_F16 ? kLift : 0.0f;
  // of a tile's weights in a thread: 2^15, the largest f16 weight; 64 of 2^kLazy in bf16
  constexpr float kMost = HT == ECAH_DTYPE_F16 ? 32768.0f : 16384.0f;
  constexpr int kKeys = S::kKeys, kRing = S::kRing, kSlots = S::kSlots;
  extern __shared__ __align__(1024) unsigned char base_p[];   // the swizzle goes by addresses
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = tc::smem_u32(base_p);
  Notes<D, E4M3>& notes = *reinterpret_cast<Notes<D, E4M3>*>(base_p + S::bytes(kRing));
  static_assert(sizeof(Notes<D, E4M3>) <= S::kNotes && S::bytes(kRing) % 16 == 0, "");
  Bars<D, E4M3>& s_bars = notes.bars;
  const uint32_t s_q = base, s_ring = base + kSlots * S::kQ, s_scales = s_ring + kRing * S::kTile,
                 s_raw = s_scales + S::kScaleRing * S::kScales;
  const kv::Cache& C = P.cache;

  grid_start();

  // ---- barriers, tensor memory
  if (tid == 0) {
    auto init = [&](unsigned long long* b, int n) { tc::bar_init(tc::smem_u32(b), n); };
    init(&s_bars.q_full, 8 * kSlots);
    init(&s_bars.q_empty, 1);
    init(&s_bars.done, 1);
    for (int i = 0; i < kRing; ++i) { init(&s_bars.kv_full[i], kLoadWarps); init(&s_bars.kv_empty[i], 1); }
    for (int i = 0; E4M3 && i < S::kRaws; ++i) { init(&s_bars.raw_full[i], kLoadWarps); init(&s_bars.raw_empty[i], kLoadWarps); }
    for (int i = 0; i < 2; ++i) { init(&s_bars.s_full[i], 1); init(&s_bars.p_full[i], 8); init(&s_bars.pv_done[i], 1); }
    tc::fence_smem();
    notes.failed = 0;
  }
  if (tid < kWalks) {
    notes.walk[tid].req = C.batch;                            // none, unless one is found below
    notes.walk[tid].fresh = true;
  }
  if (warp == kIssuer) tc::tmem_alloc(tc::smem_u32(&notes.tmem), S::kColumns);

  // ---- this block's share of the order.  The first `more` blocks take size + 1 units, the
  // others size.
  {
    struct Seen { Request r; int tiles; unsigned cost; };      // of a request; cost: of one head
    Seen* seen = reinterpret_cast<Seen*>(base_p + kSlots * S::kQ);   // the ring is not in use yet
    auto look = [&](int b0) {
      if (tid < kKeep && b0 + tid < C.batch) {
        seen[tid].r = request<kKeys>(P, b0 + tid);
        seen[tid].tiles = tiles_of<D, E4M3>(P, seen[tid].r);
      }
      __syncthreads();
      for (int i = warp; i < min(kKeep, C.batch - b0); i += kT / 32) {
        const Request r = seen[i].r;
        unsigned sum = 0;
        for (int t = lane; t < seen[i].tiles; t += 32) sum += Tile<D, E4M3>(P, r, t).cost();
        sum = __reduce_add_sync(0xFFFFFFFFu, sum);
        if (lane == 0) seen[i].cost = sum;
      }
      __syncthreads();
    };
    auto all = [&](int b0) {
      unsigned sum = 0;
      for (int i = lane; i < min(kKeep, C.batch - b0); i += 32) sum += seen[i].cost;
      return __reduce_add_sync(0xFFFFFFFFu, sum) * C.heads;
    };
    auto before = [&](unsigned v) {                           // sum of the lanes before
      unsigned inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned w = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += w;
      }
      return inc - v;
    };
    unsigned total = 0;
    for (int b0 = 0; b0 < C.batch; b0 += kKeep) {
      if (b0) __syncthreads();
      look(b0);
      total += all(b0);
    }
    const unsigned blocks = min(gridDim.x, max(1u, total / kLeast)), size = max(1u, total / blocks), more = total - size * blocks;
    const bool busy = blockIdx.x < blocks && total > 0;
    const unsigned lo = blockIdx.x * size + min(blockIdx.x, more), hi = lo + size + (blockIdx.x < more);
    if (warp < 2 && lane == 0) (warp == 0 ? notes.share.lo : notes.share.hi) = !busy ? 0 : warp == 0 ? lo : hi;
    if (tid == 64) { notes.share.size = size; notes.share.more = more; }
    unsigned run = 0;
    for (int b0 = 0; busy && b0 < C.batch && run < hi; b0 += kKeep) {
      if (C.batch > kKeep) {
        __syncthreads();
        look(b0);
      }
      const unsigned sum = all(b0), x = warp == 0 ? lo : hi;
      if (warp < 2 && x >= run && x < run + sum) {            // the item at an edge of the share
        unsigned p = run;
        int i = 0, t = 0;
        for (int i0 = 0; i0 < kKeep; i0 += 32) {              // its request,
          const unsigned c = i0 + lane < min(kKeep, C.batch - b0) ? seen[i0 + lane].cost * C.heads : 0, at = p + before(c);
          const unsigned here = __ballot_sync(0xFFFFFFFFu, x >= at && x < at + c);
          if (here) {
            i = i0 + __ffs(here) - 1;
            p = __shfl_sync(0xFFFFFFFFu, at, __ffs(here) - 1);
            break;
          }
          p = __shfl_sync(0xFFFFFFFFu, at + c, 31);
        }
        const Request r = seen[i].r;
        const int head = static_cast<int>((x - p) / max(1u, seen[i].cost));
        p += head * seen[i].cost;
        unsigned cost = 0;
        int iters = 0;
        for (int t0 = 0; t0 < seen[i].tiles; t0 += 32) {      // tile
          unsigned c = 0;
          if (t0 + lane < seen[i].tiles) {
            const Tile<D, E4M3> tile(P, r, t0 + lane);
            c = tile.cost();
            iters = tile.iters;
          }
          const unsigned at = p + before(c), here = __ballot_sync(0xFFFFFFFFu, x >= at && x < at + c);
          if (here) {
            const int l = __ffs(here) - 1;
            t = t0 + l;
            p = __shfl_sync(0xFFFFFFFFu, at, l);
            cost = __shfl_sync(0xFFFFFFFFu, c, l);
            iters = __shfl_sync(0xFFFFFFFFu, iters, l);
            break;
          }
          p = __shfl_sync(0xFFFFFFFFu, at + c, 31);
        }
        if (lane == 0 && iters <= kWhole) {
          // an edge inside an item that is not divided moves to the item's nearer end
          (warp == 0 ? notes.share.lo : notes.share.hi) = 2 * (x - p) < cost ? p : p + cost;
        }
        if (warp == 0 && lane < kWalks) {
          Walk<D, E4M3>& w = notes.walk[lane];
          w.at = p;
          w.r = r;
          w.req = b0 + i; w.head = head; w.tile = t; w.tiles = seen[i].tiles;
        }
      }
      run += sum;
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
  }
  const uint32_t tmem = notes.tmem;

  // Waits for a phase of a barrier; false when it ran out, here or in another warp: the
  // block then ends as fast as it can, and its results are NaN.
  auto wait = [&](unsigned long long* b, uint32_t parity) -> bool {
    const uint32_t bar = tc::smem_u32(b);
    bool ok = false;
    for (int i = 0; i < P.tries && !ok; ++i) {
      ok = tc::bar_test(bar, parity);
      if (!ok && *static_cast<volatile int*>(&notes.failed)) break;
    }
    ok = __all_sync(0xFFFFFFFFu, ok);
    if (!ok) *static_cast<volatile int*>(&notes.failed) = 1;
    return ok;
  };

  // An arrival of the warp once all its threads' copies so far are there; nobody waits here.
  auto arrive_copied = [&](unsigned long long* b) {
    const uint32_t bar = tc::smem_u32(b);
    asm volatile("cp.async.mbarrier.arrive.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
    __syncwarp();
    if (lane == 0) tc::bar_arrive(bar);
  };

  // a slot's 8 warps share a walk
  Walk<D, E4M3>& w = notes.walk[warp < kLoaders ? warp >> 3 : warp - kLoaders + 2];

  if (warp < 8 * kSlots) {
    // =============================================================== softmax
    const int slot = warp >> 3, half = (warp >> 2) & 1, row = (warp & 3) * 32 + lane;
    const int pair = 1 + slot * 4 + (warp & 3);               // the barrier of the two warps of these rows
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);
    const uint32_t sum_at = lanes + S::kSum + slot * D + half * (D / 2);   // this thread's half of its row of O
    constexpr int kC = S::kHalf / 32;
    uint32_t s_phase = 0, q_phase = 0;                        // a bit a buffer
    int before = 0;                                           // key tiles of the items before
    unsigned pv = 0;                                          // products O += P V of this slot so far
    // A wait that ran out: the warp goes through the motions (its barriers are awaited by
    // others), and its rows become NaN.
    bool ok = true;
    // The last product so far.  A slot's scores come after its product before, so at most
    // one is outstanding on a barrier; with one slot two are, on barriers in turn.
    auto wait_sum = [&]() {
      const unsigned x = pv - 1;
      ok = ok && (kSlots == 2 ? wait(&s_bars.pv_done[slot], x & 1) : wait(&s_bars.pv_done[x & 1], x >> 1 & 1));
      tc::fence_after();
    };
    // The 16-bit queries of an item, asked for while the item before it ends: a thread copies a
    // half of its row (a quarter of one that four threads share).
    auto ask = [&](const Walk<D, E4M3>& w, bool own_before) {
      if (!w.found || w.jb >= w.je) return;
      // Their place is free when the scores of the item before are computed; a slot with rows of
      // its own has seen its last ones, and learns from the item's first scores that the phase has
      // ended.  Where the item has none for it (a first half that sees no key) it looks here: its
      // next look, two phases ahead of the barrier, would succeed at once.
      const bool scored = slot != 0 || w.je0 > w.jb;
      if (!(own_before && kSlots == 2 && !w.few && scored)) ok = ok && wait(&s_bars.q_empty, q_phase ^ 1);
      q_phase ^= 1;
      if (ok) {
        const bool own_rows = kSlots == 2 && !w.few, quarters = kSlots == 2 && !own_rows;
        const int my = (own_rows ? slot * 128 : 0) + row, packed = w.row0 + my, token = packed / P.group;
        const bool live = my < w.rows;
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(P.q) + (live ? (w.r.q0 + token) * P.q_tok +
                               (w.head * P.group + packed - token * P.group) * P.q_head : 0));
        const uint32_t dst = s_q + (own_rows ? slot : 0) * S::kQ + row * 128;
        const int step = quarters ? 4 : 2;
#pragma unroll 4
        for (int c = quarters ? 2 * slot + half : half; c < D / 8; c += step)
          cp16(dst + (c / 8) * (128 * 128) + ((c % 8) ^ (row & 7)) * 16, src + (live ? c : 0), live);
      }
      arrive_copied(&s_bars.q_full);
    };
    if ((tid & 255) == 0) notes.walk[slot].found = notes.walk[slot].advance(P, notes.share);
    sync_some(10 + slot, 256);
    if (!E4M3) ask(notes.walk[slot], false);
    // Walks in turn: the one that is written while this item ends was read last two items ago,
    // and every warp has passed the barrier since.
    auto walk_at = [&](int turn) -> Walk<D, E4M3>& { return notes.walk[turn == 0 ? slot : kWalks + 2 * (turn - 1) + slot]; };
    for (int turn = 0;; turn = turn == 2 ? 0 : turn + 1) {
      Walk<D, E4M3>& w = walk_at(turn);
      if (!w.found) break;
      const bool own_rows = kSlots == 2 && !w.few;            // slots are halves of the rows
      const int my = (own_rows ? slot * 128 : 0) + row;       // row of the item
      const bool live = my < w.rows;
      const int packed = w.row0 + my;
      const int token = live ? packed / P.group : 0, head = w.head * P.group + packed - token * P.group;
      const int lim = live ? sees(P, w.r, token) : w.keys;    // other rows' scores are zeros, and not used
      const int least = __reduce_min_sync(0xFFFFFFFFu, lim);
      float scale = P.scale;

      if (E4M3 && w.jb < w.je) {
        // A row of queries, scaled by a power of two to a largest magnitude in [1, 2) so
        // that bf16 queries fit f16's range; the power goes into the score scale.  bf16's bits
        // fit f16's; entries below 2^-14 there are rounded by at most 2^-25.
        ok = ok && wait(&s_bars.q_empty, q_phase ^ 1);
        q_phase ^= 1;
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
        if ((own_rows || slot == 0) && ok) {
          const uint32_t dst = s_q + (own_rows ? slot : 0) * S::kQ + row * 128;
#pragma unroll 4
          for (int c = half; c < D / 8; c += 2) {
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

      float m = -INFINITY, l = 0.0f;                          // l: of this thread's columns
      bool any = false;                                       // the sum holds something
      const int step = own_rows || kSlots == 1 ? 1 : 2, jb = w.jb, je = own_rows && slot == 0 ? w.je0 : w.je;
      int buf = kSlots == 2 ? slot : 0;
      for (int j = jb + (own_rows || kSlots == 1 ? 0 : slot); j < je; j += step) {
        ok = ok && wait(&s_bars.s_full[buf], s_phase >> buf & 1);
        s_phase ^= 1u << buf;
        tc::fence_after();
        const uint32_t s_at = lanes + buf * S::kBuffer;
        const int c0 = half * S::kHalf;
        const float* sc = reinterpret_cast<const float*>(base_p + (s_scales - base) + ((before + j - jb) % S::kScaleRing) * S::kScales) + c0;
        const bool masked = (j + 1) * kKeys > least;
        const int left = lim - j * kKeys - c0;
        // 32 scores; e4m3 rows: times their key's scale
        auto read = [&](uint32_t (&r)[32], int i) {
          tc::load32(r, s_at + c0 + 32 * i);
          tc::load_wait();
          tc::pin32(r);
          if (E4M3) {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const float4 k = *reinterpret_cast<const float4*>(sc + 32 * i + c);
              float x, y;
              tc::apart(tc::mul2(tc::two(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), tc::two(k.x, k.y)), x, y);
              r[c] = __float_as_uint(x); r[c + 1] = __float_as_uint(y);
              tc::apart(tc::mul2(tc::two(__uint_as_float(r[c + 2]), __uint_as_float(r[c + 3])), tc::two(k.z, k.w)), x, y);
              r[c + 2] = __float_as_uint(x); r[c + 3] = __float_as_uint(y);
            }
          }
          if (masked) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (32 * i + c >= left) r[c] = 0xFF800000u;
          }
        };
        auto largest = [&](const uint32_t (&r)[32], float top) {
          float t0 = top, t1 = -INFINITY, t2 = -INFINITY, t3 = -INFINITY;
#pragma unroll
          for (int c = 0; c < 32; c += 8) {
            t0 = max3(t0, __uint_as_float(r[c]), __uint_as_float(r[c + 1]));
            t1 = max3(t1, __uint_as_float(r[c + 2]), __uint_as_float(r[c + 3]));
            t2 = max3(t2, __uint_as_float(r[c + 4]), __uint_as_float(r[c + 5]));
            t3 = max3(t3, __uint_as_float(r[c + 6]), __uint_as_float(r[c + 7]));
          }
          return max3(max_nan(t0, t1), t2, t3);
        };
        uint32_t w16[kC][16];
        uint64_t sum0, sum1, most;                            // of the weights; e4m3: most of their products with the scales
        auto weigh = [&](const uint32_t (&r)[32], int i, float ref) {
          // A weight is rounded by at most 2^-8 of itself in bf16 and 2^-11 in f16 (there, below
          // 2^-14, by 2^-25: 2^-32 of the row's largest, which lies at 2^7 or above), at random over
          // the keys; the sum takes it as it was.  An e4m3 value's scale goes into its weight.
          const uint64_t scale2 = tc::two(scale, scale), ref2 = tc::two(-ref, -ref);
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            float p[4];
            tc::apart(tc::fma2(tc::two(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), scale2, ref2), p[0], p[1]);
            tc::apart(tc::fma2(tc::two(__uint_as_float(r[c + 2]), __uint_as_float(r[c + 3])), scale2, ref2), p[2], p[3]);
            // All by the exponentials' unit (51 % busy with 8192 tokens).  A quarter of them by a
            // polynomial, off by 2.9e-6, took 506 us instead of 486: a slot's softmax gets longer.
#pragma unroll
            for (int e = 0; e < 4; ++e) p[e] = ex2_approx(p[e]);
            sum0 = tc::add2(tc::two(p[0], p[1]), sum0);
            sum1 = tc::add2(tc::two(p[2], p[3]), sum1);
            if (E4M3) {
              const float4 v = *reinterpret_cast<const float4*>(sc + kKeys + 32 * i + c);
              const uint64_t a = tc::mul2(tc::two(p[0], p[1]), tc::two(v.x, v.y)), b = tc::mul2(tc::two(p[2], p[3]), tc::two(v.z, v.w));
              most = tc::add2(most, tc::add2(a, b));
              tc::apart(a, p[0], p[1]);
              tc::apart(b, p[2], p[3]);
            }
            w16[i][c / 2] = pack2<HT>(p[0], p[1]);
            w16[i][c / 2 + 1] = pack2<HT>(p[2], p[3]);
          }
        };
        // The reference of the tiles before nearly always serves (scores pass it by less than
        // 2^8): weights are computed with it, and again with the largest score's where it did
        // not, which the sum of a thread's 64 weights tells.  A first tile begins with the latter.
        float ref = m == -INFINITY ? 0.0f : m;
        bool moved = !any;
#pragma unroll 1
        while (true) {
          if (moved) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < kC; ++i) {
              uint32_t r[32];
              read(r, i);
              if (E4M3) {                                     // of the weights with their scales
#pragma unroll
                for (int c = 0; c < 32; ++c) r[c] = __float_as_uint(fmaf(__uint_as_float(r[c]), scale, lg2(sc[kKeys + 32 * i + c])));
              }
              top = largest(r, top);
            }
            if (!E4M3) top *= scale;
            if (!any) sync_some(pair, 64);                    // both have read what the item before left there
            notes.other[slot][half][row] = top;
            sync_some(pair, 64);
            top = max_nan(top, notes.other[slot][half ^ 1][row]);
            const float v = fmaxf(top - lift, m), f = m == v ? 1.0f : ex2_approx(m - v);
            m = v;
            l *= f;
            if (any) {                                        // the row of O, once the product before is in it
              wait_sum();
#pragma unroll 1
              for (int d = 0; d < D / 2; d += 16) {
                uint32_t o[16];
                tc::load16(o, sum_at + d);
                tc::load_wait();
                tc::pin16(o);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tc::store16(sum_at + d, o);
              }
            }
            // a NaN or an infinite score makes the row NaN
            ref = !(top < INFINITY) ? NAN : m == -INFINITY ? 0.0f : m;
          }
          sum0 = sum1 = most = 0;
#pragma unroll
          for (int i = 0; i < kC; ++i) {
            uint32_t r[32];
            read(r, i);
            weigh(r, i, ref);
          }
          // the weights lie over scores that the other half's thread reads: both are past that here
          if (moved) {
            sync_some(pair, 64);
            break;
          }
          float a, b;
          tc::apart(E4M3 ? most : tc::add2(sum0, sum1), a, b);
          moved = any_of(pair, 64, !(a + b <= kMost) || (m == -INFINITY && left > 0));   // the last: no reference yet
          if (!moved) break;
        }
#pragma unroll
        for (int i = 0; i < kC; ++i) tc::store16(s_at + c0 / 2 + 16 * i, w16[i]);
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
      // the item after this, while the last product runs
      Walk<D, E4M3>& then = walk_at(turn == 2 ? 0 : turn + 1);
      if ((tid & 255) == 0) {
        then = w;
        then.found = then.advance(P, notes.share);
      }
      sync_some(10 + slot, 256);
      if (!E4M3) ask(then, own_rows && any);
      if (any) wait_sum();
      // Warps whose wait ran out arrive without waiting, and so may have let products begin before
      // others' weights or queries were there: the block's rows are NaN from here on.  (Those warps
      // said so before they arrived, and this warp has waited for the products since.)
      if (!ok || *static_cast<volatile int*>(&notes.failed)) l = NAN;
      notes.other[slot][half][row] = l;
      sync_some(pair, 64);
      l += notes.other[slot][half ^ 1][row];

      // ---- Few rows: both slots' sums of a row lie in its tensor-memory lane.  Each of its four
      // threads joins a quarter of their columns, in the first slot's place.
      constexpr int kQuarter = D / 4;
      const bool two_sums = kSlots == 2 && !own_rows;
      if (two_sums) {
        sync_some(pair, 64);                                  // both have read the other's sum
        notes.other[slot][half][row] = half == 0 ? m : l;
        tc::fence_before();
        sync_some(9, 512);
        tc::fence_after();
        const float2 a = make_float2(notes.other[0][0][row], notes.other[0][1][row]);
        const float2 b = make_float2(notes.other[1][0][row], notes.other[1][1][row]);
        m = fmaxf(a.x, b.x);
        const float fa = a.x == -INFINITY ? 0.0f : ex2_approx(a.x - m), fb = b.x == -INFINITY ? 0.0f : ex2_approx(b.x - m);
        l = a.y * fa + b.y * fb;
        if (a.y != a.y || b.y != b.y) l = NAN;
        const bool in_a = jb < w.je, in_b = jb + 1 < w.je;    // whether the slot had a tile
        any = in_a;
        if (in_b) {
          const uint32_t at = lanes + S::kSum + (2 * slot + half) * kQuarter;
#pragma unroll 1
          for (int d = 0; d < kQuarter; d += 8) {
            uint32_t x[8], y[8];
            tc::load8(x, at + d);
            tc::load8(y, at + D + d);
            tc::load_wait();
            tc::pin8(x);
            tc::pin8(y);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __float_as_uint(fmaf(fa, __uint_as_float(x[i]), fb * __uint_as_float(y[i])));
            tc::store8(at + d, x);
          }
          tc::store_wait();
        }
      }
      // where this thread's columns of the row's sum lie, and how many they are
      const int my_first = two_sums ? (2 * slot + half) * kQuarter : half * (D / 2), my_columns = two_sums ? kQuarter : D / 2;
      const uint32_t my_at = lanes + S::kSum + (two_sums ? 0 : slot * D) + my_first;
      const int tile = own_rows ? slot : 0;
      const bool speaks = half == 0 && (own_rows || slot == 0);   // for the row

      // ---- the item's rows, or this part of them
      const bool joined = !w.whole;
      const int first_block = w.first_block, part = static_cast<int>(blockIdx.x) - first_block;
      auto part_slot = [&](int p) { return p == 0 ? 2 * first_block + 1 : 2 * (first_block + p); };
      auto part_at = [&](int at, int tile) { return reinterpret_cast<uint4*>(P.part_o) + (static_cast<long long>(at) * kSlots + tile) * (D / 4) * 128; };
      if (!joined) {
        // a sum of zero (no key has mass) gives zeros
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* o = static_cast<uint16_t*>(P.out) + (w.r.q0 + token) * P.o_tok + head * P.o_head + my_first;
        if (live && speaks && P.lse)
          P.lse[static_cast<long long>(w.r.q0 + token) * P.hq + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
#pragma unroll 1
        for (int d = 0; d < my_columns; d += 32) {            // a multiple of 8: the last may be fewer
          uint32_t x[4][8] = {};
          if (any) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (d + 8 * i < my_columns) tc::load8(x[i], my_at + d + 8 * i);
            tc::load_wait();
#pragma unroll
            for (int i = 0; i < 4; ++i) tc::pin8(x[i]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              h[e] = l == 0.0f ? 0u : pack2<DT>(__uint_as_float(x[i][2 * e]) * inv, __uint_as_float(x[i][2 * e + 1]) * inv);
            if (live && d + 8 * i < my_columns) *reinterpret_cast<uint4*>(o + d + 8 * i) = make_uint4(h[0], h[1], h[2], h[3]);
          }
        }
        tc::fence_before();
      } else {
        // The block that arrives last joins the parts, in their order.  Where all others have
        // arrived already (a part at the end of a share joins one from the start of the next) this
        // one's sum is taken from where it is.
        const int parts = w.parts;
        unsigned* counter = P.counters + first_block;
        if (tid == 0) {
          unsigned n;
          asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(counter) : "memory");
          notes.flag = n + 1u == static_cast<unsigned>(parts);
          if (notes.flag) *counter = 0u;
        }
        sync_some(9, 256 * kSlots);
        const bool here = *static_cast<volatile int*>(&notes.flag) != 0;
        bool mine = here;
        if (!here) {
          if (live && speaks) P.part_ml[static_cast<long long>(part_slot(part)) * S::kRows + tile * 128 + row] = make_float2(m, l);
          // [128 rows' part][D / 4][128][4]: neighbouring rows side by side
          uint4* o = part_at(part_slot(part), tile) + my_first / 4 * 128 + row;
#pragma unroll 2
          for (int d = 0; d < my_columns && any; d += 8) {
            uint32_t x[8];
            tc::load8(x, my_at + d);
            tc::load_wait();
            tc::pin8(x);
            if (live) {
#pragma unroll
              for (int i = 0; i < 2; ++i) o[(d / 4 + i) * 128] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
            }
          }
          sync_some(9, 256 * kSlots);
          if (tid == 0) {
            unsigned n;
            asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(n) : "l"(counter) : "memory");
            notes.flag = n + 1u == static_cast<unsigned>(parts);
            if (notes.flag) *counter = 0u;
          }
          sync_some(9, 256 * kSlots);
          mine = *static_cast<volatile int*>(&notes.flag) != 0;
        }
        if (mine) {
          auto ml_at = [&](int x) {
            return here && x == part ? make_float2(m, l) : __ldcg(P.part_ml + static_cast<long long>(part_slot(x)) * S::kRows + tile * 128 + row);
          };
          constexpr int kKept = 4;                            // factors of so many parts are kept
          float mm = -INFINITY, ll = 0.0f, kept[kKept] = {};
          for (int x = 0; x < parts && live; ++x) mm = fmaxf(mm, ml_at(x).x);
          auto factor = [&](float v) { return v == -INFINITY ? 0.0f : ex2_approx(v - mm); };
          for (int x = 0; x < parts && live; ++x) {
            const float2 v = ml_at(x);
            const float f = factor(v.x);
            ll += v.x == -INFINITY ? (v.y != v.y ? v.y : 0.0f) : v.y * f;
#pragma unroll
            for (int i = 0; i < kKept; ++i)
              if (i == x) kept[i] = f;
          }
          const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
          uint16_t* dst = static_cast<uint16_t*>(P.out) + (w.r.q0 + token) * P.o_tok + head * P.o_head + my_first;
          if (live && speaks && P.lse) P.lse[static_cast<long long>(w.r.q0 + token) * P.hq + head] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * kLn2;
          for (int d = 0; d < my_columns; d += 16) {          // a multiple of 8: the last 8 may be none
            const bool both = d + 8 < my_columns;
            float acc[16] = {};
            auto fetch = [&](int x, uint4 (&v)[4]) {
              if (here && x == part) {
                uint32_t o[2][8] = {};
                if (any) {
                  tc::load8(o[0], my_at + d);
                  if (both) tc::load8(o[1], my_at + d + 8);
                  tc::load_wait();
                  tc::pin8(o[0]);
                  tc::pin8(o[1]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = make_uint4(o[i / 2][i % 2 * 4], o[i / 2][i % 2 * 4 + 1], o[i / 2][i % 2 * 4 + 2], o[i / 2][i % 2 * 4 + 3]);
              } else {
                const uint4* src = part_at(part_slot(x), tile) + (my_first + d) / 4 * 128 + row;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (i < 2 || both) v[i] = __ldcg(src + i * 128);
              }
            };
            auto add = [&](float f, const uint4 (&v)[4]) {    // a sum of nothing was not written: its factor is 0
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t o[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[4 * i + e] = f == 0.0f ? acc[4 * i + e] : fmaf(f, __uint_as_float(o[e]), acc[4 * i + e]);
              }
            };
            auto two_parts = [&](int x, float f, float g) {   // with their loads in flight together
              uint4 v[4] = {}, u[4] = {};
              fetch(x, v);
              if (x + 1 < parts) fetch(x + 1, u);
              add(f, v);
              if (x + 1 < parts) add(g, u);
            };
#pragma unroll
            for (int x = 0; x < kKept; x += 2)
              if (x < parts) two_parts(x, kept[x], kept[x + 1]);
#pragma unroll 1
            for (int x = kKept; x < parts; x += 2) {
              const float2 v = ml_at(x), u = ml_at(min(x + 1, parts - 1));
              two_parts(x, live ? factor(v.x) : 0.0f, live ? factor(u.x) : 0.0f);
            }
            if (live) {
              uint32_t h[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) h[i] = pack2<DT>(acc[2 * i] * inv, acc[2 * i + 1] * inv);
              *reinterpret_cast<uint4*>(dst + d) = make_uint4(h[0], h[1], h[2], h[3]);
              if (both) *reinterpret_cast<uint4*>(dst + d + 8) = make_uint4(h[4], h[5], h[6], h[7]);
            }
          }
        }
        tc::fence_before();
        sync_some(9, 256 * kSlots);                           // the flag and the part's room are free again
      }
      if (two_sums && !joined) sync_some(9, 512);             // and the first slot's sum, which four warps read
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= kLoaders && warp < kLoaders + kLoadWarps) {
    // ================================================ keys and values to the ring
    const int wl = warp - kLoaders;
    unsigned n = 0, raws = 0, tiles = 0;                      // loads; e4m3: those announced as they are cached; key tiles so far
    bool ok = true;
    auto free_slot = [&]() { return wait(&s_bars.kv_empty[n % kRing], ((n / kRing) & 1) ^ 1); };

    while (ok && w.next(P, notes.share)) {
      if (w.jb >= w.je) continue;
      const bool shared = kSlots == 2 && !w.few;
      const int* pages = C.indices + w.r.first;
      const int len = w.r.len, head = w.head, je = w.je;
      auto nth_page = [&](int key) { return P.page_shift >= 0 ? key >> P.page_shift : key / C.page_size; };
      const int ahead = shared ? 1 : 2, loads = 2 * (je - w.jb);
      // the loads in order: K jb .. (ahead of them), then V j, K j + ahead
      int jk = w.jb, jv = w.jb;
      auto turn = [&](bool* is_v) {
        *is_v = jk >= je || jk - jv >= ahead;
        return *is_v ? jv : jk;
      };
      // Rows by threads' copies, 16 at a time: groups wl, wl + 3, wl + 6 of a tile.  Lanes find
      // the rows' places, of two groups at once; past the length there are none, and zeros are
      // written.
      constexpr int kGroups = kKeys / 16;
      struct Places { unsigned off[2]; unsigned live[2]; };
      auto page_of = [&](int j, int x) -> int {
        const int g = wl + kLoadWarps * (2 * x + (lane >> 4)), key = j * kKeys + g * 16 + (lane & 15);
        return g < kGroups && j < je && key < len ? min(max(pages[nth_page(key)], 0), C.num_pages - 1) : -1;
      };
      auto place = [&](int j, const int (&page)[2], const kv::Side16& side) {
        Places p;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int key = j * kKeys + (wl + kLoadWarps * (2 * x + (lane >> 4))) * 16 + (lane & 15);
          p.off[x] = page[x] < 0 ? 0 : page[x] * side.page + static_cast<unsigned>(key - nth_page(key) * C.page_size) * side.slot + head * side.head;
          p.live[x] = __ballot_sync(0xFFFFFFFFu, page[x] >= 0);
        }
        return p;
      };
      constexpr int kChunks = D * (E4M3 ? 1 : 2) / 16, kEach = 16 * kChunks / 32;   // 16-byte chunks of a row; of a lane and group
      auto copy_rows = [&](const Places& p, const kv::Side16& side, auto to) {
#pragma unroll
        for (int gi = 0; gi < (kGroups + kLoadWarps - 1) / kLoadWarps; ++gi) {
          const int g = wl + kLoadWarps * gi;
          if (g >= kGroups) break;
          unsigned o[kEach];
#pragma unroll
          for (int x = 0; x < kEach; ++x) o[x] = __shfl_sync(0xFFFFFFFFu, p.off[gi >> 1], (gi & 1) * 16 + (x * 32 + lane) / kChunks);
#pragma unroll
          for (int x = 0; x < kEach; ++x) {
            const int c = x * 32 + lane, r = c / kChunks, col = c % kChunks;
            const bool there = (p.live[gi >> 1] >> ((gi & 1) * 16 + r)) & 1u;
            cp16(to(g * 16 + r, col), side.base + (there ? o[x] + col : 0u) * 16ull, there);
          }
        }
      };
      int page_next[2] = {page_of(jk, 0), page_of(jk, 1)};    // of the next keys: an L2 read away
      // Whole tiles come as boxes by a page's slots: of 64 elements each, dealt to the warps, or of
      // whole rows of codes.
      const int in_tile = P.boxes ? max(1, kKeys >> P.page_shift) : 0, slots = kKeys / max(1, in_tile);
      auto soon = [&](int j) {                                // its part of the page list into L1
        if (lane == 0 && P.boxes && j < je && (j + 1) * kKeys <= len)
          asm volatile("prefetch.global.L1 [%0];" ::"l"(pages + ((j * kKeys) >> P.page_shift)));
      };
      auto listed = [&](int j, int nth) { return min(max(pages[((j * kKeys) >> P.page_shift) + nth], 0), C.num_pages - 1); };
      soon(jk);
      if (!E4M3) {
        const int boxes = in_tile * S::kBlocks, mine = (boxes - wl + kLoadWarps - 1) / kLoadWarps;
        for (int i = 0; i < loads; ++i) {
          bool is_v;
          const int j = turn(&is_v);
          const bool boxes_now = P.boxes && (j + 1) * kKeys <= len;
          int page[2] = {page_next[0], page_next[1]};
          if (is_v) {                                         // values' pages were read a while ago: in L1
            ++jv;
            if (!boxes_now) { page[0] = page_of(j, 0); page[1] = page_of(j, 1); }
          } else {
            ++jk;
            soon(jk + 1);
            if (!P.boxes || (jk + 1) * kKeys > len) { page_next[0] = page_of(jk, 0); page_next[1] = page_of(jk, 1); }
          }
          const uint32_t dst = s_ring + (n % kRing) * S::kTile;
          if (boxes_now) {
            ok = free_slot();
            if (!ok) break;
            if (tc::elect()) {
              const uint32_t bar = tc::smem_u32(&s_bars.kv_full[n % kRing]);
              const void* map = is_v ? &P.v_map : &P.k_map;
              const int slot = (j * kKeys) & (C.page_size - 1);
              tc::bar_expect(bar, mine * slots * 128);
#pragma unroll 4
              for (int x = wl; x < boxes; x += kLoadWarps) {
                const int nth = x / S::kBlocks, block = x - nth * S::kBlocks;
                tc::copy_box(dst + block * (kKeys * 128) + nth * slots * 128, map, block * 64, slot, head, listed(j, nth), bar);
              }
            }
            __syncwarp();
            ++n;
            continue;
          }
          const kv::Side16& side = is_v ? P.v : P.k;
          const Places p = place(j, page, side);
          ok = free_slot();
          if (!ok) break;
          copy_rows(p, side, [&](int r, int col) { return dst + (col / 8) * (kKeys * 128) + r * 128 + ((col % 8) ^ (r & 7)) * 16; });
          arrive_copied(&s_bars.kv_full[n % kRing]);
          ++n;
        }
      } else {
        // Codes and scales as they are cached go to a ring of their own, kRaws - 1 tiles ahead, and
        // are converted from there.
        int asked = 0;
        const unsigned n0 = n;
        auto ask = [&]() {
          if (asked < loads) {
            const unsigned place_n = n0 + asked, at_n = place_n % S::kRaws;
            bool is_v;
            const int j = turn(&is_v);
            const bool boxes_now = P.boxes && (j + 1) * kKeys <= len;
            int page[2] = {page_next[0], page_next[1]};
            if (is_v) {
              ++jv;
              if (!boxes_now) { page[0] = page_of(j, 0); page[1] = page_of(j, 1); }
            } else {
              ++jk;
              soon(jk + 1);
              if (!P.boxes || (jk + 1) * kKeys > len) { page_next[0] = page_of(jk, 0); page_next[1] = page_of(jk, 1); }
            }
            ok = ok && wait(&s_bars.raw_empty[at_n], ((place_n / S::kRaws) & 1) ^ 1);
            const kv::Side16& side = is_v ? P.v : P.k;
            const uint32_t dst = s_raw + at_n * S::kRaw, bar = tc::smem_u32(&s_bars.raw_full[at_n]);
            if (!ok) {
            } else if (!boxes_now) {
              copy_rows(place(j, page, side), side, [&](int r, int col) { return dst + r * D + col * 16; });
              if (!is_v) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                  const int g = wl + kLoadWarps * (2 * x + (lane >> 4));
                  if (g >= kGroups) continue;
                  const int key = j * kKeys + g * 16 + (lane & 15);
                  const long long at = page[x] < 0 ? 0 : (static_cast<long long>(page[x]) * C.heads + head) * C.page_size + key - nth_page(key) * C.page_size;
                  const uint32_t to = dst + kKeys * D + (g * 16 + (lane & 15)) * 4;
                  cp4(to, P.k.scale + at, page[x] >= 0);
                  cp4(to + kKeys * 4, P.v.scale + at, page[x] >= 0);
                }
              }
              arrive_copied(&s_bars.raw_full[at_n]);
            } else if (wl == 0) {                             // the first warp asks for the codes,
              if (tc::elect()) {
                const void* map = is_v ? &P.v_map : &P.k_map;
                tc::bar_expect(bar, kKeys * D);
#pragma unroll 4
                for (int nth = 0; nth < in_tile; ++nth)
                  tc::copy_box(dst + nth * slots * D, map, 0, (j * kKeys) & (C.page_size - 1), head, listed(j, nth), bar);
              }
              __syncwarp();
            } else if (wl == 1 || is_v) {
              if (lane == 0) tc::bar_arrive(bar);
            } else {                                          // the last for the scales, four neighbours a copy
#pragma unroll
              for (int x = 0; x < kKeys / 64; ++x) {
                const int c = x * 32 + lane, of = c / (kKeys / 4), at = c % (kKeys / 4) * 4, key = j * kKeys + at;
                const long long from = (static_cast<long long>(listed(j, at >> P.page_shift)) * C.heads + head) * C.page_size + (key & (C.page_size - 1));
                cp16(dst + kKeys * D + c * 16, (of ? P.v.scale : P.k.scale) + from, true);
              }
              arrive_copied(&s_bars.raw_full[at_n]);
            }
            if (ok) raws = place_n + 1;
          }
          ++asked;
        };
        int kk = w.jb, vv = w.jb;                             // the same order again, for what is converted
#pragma unroll
        for (int x = 0; x < S::kRaws - 1; ++x) ask();
        for (int i = 0; i < loads; ++i) {
          const bool is_v = kk >= je || kk - vv >= ahead;
          if (is_v) ++vv; else ++kk;
          ask();
          ok = ok && wait(&s_bars.raw_full[n % S::kRaws], (n / S::kRaws) & 1) && free_slot();
          if (!ok) break;
          const uint32_t dst = s_ring + (n % kRing) * S::kTile;
          const unsigned char* raw = base_p + (s_raw - base) + (n % S::kRaws) * S::kRaw;
#pragma unroll
          for (int gi = 0; gi < (kGroups + kLoadWarps - 1) / kLoadWarps; ++gi) {
            const int g = wl + kLoadWarps * gi;
            if (g >= kGroups) break;
            uint4 codes[kEach];
#pragma unroll
            for (int x = 0; x < kEach; ++x) {
              const int c = x * 32 + lane;
              codes[x] = *reinterpret_cast<const uint4*>(raw + (g * 16 + c / kChunks) * D + c % kChunks * 16);
            }
#pragma unroll
            for (int x = 0; x < kEach; ++x) {
              const int c = x * 32 + lane, r = g * 16 + c / kChunks, col = c % kChunks;
              const uint4 v = codes[x];
              uint32_t h[8];
              e4m3x4(v.x, h[0], h[1]);
              e4m3x4(v.y, h[2], h[3]);
              e4m3x4(v.z, h[4], h[5]);
              e4m3x4(v.w, h[6], h[7]);
              const uint32_t at = dst + (col / 4) * (kKeys * 128) + r * 128;
              const int c0 = (col % 4) * 2;
              st16(at + (c0 ^ (r & 7)) * 16, h[0], h[1], h[2], h[3]);
              st16(at + ((c0 + 1) ^ (r & 7)) * 16, h[4], h[5], h[6], h[7]);
            }
          }
          if (!is_v) {
            float* sc = reinterpret_cast<float*>(base_p + (s_scales - base) + (tiles % S::kScaleRing) * S::kScales);
            const float* cached = reinterpret_cast<const float*>(raw + kKeys * D);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int g = wl + kLoadWarps * (2 * x + (lane >> 4)), r = g * 16 + (lane & 15);
              if (g >= kGroups) continue;
              sc[r] = cached[r];
              sc[kKeys + r] = max_nan(cached[kKeys + r], 8e-28f);   // 2^-90
            }
            ++tiles;
          }
          tc::fence_smem();
          __syncwarp();
          if (lane == 0) {
            tc::bar_arrive(tc::smem_u32(&s_bars.kv_full[n % kRing]));
            tc::bar_arrive(tc::smem_u32(&s_bars.raw_empty[n % S::kRaws]));
          }
          ++n;
        }
      }
    }
    if (lane == 0) notes.brought[wl] = E4M3 ? raws : n;
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == kIssuer) {
    // ================================================================ products
    // One thread does all of it: what a product waits for is looked at in a few instructions.
    if (tc::elect()) {
      struct Place {                                          // in the ring
        int slot;
        uint32_t parity;
        __device__ __forceinline__ Place after() const { return slot + 1 == kRing ? Place{0, parity ^ 1} : Place{slot + 1, parity}; }
      };
      Place n = {0, 0};                                       // the next load to take
      unsigned products = 0;                                  // O += P V
      uint32_t q_phase = 0, p_phase = 0;                      // a bit a buffer
      bool ok = true;
      constexpr uint32_t score = tc::product(HT == ECAH_DTYPE_BF16, kKeys, false), sum = tc::product(HT == ECAH_DTYPE_BF16, D, true);
      const uint64_t q_desc = tc::tile_desc(s_q, 0), k_desc = tc::tile_desc(s_ring, 0), v_desc = tc::tile_desc(s_ring, kKeys * 128);
      auto await = [&](unsigned long long* b, uint32_t parity) -> bool {
        const uint32_t bar = tc::smem_u32(b);
        for (int i = 0; i < P.tries; ++i) {
          if (tc::bar_test(bar, parity)) {
            tc::fence_after();
            if (!E4M3) tc::fence_smem();                      // threads' copies are not fenced where they are made
            return true;
          }
          if (*static_cast<volatile int*>(&notes.failed)) break;
        }
        *static_cast<volatile int*>(&notes.failed) = 1;
        return false;
      };
      auto scores = [&](int buf, int q_tile, Place at) {
        const uint64_t a = q_desc + q_tile * (S::kQ >> 4), b = k_desc + at.slot * (S::kTile >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc::mma(tmem + buf * S::kBuffer, a + (k / 4) * (128 * 128 >> 4) + (k % 4) * 2, b + (k / 4) * (kKeys * 128 >> 4) + (k % 4) * 2, score, k > 0);
        tc::commit(tc::smem_u32(&s_bars.s_full[buf]));
      };
      auto weigh = [&](int slot, int buf, Place at, bool add) {
        const uint64_t b = v_desc + at.slot * (S::kTile >> 4);
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          tc::mma_ts(tmem + S::kSum + slot * D, tmem + buf * S::kBuffer + k * 8, b + k * (2048 >> 4), sum, add || k > 0);
        tc::commit(tc::smem_u32(&s_bars.pv_done[kSlots == 2 ? slot : products & 1]));
        ++products;
      };
      auto release = [&](Place at) { tc::commit(tc::smem_u32(&s_bars.kv_empty[at.slot])); };
      auto arrived = [&](Place at) { return await(&s_bars.kv_full[at.slot], at.parity); };
      auto weights = [&](int buf) {
        const bool there = await(&s_bars.p_full[buf], p_phase >> buf & 1);
        p_phase ^= 1u << buf;
        return there;
      };
      while (ok && w.advance(P, notes.share)) {
        const int count = w.je - w.jb, first = w.je0 - w.jb;  // first: tiles of the first half
        if (count <= 0) continue;
        const bool few = w.few;
        if (!(ok = await(&s_bars.q_full, q_phase))) break;
        q_phase ^= 1;
        if (kSlots == 2 && !few) {
          if (!(ok = arrived(n))) break;
          if (first > 0) scores(0, 0, n);
          scores(1, 1, n);
          release(n);
          n = n.after();
          for (int x = 0; x < count && ok; ++x) {             // load n: V x; the one after: K x + 1
            const bool again = x + 1 < count;
            const Place next = n.after();
            if (!(ok = arrived(n))) break;
            if (again && !(ok = arrived(next))) break;
            if (x < first) {
              if (!(ok = weights(0))) break;
              weigh(0, 0, n, x > 0);
              if (x + 1 < first) scores(0, 0, next);
            }
            if (!(ok = weights(1))) break;
            weigh(1, 1, n, x > 0);
            release(n);
            if (again) {
              scores(1, 1, next);
              release(next);
            }
            n = again ? next.after() : next;
          }
        } else {
          const int lead = min(2, count);
          for (int x = 0; x < lead && ok; ++x) {
            if (!(ok = arrived(n))) break;
            scores(x, 0, n);
            release(n);
            n = n.after();
          }
          for (int x = 0; x < count && ok; ++x) {             // load n: V x; the one after: K x + 2
            if (!(ok = arrived(n)) || !(ok = weights(x & 1))) break;
            weigh(kSlots == 2 ? x & 1 : 0, x & 1, n, x >= kSlots);
            release(n);
            n = n.after();
            if (x + 2 < count) {
              if (!(ok = arrived(n))) break;
              scores(x & 1, 0, n);
              release(n);
              n = n.after();
            }
          }
        }
        if (ok) tc::commit(tc::smem_u32(&s_bars.q_empty));
      }
      // nothing is in flight when the tensor memory is given back
      tc::commit(tc::smem_u32(&s_bars.done));
      for (int i = 0; i < kTries && !tc::bar_test(tc::smem_u32(&s_bars.done), 0); ++i) {}
    }
    __syncwarp();
  }

  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == kIssuer) tc::tmem_free(tmem, S::kColumns);
  // Where a wait ran out the copy engine may still be bringing tiles that nobody waited for: they
  // land before the block ends and its shared memory is another's.  A loader that stopped first
  // owes the tiles that another announced its arrival (one on a barrier at the most, since a place
  // is used again only after all have arrived); nobody else looks at the barriers any more.
  if (notes.failed && warp >= kLoaders && warp < kLoaders + kLoadWarps) {
    constexpr unsigned ring = E4M3 ? S::kRaws : kRing;
    unsigned long long* full = E4M3 ? s_bars.raw_full : s_bars.kv_full;
    unsigned all = 0;
    for (int i = 0; i < kLoadWarps; ++i) all = max(all, notes.brought[i]);
    for (unsigned x = notes.brought[warp - kLoaders]; x < all && lane == 0; ++x) tc::bar_arrive(tc::smem_u32(&full[x % ring]));
    for (unsigned x = all - min(all, ring); x < all; ++x)
      for (int i = 0; i < kTries && !tc::bar_test(tc::smem_u32(&full[x % ring]), x / ring & 1); ++i) {}
  }
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
  const bool e4m3 = c.kv_dtype == ECAH_KV_E4M3;
  const cuuint64_t size = e4m3 ? 1 : 2, row = static_cast<cuuint64_t>(c.head_dim) * size;
  const cuuint64_t sizes[4] = {static_cast<cuuint64_t>(c.head_dim), static_cast<cuuint64_t>(c.page_size), static_cast<cuuint64_t>(c.num_kv_heads),
                               static_cast<cuuint64_t>(c.num_pages)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(s.slot) * size, static_cast<cuuint64_t>(s.head) * size, static_cast<cuuint64_t>(s.page) * size};
  for (int i = 0; i < 3; ++i) {
    if (sizes[i + 1] == 1) strides[i] = row;                  // of a dimension of one the stride may be anything
    if (strides[i] == 0 || strides[i] >= 1ull << 40) return false;
  }
  // 16-bit rows into swizzled blocks of 64 elements; rows of codes as they are
  const cuuint32_t box[4] = {e4m3 ? static_cast<cuuint32_t>(c.head_dim) : 64u, static_cast<cuuint32_t>(slots), 1, 1}, steps[4] = {1, 1, 1, 1};
  return encode(map, e4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : c.kv_dtype == ECAH_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, s.base, sizes, strides,
                box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, e4m3 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
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
  // units of work are counted in 32 bits
  const int keys = c.head_dim <= 128 ? 128 : 64, item = c.head_dim <= 128 ? 256 : 128;
  const double items = (static_cast<double>(a->tokens) * group / item + c.batch) * c.num_kv_heads;
  if (items * (prefill::kItemCost + prefill::kCost * (static_cast<double>(c.num_indices) * c.page_size / keys + 2.0)) >= 2147483648.0)
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
  // swizzle goes by 8 rows); smaller or odd pages go through threads (8192 tokens in short
  // runs: by the engine with pages of 8 and 16 tokens 538 and 490 us, by threads with pages of
  // 4, 12 and 24 tokens 678, 792 and 793 us).
  P.boxes = P.page_shift >= 3 && (!e4m3 || (aligned16(c.k_scale) && aligned16(c.v_scale))) && prefill::box_map(&P.k_map, P.cache.k, c, std::min(c.page_size, keys)) &&
            prefill::box_map(&P.v_map, P.cache.v, c, std::min(c.page_size, keys));
  return launch_kernel(v.fn, dim3(sms), prefill::kT, v.smem, reinterpret_cast<cudaStream_t>(stream), P) ? ECAH_OK : ECAH_ERR_LAUNCH;
}

}  // extern "C"
