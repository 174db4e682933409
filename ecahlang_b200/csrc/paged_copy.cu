// Copies of cache pages in all layers: ecah_paged_copy (contract in
// include/ecah_sampler.h).

#include <algorithm>

#include "host_util.h"
#include "paged.cuh"

namespace ecah {
namespace copy {

// Nothing is computed.  Bound: HBM, every byte read once and written once.
//
// Split: one launch for up to kLayers layers (their pointers travel in the launch's
// arguments), a block row for each layer's keys, values and scales; the 16-byte
// chunks of all pairs of such a side are dealt to threads in order, kUnroll a thread
// with all loads in flight, so short pages fill blocks too.
//
// Measured on one B200, passes through the Python entry point one after another: 2000
// pages of 16 tokens of 8 heads of 128 in 4 layers (bf16) 162 to 171 us (6.1 to 6.5 TB/s, 94 to
// 99 % of a copy's rate), 127 pages of an e4m3 cache in 7 layers 7.3 (7.1 on the device: the
// lists are read, then the rows, then they are written), a fork's 3 pages in 28 layers 7.2 (2.6
// on the device; the host checks 28 layers).

constexpr int kT = 256;
constexpr int kUnroll = 4;
constexpr int kLayers = 64;

// A page's live bytes: outer runs (slots by heads) of inner 16-byte chunks.  What
// lies behind one another in memory is one run.
struct Side {
  long long page, slot, head;  // strides in chunks
  int heads;                   // runs a slot, 1 where a slot's heads (or a head's slots) are one run
  int run;                     // chunks of a run that do not depend on the tokens
  int slots_in_run;            // a run grows with the tokens
  int whole;                   // chunks of a whole page
};

struct Params {
  void* base[kLayers][4];      // k, v, k_scale, v_scale
  Side side[2];
  const int *src, *dst, *tokens;
  int pairs, num_pages, page_size, heads;
  int sides;                   // of a layer: keys and values, or their scales too
};

__device__ __forceinline__ bool pair_of(const Params& P, int i, int* src, int* dst, int* tokens) {
  *src = P.src[i];
  *dst = P.dst[i];
  *tokens = P.tokens ? min(max(P.tokens[i], 0), P.page_size) : P.page_size;
  return *tokens > 0 && *src >= 0 && *dst >= 0 && *src < P.num_pages && *dst < P.num_pages && *src != *dst;
}

__global__ void __launch_bounds__(kT) copy_kernel(const __grid_constant__ Params P) {
  grid_start();
  const int layer = blockIdx.y / P.sides, which = blockIdx.y - layer * P.sides;
  const unsigned first = blockIdx.x * (kT * kUnroll) + threadIdx.x;
  if (which < 2) {
    const Side& s = P.side[which];
    uint4* base = static_cast<uint4*>(P.base[layer][which]);
    uint4 v[kUnroll];
    uint4* to[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const unsigned g = first + u * kT, pair = g / s.whole, c = g - pair * s.whole;
      to[u] = nullptr;
      int src, dst, tokens;
      if (pair >= static_cast<unsigned>(P.pairs) || !pair_of(P, pair, &src, &dst, &tokens)) continue;
      const unsigned run = s.slots_in_run ? s.run * tokens : s.run, runs = s.slots_in_run ? s.heads : s.heads * tokens;
      unsigned o = 0, i = c;
      if (c >= run) {                        // not the first run
        if (runs <= 1) continue;
        o = c / run;
        i = c - o * run;
        if (o >= runs) continue;
      }
      const unsigned slot = s.slots_in_run ? 0 : o / s.heads, head = s.slots_in_run ? o : o - slot * s.heads;
      const long long at = slot * s.slot + head * s.head + i;
      v[u] = __ldcs(base + src * s.page + at);
      to[u] = base + dst * s.page + at;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (to[u]) __stcs(to[u], v[u]);
  } else {
    float* base = static_cast<float*>(P.base[layer][which]);
    const unsigned whole = P.heads * P.page_size;
    float v[kUnroll];
    float* to[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const unsigned g = first + u * kT, pair = g / whole, c = g - pair * whole;
      to[u] = nullptr;
      int src, dst, tokens;
      if (pair >= static_cast<unsigned>(P.pairs) || !pair_of(P, pair, &src, &dst, &tokens) || c % P.page_size >= static_cast<unsigned>(tokens)) continue;
      v[u] = base[static_cast<long long>(src) * whole + c];
      to[u] = base + static_cast<long long>(dst) * whole + c;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (to[u]) *to[u] = v[u];
  }
}

static Side side_of(long long page, long long slot, long long head, int slots, int heads, int row) {
  Side s = {};
  s.page = page; s.slot = slot; s.head = head;
  s.whole = slots * heads * row;
  const bool heads_run = heads == 1 || head == row;                        // a slot's heads are one run
  const bool slots_follow = slots == 1 || slot == static_cast<long long>(row) * (heads_run ? heads : 1);
  s.heads = heads_run ? 1 : heads;
  s.run = heads_run ? heads * row : row;
  s.slots_in_run = slots_follow;
  return s;
}

}  // namespace copy
}  // namespace ecah

using namespace ecah;

extern "C" int ecah_paged_copy(const ecah_copy_args* a, void* stream) {
  if (!a) return ECAH_ERR_NULL;
  if (a->abi_version != ECAH_SAMPLER_ABI_VERSION) return ECAH_ERR_ABI;
  const bool e4m3 = a->kv_dtype == ECAH_KV_E4M3;
  if (!e4m3 && a->kv_dtype != ECAH_DTYPE_F16 && a->kv_dtype != ECAH_DTYPE_BF16) return ECAH_ERR_DTYPE;
  if (a->num_pages < 0 || a->page_size < 1 || a->num_kv_heads < 1 || !kv::head_dim_ok(a->head_dim) || a->layers < 0 || a->pairs < 0)
    return ECAH_ERR_SHAPE;
  const long long unit = e4m3 ? 16 : 8;
  for (long long s : {a->k_page_stride, a->k_slot_stride, a->k_head_stride, a->v_page_stride, a->v_slot_stride, a->v_head_stride})
    if (s < 0 || s % unit) return ECAH_ERR_SHAPE;
  if (a->layers == 0 || a->pairs == 0 || a->num_pages == 0) return ECAH_OK;
  if (!a->k_caches || !a->v_caches || !a->src || !a->dst) return ECAH_ERR_NULL;
  if (e4m3 && (!a->k_scales || !a->v_scales)) return ECAH_ERR_NULL;
  for (int i = 0; i < a->layers; ++i) {
    if (!a->k_caches[i] || !a->v_caches[i] || (e4m3 && (!a->k_scales[i] || !a->v_scales[i]))) return ECAH_ERR_NULL;
    if (!aligned16(a->k_caches[i]) || !aligned16(a->v_caches[i])) return ECAH_ERR_SHAPE;
  }
  const int row = static_cast<int>(a->head_dim / unit);
  const double whole = static_cast<double>(a->page_size) * a->num_kv_heads * row;
  const double chunks = whole * a->pairs;
  // chunks of a side are counted in 32 bits (64 GB of a layer's keys in one call)
  if (whole >= 2147483648.0 || chunks >= 4294967296.0 - copy::kT * copy::kUnroll) return ECAH_ERR_SHAPE;
  copy::Params P;
  P.side[0] = copy::side_of(a->k_page_stride / unit, a->k_slot_stride / unit, a->k_head_stride / unit, a->page_size, a->num_kv_heads, row);
  P.side[1] = copy::side_of(a->v_page_stride / unit, a->v_slot_stride / unit, a->v_head_stride / unit, a->page_size, a->num_kv_heads, row);
  P.src = a->src; P.dst = a->dst; P.tokens = a->tokens;
  P.pairs = a->pairs; P.num_pages = a->num_pages; P.page_size = a->page_size; P.heads = a->num_kv_heads;
  P.sides = e4m3 ? 4 : 2;
  const long long per = copy::kT * copy::kUnroll;
  const unsigned blocks = static_cast<unsigned>((static_cast<long long>(P.side[0].whole) * a->pairs + per - 1) / per);
  for (int at = 0; at < a->layers; at += copy::kLayers) {
    const int n = std::min(a->layers - at, copy::kLayers);
    for (int i = 0; i < n; ++i) {
      P.base[i][0] = a->k_caches[at + i];
      P.base[i][1] = a->v_caches[at + i];
      P.base[i][2] = e4m3 ? a->k_scales[at + i] : nullptr;
      P.base[i][3] = e4m3 ? a->v_scales[at + i] : nullptr;
    }
    if (!launch_kernel(copy::copy_kernel, dim3(blocks, P.sides * n), copy::kT, 0, reinterpret_cast<cudaStream_t>(stream), P)) return ECAH_ERR_LAUNCH;
  }
  return ECAH_OK;
}
