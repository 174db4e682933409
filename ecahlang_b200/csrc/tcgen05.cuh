// Fifth-generation tensor-core instructions (tcgen05), tensor memory and mbarriers
// as inline PTX.
#pragma once

#include <cstdint>

namespace ecah {
namespace tc {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// ---------------------------------------------------------------- mbarriers
__device__ __forceinline__ void bar_init(uint32_t bar, int arrivals) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// One look at a phase; it may itself wait a while.
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// An arrival that announces bytes to come by the copy engine.
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// A box of a tensor to shared memory by the copy engine, counted by a barrier.
__device__ __forceinline__ void copy_box(uint32_t dst, const void* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}
// Orders this thread's ordinary accesses to shared memory before the tensor cores'.
__device__ __forceinline__ void fence_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ------------------------------------------------------------ tensor memory
__device__ __forceinline__ void tmem_alloc(uint32_t dst, int columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t at, int columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

#define ECAH_R8(r, o) "+r"((r)[o]), "+r"((r)[o + 1]), "+r"((r)[o + 2]), "+r"((r)[o + 3]), "+r"((r)[o + 4]), "+r"((r)[o + 5]), "+r"((r)[o + 6]), "+r"((r)[o + 7])
#define ECAH_W8(r, o) "=r"((r)[o]), "=r"((r)[o + 1]), "=r"((r)[o + 2]), "=r"((r)[o + 3]), "=r"((r)[o + 4]), "=r"((r)[o + 5]), "=r"((r)[o + 6]), "=r"((r)[o + 7])
#define ECAH_I8(r, o) "r"((r)[o]), "r"((r)[o + 1]), "r"((r)[o + 2]), "r"((r)[o + 3]), "r"((r)[o + 4]), "r"((r)[o + 5]), "r"((r)[o + 6]), "r"((r)[o + 7])

// 32 columns of this thread's lane; the values are there after load_wait.
__device__ __forceinline__ void load32(uint32_t (&r)[32], uint32_t at) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : ECAH_W8(r, 0), ECAH_W8(r, 8), ECAH_W8(r, 16), ECAH_W8(r, 24) : "r"(at));
}
__device__ __forceinline__ void load16(uint32_t (&r)[16], uint32_t at) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : ECAH_W8(r, 0), ECAH_W8(r, 8) : "r"(at));
}
__device__ __forceinline__ void load8(uint32_t (&r)[8], uint32_t at) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : ECAH_W8(r, 0) : "r"(at));
}
__device__ __forceinline__ void load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Nothing that uses the values is moved before this.
__device__ __forceinline__ void pin32(uint32_t (&r)[32]) {
  asm volatile("" : ECAH_R8(r, 0), ECAH_R8(r, 8), ECAH_R8(r, 16), ECAH_R8(r, 24));
}
__device__ __forceinline__ void pin8(uint32_t (&r)[8]) { asm volatile("" : ECAH_R8(r, 0)); }
__device__ __forceinline__ void store8(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), ECAH_I8(r, 0) : "memory");
}
__device__ __forceinline__ void pin16(uint32_t (&r)[16]) { asm volatile("" : ECAH_R8(r, 0), ECAH_R8(r, 8)); }
__device__ __forceinline__ void store16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
               "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(at), ECAH_I8(r, 0), ECAH_I8(r, 8) : "memory");
}
__device__ __forceinline__ void store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// --------------------------------------------------- pairs of float32 values
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void apart(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// ----------------------------------------------------------------- products
// A tile in shared memory in rows of 128 bytes whose 16-byte chunks are swizzled by
// the row's place among 8.  `lead`: bytes between neighbouring blocks of 64 elements
// where the rows are the summed dimension (else unused); groups of 8 rows follow
// one another.
__device__ __forceinline__ uint64_t tile_desc(uint32_t at, uint32_t lead) {
  return static_cast<uint64_t>((at & 0x3FFFFu) >> 4) | static_cast<uint64_t>(lead >> 4) << 16 | static_cast<uint64_t>(1024 >> 4) << 32 |
         1ull << 46 | 2ull << 61;
}
// One thread of the warp, the same for all its calls.  The instructions below take their
// operands from the warp's uniform registers: behind this choice the compiler needs no
// loop over the active threads to bring them there, as behind `lane == 0`.
__device__ __forceinline__ bool elect() {
  uint32_t one;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xFFFFFFFF; selp.u32 %0, 1, 0, p; }" : "=r"(one));
  return one != 0;
}
// 128 x n results in float32 of 16-bit operands; rows_summed: B's rows are the summed dimension.
constexpr uint32_t product(bool bf16, int n, bool rows_summed) {
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (rows_summed ? 1u << 16 : 0u) | static_cast<uint32_t>(n >> 3) << 17 | 8u << 24;
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t what, bool add) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
               ::"r"(d), "l"(a), "l"(b), "r"(what), "r"(static_cast<uint32_t>(add)) : "memory");
}
// A in tensor memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t what, bool add) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }"
               ::"r"(d), "r"(a), "l"(b), "r"(what), "r"(static_cast<uint32_t>(add)) : "memory");
}
// The barrier gets an arrival when all products that this thread issued are done.
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

}  // namespace tc
}  // namespace ecah
