// PTX wrappers of the fifth-generation tensor cores, tensor memory, barriers
// and tensor copies (sm_100a), as the orthogonalisation kernels use them: one block (cta_group::1),
// f16 operands in shared memory with 128-byte swizzle, 32-bit accumulators.
//
// Every wait on a barrier gives up after `limit` cycles: it then sets the block's
// `dead` word, on which every other wait of the block gives up too.
#pragma once
#include <cuda.h>

#include <cstdint>

namespace blitz {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
// by the lane of a whole warp that has `on`
__device__ __forceinline__ void mbar_arrive(uint32_t on, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.u32 e, %1, 0;\n @e mbarrier.arrive.shared::cta.b64 _, [%0];\n}" ::"r"(bar), "r"(on)
      : "memory");
}
// 1 in one lane of a whole warp, always the same one
__device__ __forceinline__ uint32_t elected() {
  uint32_t on;
  asm volatile("{\n .reg .pred e;\n .reg .b32 r;\n elect.sync r|e, 0xffffffff;\n selp.b32 %0, 1, 0, e;\n}" : "=r"(on));
  return on;
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.b32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// false: gave up (or another thread of the block has).  The limit is in cycles of this SM's clock:
// the global timer takes about a microsecond to read, and most waits are shorter.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* dead, long long limit) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try(bar, parity)) {
    if (*dead) return false;
    if (clock64() - t0 > limit) {
      *dead = 1;
      return false;
    }
  }
  return true;
}
// The same answer for every lane of a whole warp: a wait can end for one lane in the moment
// in which another gives up, and lanes that go different ways from there would wait for each
// other for ever, one part at the warp's next barrier, the other at the block's.
__device__ __forceinline__ bool whole_warp(bool waited) { return __all_sync(0xffffffffu, waited); }

// by the lane of a whole warp that has `on`, as the products below
__device__ __forceinline__ void tma_load(uint32_t on, uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.u32 e, %6, 0;\n"
      " @e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];\n}" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar), "r"(on)
      : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t on, uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.u32 e, %2, 0;\n"
      " @e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}" ::"r"(bar),
      "r"(bytes), "r"(on)
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// clusters: the address of a peer's shared memory, stores, arrivals and waits across it
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// this block's shared memory to a peer's; bar: the peer's
__device__ __forceinline__ void peer_copy(uint32_t on, uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.u32 e, %4, 0;\n"
      " @e cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n}" ::"r"(dst),
      "r"(src), "r"(bytes), "r"(bar), "r"(on)
      : "memory");
}
__device__ __forceinline__ void peer_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.b32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile int* dead, long long limit) {
  if (mbar_try_cluster(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_cluster(bar, parity)) {
    if (*dead) return false;
    if (clock64() - t0 > limit) {
      *dead = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Shared-memory matrix descriptors, 128-byte swizzle, 1024 bytes from one group of 8 rows to
// the next: the lower word holds the address and the leading stride (both in units of 16
// bytes), the upper one never changes.
__device__ __forceinline__ uint32_t smem_desc(uint32_t addr, uint32_t leading) {
  return ((addr >> 4) & 0x3fff) | (leading >> 4) << 16;
}
constexpr uint32_t kDescUpper = (1024u >> 4) | 1u << 14 | 2u << 29;
// f16 x f16 -> f32, 128 rows; b_mn: B lies in memory with n contiguous
__device__ __forceinline__ uint32_t instruction_desc(int bn, bool b_mn) {
  return 1u << 4 | (b_mn ? 1u << 16 : 0u) | (uint32_t)(bn >> 3) << 17 | (128u >> 4) << 24;
}
// One product and one commit (and, above, copies).  The whole warp calls these with the
// same operands and the lane that has `on` issues: where a branch picks the lane instead, the
// compiler cannot see that the operands are the same for the warp and spends 180
// cycles a product on moving them to uniform registers.
__device__ __forceinline__ void mma(uint32_t on, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n .reg .pred p, e;\n .reg .b64 da, db;\n setp.ne.u32 e, %5, 0;\n setp.ne.u32 p, %4, 0;\n"
      " mov.b64 da, {%1, %6};\n mov.b64 db, {%2, %6};\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(on), "n"(kDescUpper)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t on, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.u32 e, %1, 0;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar), "r"(on)
      : "memory");
}
__device__ __forceinline__ void tmem_alloc(uint32_t* where, int columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(where)),
               "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, int columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, float* v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// what this thread wrote is seen by the copies and products issued after the next barrier
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_async_global() { asm volatile("fence.proxy.async.global;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_before_sync() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tcgen05_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

}  // namespace blitz
