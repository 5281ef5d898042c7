// The pieces of sm_100a's matrix path that the softmax kernels use: mbarriers with a longer bounded wait
// than w2v_device.cuh has, TMA tile loads, shared-memory descriptors, tcgen05 products and tensor-memory loads.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "w2v_device.cuh"

namespace w2v {

// One lane of a converged warp.  Code behind it is known to run in one thread, which keeps what the
// tensor and copy instructions take as uniform operands out of vector registers; `lane == 0` does not.
__device__ __forceinline__ bool elected() {
  uint32_t yes;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(yes));
  return yes != 0;
}

// Two CTAs of a cluster work as a pair on one tile; the one of rank 0 issues their products.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Address, in the cluster's window, of the same place in the shared memory of rank 0.
__device__ __forceinline__ uint32_t in_leader(const void *p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_addr(p)));
  return a;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrives on a barrier of the other CTA.  What it tells is that tensor memory has been read, which the
// tcgen05 fences order; a release at cluster scope would wait for the thread's stores to memory too.
__device__ __forceinline__ void mbar_arrive_leader(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Waits for the phase of `parity` to complete.  False when it did not within about two seconds or
// when another role of the block has given up already (`gave_up`, in shared memory).
__device__ __forceinline__ bool mbar_wait(u64 *bar, unsigned parity, volatile int *gave_up) {
  if (mbar_try_wait(bar, parity)) return true;
  uint64_t begin, now;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(begin));
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 256; i++)
      if (mbar_try_wait(bar, parity)) return true;
    if (*gave_up) return false;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (now - begin > 2000000000ull) {
      *gave_up = 1;
      return false;
    }
  }
}

// Into this CTA's shared memory; the bytes are counted on a barrier that may be the other CTA's.
__device__ __forceinline__ void tma_load_2d(void *dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(smem_addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

// Shared-memory operand with 128-byte swizzle.  K-major: 8 rows of 128 bytes are a group, `stride`
// bytes from one group of rows to the next.  MN-major: 64 elements of M or N in 128 bytes, 8 of K a
// group, `stride` bytes from one such group to the next and `leading` bytes to the next 64 of M or N.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t leading, uint32_t stride) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)((leading >> 4) & 0x3FFF) << 16 |
         (uint64_t)((stride >> 4) & 0x3FFF) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// kind::f16 instruction descriptor: fp32 accumulators, both operands bf16 or both fp16.
__host__ __device__ constexpr uint32_t mma_desc(bool bf16, bool a_mn, bool b_mn, int m, int n) {
  return 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (a_mn ? 1u : 0u) << 15 | (b_mn ? 1u : 0u) << 16 |
         (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// Arrives on the barrier, in both CTAs, when the products issued so far are done.
__device__ __forceinline__ void mma_commit(u64 *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_addr(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void tmem_alloc(uint32_t *to, unsigned columns) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(to)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, unsigned columns) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}
__device__ __forceinline__ void tmem_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes of tensor memory: one row a thread.
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&x)[32]) {
  uint32_t *r = reinterpret_cast<uint32_t *>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&x)[16]) {
  uint32_t *r = reinterpret_cast<uint32_t *>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// 2^-22 relative, zero below 2^-126: no more than the logit's own rounding makes of its exponential (a logit of 16
// is rounded by 2^-20), and one instruction where a tile has 65536 of them.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace w2v
