// c4s_tc.cuh -- tensor-core building blocks of sm_100a shared by the LM head
// and the linear layer: tcgen05 / TMEM, TMA tile loads and bounded mbarrier
// waits (inline PTX).
#pragma once

#include <cuda.h>

namespace c4s {

__device__ __forceinline__ void tmem_alloc(unsigned* dst, unsigned ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(ncols)
               : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(unsigned taddr, unsigned ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// D (+)= A B^T of one K = 16 step, kind::f16 (both operands bf16, or both fp16, as idesc says).
__device__ __forceinline__ void umma_f16(unsigned tmem_d, unsigned long long adesc, unsigned long long bdesc,
                                         unsigned idesc, unsigned accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_commit(unsigned long long* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y,
                                            unsigned long long* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(smem_u32(dst)),
      "l"(reinterpret_cast<unsigned long long>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
// Shared-memory matrix descriptor of a K-major 128-byte-swizzled tile (rows of
// 64 bf16 = 128 B, 8-row swizzle atoms of 1024 B): start address >> 4 (bits
// 0-13), leading byte offset 16 B (unused by swizzled K-major layouts; field
// 1), stride byte offset 1024 B between 8-row groups (bits 32-45), version 1
// (bits 46-47), layout SWIZZLE_128B (2 at bits 61-63). The tile must be
// 1024-byte aligned; the K = 16 steps inside the 64-wide tile advance the
// start address by 32 B.
__device__ __forceinline__ unsigned long long sw128_desc(const void* tile) {
  const unsigned a = smem_u32(tile);
  return (unsigned long long)((a & 0x3FFFFu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// 32 TMEM lanes x 32 consecutive 32-bit columns into 32 registers per thread
// (thread t of the warp gets lane base + t).
__device__ __forceinline__ void tmem_ld32(unsigned taddr, unsigned (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Bounded wait for an mbarrier phase (about 1 s of wall time).
__device__ __forceinline__ bool mbar_wait_1s(unsigned long long* bar, unsigned parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = globaltimer_ns();
  for (unsigned it = 0; it < (1u << 30); ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 63u && globaltimer_ns() - t0 > 1000000000ull) return false;
  }
  return false;
}

// True in one lane of a converged warp. The loops that feed a pipeline are
// walked by whole warps and issue under this: addresses and descriptors then
// stay in uniform registers. From a branch that only lane 0 takes, a 64-wide
// k-block of copies and products took 640 cycles whatever its bytes; 350 so.
__device__ __forceinline__ bool elect_one() {
  unsigned p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// The same for a whole converged warp that feeds a pipeline, on a
// shared-memory address: a tight loop first, the timer only after many tries.
// Every lane gets the same answer.
__device__ __forceinline__ bool mbar_wait_hot(unsigned bar, unsigned parity) {
  unsigned ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .u32 n;\n\t"
      "mov.u32 n, 0;\n"
      "C4S_TRY:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra C4S_DONE;\n\t"
      "add.u32 n, n, 1;\n\t"
      "setp.lt.u32 p, n, 4096;\n\t"
      "@p bra C4S_TRY;\n"
      "C4S_DONE:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  if (__all_sync(FULL, ok)) return true;
  const unsigned long long t0 = globaltimer_ns();
  for (unsigned it = 0; it < (1u << 30); ++it) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (__all_sync(FULL, ok)) return true;
    if (__any_sync(FULL, (it & 63u) == 63u && globaltimer_ns() - t0 > 1000000000ull)) return false;
  }
  return false;
}
__device__ __forceinline__ void mbar_expect_tx(unsigned bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_tile(unsigned dst, const CUtensorMap* map, int x, int y, unsigned bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(dst),
      "l"(reinterpret_cast<unsigned long long>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

// The same for a whole warp that has nothing else to do: one lane polls, with
// pauses, and leaves the issue slots to the warps that feed the pipeline.
__device__ __forceinline__ bool mbar_wait_warp(unsigned long long* bar, unsigned parity) {
  unsigned ok = 0;
  if ((threadIdx.x & 31) == 0) {
    ok = mbar_try_wait(bar, parity);
    if (!ok) {
      const unsigned long long t0 = globaltimer_ns();
      for (unsigned it = 0; it < (1u << 28) && !ok; ++it) {
        __nanosleep(64);
        ok = mbar_try_wait(bar, parity);
        if ((it & 63u) == 63u && globaltimer_ns() - t0 > 1000000000ull) break;
      }
    }
  }
  ok = __shfl_sync(FULL, ok, 0);
  // every lane passes the barrier itself, for what it orders
  return ok && mbar_wait_1s(bar, parity);
}

}  // namespace c4s
