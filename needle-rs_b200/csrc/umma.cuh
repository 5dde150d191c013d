// Tensor-core primitives (mbarriers, tcgen05, tensor memory) shared by the
// kernels that issue tcgen05.mma.
#pragma once
#include <stdint.h>

namespace nb {

constexpr unsigned long long WAIT_NS = 1000000000ull;  // bound of every wait: one second

__device__ __forceinline__ uint32_t su32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(su32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Wait for phase `parity` of `bar`. Gives up after WAIT_NS (raising *werr) or
// as soon as another role of the CTA gave up (`abort`), returning false. Between polls a
// waiter sleeps `backoff_ns` so waiting warps leave the issue slots to the
// warps that decode weights on the same schedulers.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort, int* werr,
                                          unsigned backoff_ns = 0) {
  if (mbar_try(bar, parity)) return true;
  const unsigned long long t0 = now_ns();
  while (true) {
    if (backoff_ns) __nanosleep(backoff_ns);
    if (mbar_try(bar, parity)) return true;
    if (*abort) return false;
    if (now_ns() - t0 > WAIT_NS) {
      *abort = 1;
      atomicExch(werr, 1);
      return false;
    }
  }
}

// mbar_wait for short waits between warps of a block: a bare loop on the
// barrier, which the hardware holds for a while per try (a time hint would put a
// software sleep between two tries), bounded by the SM's clock (about a second),
// whose reading costs a few cycles where the global timer's costs hundreds.
constexpr long long WAIT_CLOCKS = 1ll << 31;
__device__ __forceinline__ bool mbar_wait_spin(uint64_t* bar, uint32_t parity, volatile uint32_t* abort, int* werr) {
  const long long t0 = clock64();
  while (true) {
#pragma unroll 1
    for (int n = 0; n < 64; ++n)
      if (mbar_try(bar, parity)) return true;
    if (*abort) return false;
    if (clock64() - t0 > WAIT_CLOCKS) {
      *abort = 1;
      atomicExch(werr, 1);
      return false;
    }
  }
}

// Drain wait used on the abort path: ignores the abort flag, bounded in time.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
  const unsigned long long t0 = now_ns();
  while (!mbar_try(bar, parity) && now_ns() - t0 <= WAIT_NS) {
  }
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// K-major operand tile, 128-byte swizzle: rows of 128 B, 8-row atoms 1024 B
// apart (stride byte offset), start address in 16-byte units.
__device__ __forceinline__ uint64_t sw128_desc(const void* tile) {
  const uint64_t start = (su32(tile) & 0x3FFFF) >> 4;
  return start | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(su32(bar))
               : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

}  // namespace nb
