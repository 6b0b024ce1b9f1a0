// Barriers and bulk copies of the layer operators' pipelines. Every wait is
// bounded (2 s at 2 GHz): a role that gives up raises the CTA's abort flag, the
// others stop at their next wait, and the CTA waits (bounded) for its own
// copies before it ends.
#pragma once

#include <stdint.h>

namespace exl3 {

constexpr long long kWaitClocks = 4000000000ll;

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void bar_init_fence() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// true when the phase completed; false on timeout (which raises the abort
// flag) or when another role has aborted
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  long long start = 0;
  for (uint32_t it = 1;; ++it) {
    if (bar_try(bar, parity)) return true;
    if ((it & 63u) == 0u) {
      if (*abort_flag) return false;
      const long long now = clock64();
      if (start == 0) start = now;
      if (now - start > kWaitClocks) {
        *abort_flag = 1;
        return false;
      }
    }
  }
}
// the shutdown path's wait: bounded, whatever the abort flag says
__device__ __forceinline__ void bar_drain(uint32_t bar, uint32_t parity) {
  const long long start = clock64();
  while (!bar_try(bar, parity))
    if (clock64() - start > kWaitClocks) return;
}
// global to shared, 16-byte aligned on both sides, a multiple of 16 bytes
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

}  // namespace exl3
