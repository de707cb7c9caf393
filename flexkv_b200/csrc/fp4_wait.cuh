// Waits between the warps of a CTA: barriers in shared memory, and their limit.
#pragma once

#include <cstdint>

namespace fkv {
namespace {

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t *m, int count) {
  asm volatile("mbarrier.init.shared.b64 [%0], %1;" ::"r"(smem_addr(m)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t *m) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_addr(m)) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t *m, int parity) {
  int ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n selp.b32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_addr(m)), "r"(parity)
      : "memory");
  return ok;
}
// A wait has a limit (a try that fails lasts 4 us, the whole of them a second).
// One that runs out is counted (fkv_fp4_wait_timeouts) and the kernel goes on as
// if it had come, each later wait of the thread with a single try: it ends, and
// its output is not to be used.
__device__ unsigned long long g_wait_timeouts;
struct Patience {
  int tries = 1 << 18;
  __device__ __forceinline__ void wait(uint64_t *m, int parity) {
    for (int i = 0; i < tries; ++i)
      if (mbar_try(m, parity)) return;
    if (tries > 1) atomicAdd(&g_wait_timeouts, 1ull);
    tries = 1;
  }
};

}  // namespace
}  // namespace fkv
