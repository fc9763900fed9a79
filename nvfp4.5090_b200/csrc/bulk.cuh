// Bulk copies into shared memory on an mbarrier, with bounded waits: shared by
// the kernels that stage contiguous rows or tiles ahead.
#pragma once

#include "common.cuh"

namespace nvfp4b200 {
namespace bulk {

constexpr long long WAIT_CYCLES = 4000000000ll;   // about 2 s

__device__ __forceinline__ uint32_t addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// One thread, before a __syncthreads(): `n` barriers that `count` arrivals complete.
__device__ __forceinline__ void init(uint64_t* bars, int n, uint32_t count = 1) {
  for (int i = 0; i < n; ++i)
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(addr(bars + i)), "r"(count) : "memory");
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

__device__ __forceinline__ void expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(addr(bar)), "r"(bytes) : "memory");
}

// Source, destination and size are multiples of 16 bytes.
__device__ __forceinline__ void copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(addr(dst)),
               "l"(src), "r"(bytes), "r"(addr(bar))
               : "memory");
}

// CLUSTER: for what another CTA of the cluster wrote.
template <bool CLUSTER>
__device__ __forceinline__ bool test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  if (CLUSTER)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(addr(bar)), "r"(parity)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(addr(bar)), "r"(parity)
        : "memory");
  return ok != 0;
}

// False when the phase did not complete within the limit.
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
  if (test<CLUSTER>(bar, parity)) return true;
  const long long t0 = clock64();
  while (!test<CLUSTER>(bar, parity))
    if (clock64() - t0 > WAIT_CYCLES) return false;
  return true;
}

}  // namespace bulk
}  // namespace nvfp4b200
