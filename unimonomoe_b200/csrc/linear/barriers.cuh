// Barriers in shared memory: what ../ptx_sm100.cuh lacks of them.
#pragma once
#include <cstdint>
#include "../ptx_sm100.cuh"

namespace mono {
namespace lin {

// Whether phase `parity` is complete, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}

}  // namespace lin
}  // namespace mono
