// What the tensor-core kernels that attend with query rows in tensor-memory lanes share (umma_prompt.cuh, umma_tree.cuh).
#pragma once

#include <type_traits>

#include "paged.cuh"
#include "row_attention.cuh"
#include "umma_attention.cuh"

namespace pjrtx {
namespace umma {

// Probabilities go to the tensor core in the element type, and the sum is taken of them as they are then, so that equal values under all
// keys give that value. In f16 they are multiplied by 2^11 first: f16 then holds them down to 2^-35 of the largest, and not only to 2^-24.
// They are relative to a maximum that follows the row's when that has grown by 2^8 (f16: 2^4, so that they stay below 2^16): the factor
// cancels in the division, and the results in tensor memory are rescaled that much more rarely.
template <bool BF16> struct Probability { static constexpr float kLift = 0.f, kGrow = 8.f; };
template <> struct Probability<false> { static constexpr float kLift = 11.f, kGrow = 4.f; };

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
template <int REGISTERS>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGISTERS));
}
template <int REGISTERS>
__device__ __forceinline__ void leave_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGISTERS));
}
// Whether one of two packed 16-bit elements is infinite or NaN.
template <bool BF16>
__device__ __forceinline__ bool odd_pair(uint32_t w) {
  constexpr uint32_t kExponent = BF16 ? 0x7f80u : 0x7c00u;
  return (w & kExponent) == kExponent || (w >> 16 & kExponent) == kExponent;
}

}  // namespace umma
}  // namespace pjrtx
