// What the tensor-core kernels that attend with query rows in tensor-memory lanes share (umma_prompt.cuh, umma_tree.cuh).
#pragma once

#include <type_traits>

#include "arith.cuh"
#include "paged.cuh"
#include "row_attention.cuh"
#include "umma_attention.cuh"

namespace pjrtx {
namespace umma {

// Probabilities go to the tensor core in the element type: two 16-bit numbers for each would make the second product twice as long, and as
// one they add about as much to a result's error as its own rounding does. Their sum is taken before they are rounded, since the log-sum-exp
// is f32 (of the rounded ones it would be off by up to 2^-9). In f16 they are multiplied by 2^11 first: f16 then holds them down to
// 2^-35 of the largest, and not only to 2^-24.
// They are relative to a maximum that follows the row's when that has grown by 2^8 (f16: 2^4, so that they stay below 2^16): the factor
// cancels in the division, and the results in tensor memory are rescaled that much more rarely. Where one row of a warp has to, all of them
// follow theirs, so that the next time is later.
template <bool BF16> struct Probability { static constexpr float kLift = 0.f, kGrow = 8.f; };
template <> struct Probability<false> { static constexpr float kLift = 11.f, kGrow = 4.f; };

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// The largest of N of a row's scores and of those before them, which `mx` has in four chains.
template <int N>
__device__ __forceinline__ float max_of(const float* s, float (&mx)[4]) {
#pragma unroll
  for (int e = 0; e < N; e += 8)
#pragma unroll
    for (int i = 0; i < 4; i++) mx[i] = max3(mx[i], s[e + 2 * i], s[e + 2 * i + 1]);
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}

// Waits end that long after now; launches say how long.
__device__ __forceinline__ WaitBudget budget_from_now(unsigned long long timeout_ns, volatile int* abort) {
  return WaitBudget{global_timer_ns() + timeout_ns, abort};
}

__device__ __forceinline__ void tmem_store_16(uint32_t addr, const float* v) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15])
      : "memory");
}

// Probabilities 2^(s * scale + shift) of 32 scores into 16 columns of tensor memory, as pairs of the element type; `part` adds them up.
// All by the exponential unit, 16 results a cycle and SM: to compute some on the FMA units instead (a polynomial behind a split of the
// exponent) made every case slower, 2 to 15 %, by the code that it takes.
template <bool BF16>
__device__ __forceinline__ void store_probabilities(const float (&s)[32], float scale, float shift, Pair (&part)[2], uint32_t to) {
  const Pair scale2 = pair_of(scale, scale), shift2 = pair_of(shift, shift);
  float packed[16];
#pragma unroll
  for (int e = 0; e < 16; e++) {
    const float2 x = pair_split(pair_fma(pair_of(s[2 * e], s[2 * e + 1]), scale2, shift2));
    const float2 y = make_float2(exp2_approx(x.x), exp2_approx(x.y));
    part[e & 1] = pair_add(part[e & 1], pair_of(y.x, y.y));
    packed[e] = __uint_as_float(pack_pair<BF16>(y.x, y.y));
  }
  tmem_store_16(to, packed);
}
// Whether one of two packed 16-bit elements is infinite or NaN.
template <bool BF16>
__device__ __forceinline__ bool odd_pair(uint32_t w) {
  constexpr uint32_t kExponent = BF16 ? 0x7f80u : 0x7c00u;
  return (w & kExponent) == kExponent || (w >> 16 & kExponent) == kExponent;
}

// Whether one of them is infinite.
template <bool BF16>
__device__ __forceinline__ bool infinite_pair(uint32_t w) {
  constexpr uint32_t kInfinity = BF16 ? 0x7f80u : 0x7c00u;
  return (w & 0x7fffu) == kInfinity || (w >> 16 & 0x7fffu) == kInfinity;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A map of `rank` axes, head_dim first, for boxes of 64 elements; `strides` (elements) are those of the axes behind the first. An axis of
// one element may come with any stride, which the encoder does not take.
inline bool encode_map(CUtensorMap* map, const void* base, bool f16, int rank, const long long* extents, const long long* strides, const int* box) {
  static const EncodeTiledFn encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess) f = nullptr;
    return (EncodeTiledFn)f;
  }();
  if (!encode) return false;
  cuuint64_t dims[4], bytes[3];
  cuuint32_t boxes[4], steps[4];
  for (int d = 0; d < rank; d++) {
    dims[d] = (cuuint64_t)extents[d];
    boxes[d] = (cuuint32_t)box[d];
    steps[d] = 1;
    if (d) bytes[d - 1] = (cuuint64_t)(extents[d] == 1 ? extents[0] : strides[d - 1]) * 2;
  }
  return encode(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base), dims, bytes,
                boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace umma
}  // namespace pjrtx
