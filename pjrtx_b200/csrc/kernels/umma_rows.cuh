// What the tensor-core kernels that attend with query rows in tensor-memory lanes share (umma_prompt.cuh, umma_tree.cuh).
#pragma once

#include <type_traits>

#include "arith.cuh"
#include "paged.cuh"
#include "row_attention.cuh"
#include "umma_attention.cuh"

namespace pjrtx {
namespace umma {

// A probability goes to the tensor core as two numbers of the element type: as one, it would be as far off as the result's own rounding, and results
// 1.1 to 1.4 times as far from the exact ones as that leaves them (1.0 so). The second product and the split take 20 to 30 % of
// long prompts (4 x 2048 tokens, 32 heads of 128 over 8: 146 us with one number, 181 with two) and 5 to 10 % of trees over cached rows, which are
// bound by these. The sum is taken in f32, before. In f16 they are multiplied by 2^11 first: f16 then holds them down to 2^-35 of
// the largest, and not only to 2^-24.
// They are relative to a maximum that follows the row's when that has grown by 2^8 (f16: 2^4, so that they stay below 2^16; by 2^3 long prompts take
// 3 % more): the factor cancels in the division, and the results in tensor memory are rescaled that much more rarely. Where one row of a warp has
// to, all of them follow theirs, so that the next time is later.
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

// A block of threads leaves behind the copies and products that it has under way, whichever of its warps has given up: these waits are for them
// alone, which end by themselves, and take 17 ms at most, where a barrier's other arrivals do not come.
constexpr unsigned long long kLandNs = 1ull << 24;
__device__ __forceinline__ void wait_landed(uint64_t* bar, unsigned parity, unsigned long long until) {
  while (!mbar_try_wait(bar, parity) && global_timer_ns() < until) {
  }
}

__device__ __forceinline__ void tmem_store_16(uint32_t addr, const float* v) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15])
      : "memory");
}

// (y.x, y.y) >= 0 as the sum of two pairs, what is left of it when cut off and the rest, rounded: off by 2^-16 of it in bf16 and 2^-22 in f16, or,
// where the rest is subnormal, by 2^-25 (2^-36 of the largest).
template <bool BF16>
__device__ __forceinline__ uint2 split_probabilities(float2 y) {
  uint32_t high;
  float2 cut;
  if (BF16) {
    high = __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x7632);
    cut = make_float2(__uint_as_float(__float_as_uint(y.x) & 0xffff0000u), __uint_as_float(__float_as_uint(y.y) & 0xffff0000u));
  } else {
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(high) : "f"(y.y), "f"(y.x));
    cut = __half22float2(*reinterpret_cast<const __half2*>(&high));
  }
  const float2 rest = pair_split(pair_fma(pair_of(cut.x, cut.y), pair_of(-1.f, -1.f), pair_of(y.x, y.y)));
  return make_uint2(high, pack_pair<BF16>(rest.x, rest.y));
}

// Probabilities 2^(s * scale + shift) of 32 scores, in the place of these: of 16 keys, eight columns of their first numbers and eight of the second ones,
// as pairs; `part` adds them up.
// All by the exponential unit, 16 results a cycle and SM: to compute some on the FMA units instead (a polynomial behind a split of the
// exponent) made every case slower, 2 to 15 %, by the code that it takes.
template <bool BF16>
__device__ __forceinline__ void store_probabilities(const float (&s)[32], float scale, float shift, Pair (&part)[2], uint32_t to) {
  const Pair scale2 = pair_of(scale, scale), shift2 = pair_of(shift, shift);
#pragma unroll
  for (int h = 0; h < 32; h += 16) {
    float packed[16];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float2 x = pair_split(pair_fma(pair_of(s[h + 2 * e], s[h + 2 * e + 1]), scale2, shift2));
      const float2 y = make_float2(exp2_approx(x.x), exp2_approx(x.y));
      part[e & 1] = pair_add(part[e & 1], pair_of(y.x, y.y));
      const uint2 numbers = split_probabilities<BF16>(y);
      packed[e] = __uint_as_float(numbers.x);
      packed[8 + e] = __uint_as_float(numbers.y);
    }
    tmem_store_16(to + h, packed);
  }
}

// results += P . V for 16 keys, P at `probabilities` as above.
__device__ __forceinline__ void mma_values(uint32_t results, uint32_t probabilities, uint64_t v, uint32_t idesc, uint32_t accumulate) {
  mma_f16_tmem_a(results, probabilities, v, idesc, accumulate);
  mma_f16_tmem_a(results, probabilities + 8, v, idesc, 1u);
}

// Whether one of two packed 16-bit elements is infinite or NaN.
template <bool BF16>
__device__ __forceinline__ bool odd_pair(uint32_t w) {
  constexpr uint32_t kExponent = BF16 ? 0x7f80u : 0x7c00u;
  return (w & kExponent) == kExponent || (w >> 16 & kExponent) == kExponent;
}

// Of 32 columns of values that a row sees, those with a NaN, an infinity, a negative one. What the row's results there are follows from these alone, as long as
// its scores are finite: a probability above 0 times infinity is infinite, however small it is, and the tensor core makes NaN of it where one of the
// probability's two numbers is 0.
struct OddColumns {
  unsigned nan, plus, minus;
  __device__ __forceinline__ void add(const OddColumns& o) {
    nan |= o.nan;
    plus |= o.plus;
    minus |= o.minus;
  }
  __device__ __forceinline__ void join_lanes() {
    nan = __reduce_or_sync(0xffffffffu, nan);
    plus = __reduce_or_sync(0xffffffffu, plus);
    minus = __reduce_or_sync(0xffffffffu, minus);
  }
  __device__ __forceinline__ unsigned any() const { return nan | plus | minus; }
  // Result of column e, one of any().
  __device__ __forceinline__ float of(int e) const {
    return nan >> e & 1 || (plus & minus) >> e & 1 ? __int_as_float(0x7fffffff) : plus >> e & 1 ? INFINITY : -INFINITY;
  }
};

// Whether one of a row's elements is infinite or NaN.
template <bool BF16>
__device__ __forceinline__ bool odd_row(const unsigned short* x, int head_dim) {
  bool found = false;
#pragma unroll 1
  for (int d = 0; d < head_dim; d += 8) {
    const uint4 w = *reinterpret_cast<const uint4*>(x + d);
    found = found || odd_pair<BF16>(w.x) || odd_pair<BF16>(w.y) || odd_pair<BF16>(w.z) || odd_pair<BF16>(w.w);
  }
  return found;
}

// Those of columns c .. c + 31 of a key's values. A row that sees a key with an infinite element and has a finite sum has a score of -inf there: a
// probability of 0, which makes NaN of an infinity.
template <bool BF16>
__device__ __forceinline__ OddColumns odd_columns(const unsigned short* k, const unsigned short* v, int c, int head_dim) {
  OddColumns o = {0, 0, 0};
#pragma unroll 1
  for (int d = 0; d < 32 && c + d < head_dim; d += 8) {
    const uint4 x = *reinterpret_cast<const uint4*>(v + c + d);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint32_t y = w[e / 2] >> (e % 2 * 16) & 0xffffu, infinity = BF16 ? 0x7f80u : 0x7c00u, bit = 1u << (d + e);
      if ((y & 0x7fffu) > infinity) o.nan |= bit;
      if (y == infinity) o.plus |= bit;
      if (y == (infinity | 0x8000u)) o.minus |= bit;
    }
  }
  if ((o.plus | o.minus) && odd_row<BF16>(k, head_dim)) o = {o.any(), 0, 0};
  return o;
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
