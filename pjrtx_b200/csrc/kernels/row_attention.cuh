// Attention of a tile of query rows over the keys that each of them sees, on the CUDA cores and in f32:
//
//   s_ij = scale * q_i . k_j (j seen by i),  m_i = max s_ij,  l_i = sum e^(s_ij - m_i),  out_i = sum e^(s_ij - m_i) v_j / l_i
//
// A row sees the keys below its limit, and of 64 keys from `base` on those in its word of bits: for a prompt the limit is the position
// and there are no bits, for a tree of drafted tokens the limit is the cached length and the bits are the ancestors.
//
// 256 threads, 64 rows and 64 keys at a time: a thread has four rows by four keys of the scores, then four rows by a sixteenth of the
// dimensions of the values, two products an instruction; the running maximum and sum of a row are in the sixteen threads that have it.
// What a row does not see enters nothing: scores are replaced, and where values of a block are infinite or NaN the products with
// hidden keys are left out one by one.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "arith.cuh"

namespace pjrtx {
namespace rows {

constexpr int kRows = 64, kKeys = 64, kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// What a query row sees.
struct Sight {
  int limit;                // keys below it
  unsigned long long bits;  // and of the keys from `base` on
};
__device__ __forceinline__ bool sees(const Sight& s, int key, int base) {
  return key < s.limit || (key >= base && key - base < 64 && (s.bits >> (key - base) & 1));
}

template <typename T> __device__ __forceinline__ void unpack16(const uint4& x, float* to);
template <> __device__ __forceinline__ void unpack16<float>(const uint4& x, float* to) {
  to[0] = __uint_as_float(x.x);
  to[1] = __uint_as_float(x.y);
  to[2] = __uint_as_float(x.z);
  to[3] = __uint_as_float(x.w);
}
template <> __device__ __forceinline__ void unpack16<__half>(const uint4& x, float* to) {
  const __half2* h = reinterpret_cast<const __half2*>(&x);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = __half22float2(h[i]);
    to[2 * i] = f.x;
    to[2 * i + 1] = f.y;
  }
}
template <> __device__ __forceinline__ void unpack16<__nv_bfloat16>(const uint4& x, float* to) {
  const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    to[2 * i] = __uint_as_float(w[i] << 16);
    to[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ bool odd(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }  // infinite or NaN

template <int D>
struct Shared {
  static constexpr int kPitch = D + 4;  // rows of neighbouring threads fall on different banks
  float q[kRows][kPitch];
  float k[kKeys][kPitch];
  float v[kKeys][D];
  float p[kRows][kKeys + 4];
};

// Sums of a thread: rows ty * 4 + i, dimensions c * 64 + tx * 4 + 0..3 for c < D / 64 (ty = thread / 16, tx = thread % 16).
template <int D>
struct Sums {
  Pair o[4][D / 64][2];
  float m[4], l[4];  // in units of ln 2; the same in the sixteen threads of a row
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
      for (int c = 0; c < D / 64; c++) o[i][c][0] = o[i][c][1] = 0;
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
  }
};

// Rows of `count` x head_dim elements into shared memory; row(i) is a row's address or null, which gives zeros. True where a value is odd.
template <typename T, int D, int PITCH, typename Row>
__device__ __forceinline__ bool load_rows(float (*to)[PITCH], int head_dim, Row row) {
  constexpr int kPer = 16 / (int)sizeof(T), kPieces = D / kPer;
  bool found = false;
  for (int i = threadIdx.x; i < 64 * kPieces; i += kThreads) {
    const int r = i / kPieces, d = i % kPieces * kPer;
    const T* from = row(r);
    float x[kPer];
    if (from && d < head_dim) {
      unpack16<T>(*reinterpret_cast<const uint4*>(from + d), x);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; e++) x[e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < kPer; e += 4) {
      *reinterpret_cast<float4*>(&to[r][d + e]) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
      found = found || odd(x[e]) || odd(x[e + 1]) || odd(x[e + 2]) || odd(x[e + 3]);
    }
  }
  return found;
}

// Keys key0..key0 + 63 (those before `keys`) into the sums. The queries are in shared memory. key(t) and value(t): addresses or null.
template <typename T, int D, typename Key, typename Value>
__device__ __forceinline__ void block_of_keys(Shared<D>& s, Sums<D>& sum, const Sight (&sight)[4], int key0, int keys, int base, int head_dim,
                                              float scale2, Key key, Value value) {
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  __syncthreads();  // the block before has been read
  load_rows<T, D>(s.k, head_dim, [&](int r) { return key0 + r < keys ? key(key0 + r) : nullptr; });
  const bool found = load_rows<T, D>(s.v, head_dim, [&](int r) { return key0 + r < keys ? value(key0 + r) : nullptr; });
  const bool careful = __syncthreads_or(found);
  Pair a[4][4];
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) a[i][j] = 0;
#pragma unroll 4
  for (int d = 0; d < D; d += 4) {
    ulonglong2 q[4], k[4];
#pragma unroll
    for (int i = 0; i < 4; i++) q[i] = *reinterpret_cast<const ulonglong2*>(&s.q[ty * 4 + i][d]);
#pragma unroll
    for (int j = 0; j < 4; j++) k[j] = *reinterpret_cast<const ulonglong2*>(&s.k[tx + 16 * j][d]);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) a[i][j] = pair_fma(q[i].y, k[j].y, pair_fma(q[i].x, k[j].x, a[i][j]));
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float x[4], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float2 f = pair_split(a[i][j]);
      const int t = key0 + tx + 16 * j;
      x[j] = t < keys && sees(sight[i], t, base) ? (f.x + f.y) * scale2 : -INFINITY;
      top = fmaxf(top, x[j]);
    }
#pragma unroll
    for (int w = 8; w; w /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, w));
    top = fmaxf(top, sum.m[i]);
    const float shift = top == -INFINITY ? 0.f : top, corr = top == sum.m[i] ? 1.f : exp2_fast(sum.m[i] - shift);
    float total = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x[j] = exp2_fast(x[j] - shift);
      s.p[ty * 4 + i][tx + 16 * j] = x[j];
      total += x[j];
    }
#pragma unroll
    for (int w = 8; w; w /= 2) total += __shfl_xor_sync(~0u, total, w);
    sum.l[i] = fmaf(sum.l[i], corr, total);
    sum.m[i] = top;
    const Pair c2 = pair_of(corr, corr);
#pragma unroll
    for (int c = 0; c < D / 64; c++) {
      sum.o[i][c][0] = pair_mul(sum.o[i][c][0], c2);
      sum.o[i][c][1] = pair_mul(sum.o[i][c][1], c2);
    }
  }
  __syncwarp();  // a row's probabilities are written and read by the same warp
  if (careful) {
    for (int t = 0; t < kKeys; t++) {
      if (key0 + t >= keys) break;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (!sees(sight[i], key0 + t, base)) continue;
        const float p = s.p[ty * 4 + i][t];
        const Pair p2 = pair_of(p, p);
#pragma unroll
        for (int c = 0; c < D / 64; c++) {
          const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&s.v[t][c * 64 + tx * 4]);
          sum.o[i][c][0] = pair_fma(p2, v.x, sum.o[i][c][0]);
          sum.o[i][c][1] = pair_fma(p2, v.y, sum.o[i][c][1]);
        }
      }
    }
    return;
  }
#pragma unroll 2
  for (int t = 0; t < kKeys; t += 4) {
    float4 p[4];
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = *reinterpret_cast<const float4*>(&s.p[ty * 4 + i][t]);
#pragma unroll
    for (int u = 0; u < 4; u++) {
      ulonglong2 v[D / 64];
#pragma unroll
      for (int c = 0; c < D / 64; c++) v[c] = *reinterpret_cast<const ulonglong2*>(&s.v[t + u][c * 64 + tx * 4]);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float x = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
        const Pair p2 = pair_of(x, x);
#pragma unroll
        for (int c = 0; c < D / 64; c++) {
          sum.o[i][c][0] = pair_fma(p2, v[c].x, sum.o[i][c][0]);
          sum.o[i][c][1] = pair_fma(p2, v[c].y, sum.o[i][c][1]);
        }
      }
    }
  }
}

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// Four neighbouring elements of a result; rows and dimensions are multiples of four elements of f32 and of eight of 16 bits.
template <typename T>
__device__ __forceinline__ void store4(T* to, float4 x) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(to) = x;
  } else {
    T y[4] = {from_float<T>(x.x), from_float<T>(x.y), from_float<T>(x.z), from_float<T>(x.w)};
    *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(y);
  }
}

// What a row's sums are divided by, and its log-sum-exp: rows that have seen nothing give zeros and -inf.
__device__ __forceinline__ float inverse_of(float l) { return l > 0.f ? 1.f / l : l != l ? l : 0.f; }
__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.f ? -INFINITY : fmaf(m, kLn2, logf(l)); }

}  // namespace rows
}  // namespace pjrtx
