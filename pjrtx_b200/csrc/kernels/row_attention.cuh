// Attention of a tile of query rows over the keys that each of them sees, on the CUDA cores and in f32:
//
//   s_ij = scale * q_i . k_j (j seen by i),  m_i = max s_ij,  l_i = sum e^(s_ij - m_i),  out_i = sum e^(s_ij - m_i) v_j / l_i
//
// A row sees the keys below its limit, and of 64 keys from `base` on those in its word of bits: for a prompt the limit is the position
// and there are no bits, for a tree of drafted tokens the limit is the cached length and the bits are the ancestors.
//
// 256 threads, 16, 32 or 64 rows and 64 keys (32 of 256 dimensions) at a time: a thread has up to four rows by four keys of the
// scores, then its rows by a sixteenth of the dimensions of the values, two products an instruction; the running maximum and sum of a row are in
// the sixteen threads that have it. The next keys and values come by cp.async while these are at work. One or two rows a
// thread are for trees of few rows, which would compute rows that are not there. Bound by FMAs and the reads of shared memory beside them:
// 16 sequences of up to 2000 rows, 32 heads of 128 over 8, take 173 us with 8 nodes, 154 with one and 634 with 40; prompts of 4 x 2048 tokens
// of such heads 3.9 ms (35 TFLOP/s), 517 tokens 76 us, 48 prompts of 67 to 200, four heads of 64 over two, 30 from long to short and 37
// in no order. A warp leaves out keys that none of its rows sees, half a block of scores or four values at a time (517 tokens 82 us without).
// What a row does not see enters nothing: scores are replaced, and where values of a block are infinite or NaN the products with
// hidden keys are left out one by one.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "arith.cuh"

namespace pjrtx {
namespace rows {

constexpr int kThreads = 256;
__host__ __device__ constexpr int keys_of(int d) { return d == 256 ? 32 : 64; }  // of a block
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

template <int D, int R>  // R rows a thread
struct Shared {
  static constexpr int kRows = 16 * R, kKeys = keys_of(D), kPitch = D + 4;  // rows of neighbouring threads fall on different banks
  float q[kRows][kPitch];
  float k[2][kKeys][kPitch];
  float v[2][kKeys][D];
  float p[kRows][kKeys + 4];
};

// Sums of a thread: rows ty * R + i, dimensions c * 64 + tx * 4 + 0..3 for c < D / 64 (ty = thread / 16, tx = thread % 16).
template <int D, int R>
struct Sums {
  Pair o[R][D / 64][2];
  float m[R], l[R];  // in units of ln 2; the same in the sixteen threads of a row
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < R; i++) {
#pragma unroll
      for (int c = 0; c < D / 64; c++) o[i][c][0] = o[i][c][1] = 0;
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
  }
};

__device__ __forceinline__ void copy16_or_zero(float* to, const float* from, bool there, const float* any) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(there ? from : any), "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Rows of a block are copied by warps, ROWS / 8 neighbouring ones each, a lane 16 bytes: visit(i, row, d) for each piece that this lane has,
// row `i` of the warp's.
template <int D, int ROWS, typename Visit>
__device__ __forceinline__ void pieces_of_lane(Visit visit) {
  constexpr int kPieces = D / 4, kAcross = kPieces >= 32 ? 1 : 32 / kPieces, kOfWarp = ROWS / 8;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll 4
  for (int i0 = 0; i0 < kOfWarp; i0 += kAcross) {
    const int i = i0 + lane / kPieces;
#pragma unroll
    for (int d = lane % kPieces * 4; d < D; d += 128) visit(i, warp * kOfWarp + i, d);
  }
}

// Requests the rows of a block, `row` being the address of row `lane` of the warp's part (null: zeros).
template <int D, int ROWS, int PITCH>
__device__ __forceinline__ void request_rows(float (*to)[PITCH], const float* row, int head_dim, const float* any) {
  const unsigned long long at = reinterpret_cast<unsigned long long>(row);
  pieces_of_lane<D, ROWS>([&](int i, int r, int d) {
    const float* from = reinterpret_cast<const float*>(__shfl_sync(~0u, at, i));
    copy16_or_zero(&to[r][d], from + d, from && d < head_dim, any);
  });
}

// Block `stage & 1`: keys key0 .. (those before `keys`), which has been requested, into the sums; requests the next one by `next()`. The
// queries are in shared memory once the first block is. No row of the warp sees keys from `reach` on.
template <bool HALVES, int D, int R, typename Next>
__device__ __forceinline__ void block_of_keys(Shared<D, R>& s, Sums<D, R>& sum, const Sight (&sight)[R], int stage, int key0, int keys, int reach,
                                              int base, float scale2, Next next) {
  constexpr int kKeys = keys_of(D), kColumns = kKeys / 16;
  const int end = min(kKeys, reach - key0);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float(*const sk)[D + 4] = s.k[stage & 1];
  float(*const sv)[D] = s.v[stage & 1];
  copies_wait();
  bool found = false;
  pieces_of_lane<D, kKeys>([&](int, int r, int d) {
    const float4 x = *reinterpret_cast<const float4*>(&sv[r][d]);
    found = found || odd(x.x) || odd(x.y) || odd(x.z) || odd(x.w);
  });
  const bool careful = __syncthreads_or(found);  // all rows have landed, and the other stage has been read
  next();
  if (end <= 0) return;
  Pair a[R][kColumns];
#pragma unroll
  for (int i = 0; i < R; i++)
#pragma unroll
    for (int j = 0; j < kColumns; j++) a[i][j] = 0;
  auto products = [&](auto columns) {
    constexpr int kOf = decltype(columns)::value;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      ulonglong2 q[R], k[kOf];
#pragma unroll
      for (int i = 0; i < R; i++) q[i] = *reinterpret_cast<const ulonglong2*>(&s.q[ty * R + i][d]);
#pragma unroll
      for (int j = 0; j < kOf; j++) k[j] = *reinterpret_cast<const ulonglong2*>(&sk[tx + 16 * j][d]);
#pragma unroll
      for (int i = 0; i < R; i++)
#pragma unroll
        for (int j = 0; j < kOf; j++) a[i][j] = pair_fma(q[i].y, k[j].y, pair_fma(q[i].x, k[j].x, a[i][j]));
    }
  };
  if (HALVES && end <= kKeys / 2) products(std::integral_constant<int, kColumns / 2>());
  else products(std::integral_constant<int, kColumns>());
#pragma unroll
  for (int i = 0; i < R; i++) {
    float x[kColumns], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kColumns; j++) {
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
    for (int j = 0; j < kColumns; j++) {
      x[j] = exp2_fast(x[j] - shift);
      s.p[ty * R + i][tx + 16 * j] = x[j];
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
    for (int t = 0; t < end; t++) {
#pragma unroll
      for (int i = 0; i < R; i++) {
        if (!sees(sight[i], key0 + t, base)) continue;
        const float p = s.p[ty * R + i][t];
        const Pair p2 = pair_of(p, p);
#pragma unroll
        for (int c = 0; c < D / 64; c++) {
          const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sv[t][c * 64 + tx * 4]);
          sum.o[i][c][0] = pair_fma(p2, v.x, sum.o[i][c][0]);
          sum.o[i][c][1] = pair_fma(p2, v.y, sum.o[i][c][1]);
        }
      }
    }
    return;
  }
#pragma unroll 2
  for (int t = 0; t < end; t += 4) {
    float4 p[R];
#pragma unroll
    for (int i = 0; i < R; i++) p[i] = *reinterpret_cast<const float4*>(&s.p[ty * R + i][t]);
#pragma unroll
    for (int u = 0; u < 4; u++) {
      ulonglong2 v[D / 64];
#pragma unroll
      for (int c = 0; c < D / 64; c++) v[c] = *reinterpret_cast<const ulonglong2*>(&sv[t + u][c * 64 + tx * 4]);
#pragma unroll
      for (int i = 0; i < R; i++) {
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
