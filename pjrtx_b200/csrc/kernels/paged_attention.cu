// Attention of one new token per sequence over a paged key-value cache.
//
//   s_t = scale * q . k_t (t < length),  m = max s,  l = sum e^(s_t - m),  out = sum e^(s_t - m) v_t / l,  lse = m + ln l
//
// A sequence without rows gives zeros and an lse of -inf. Rows beyond the length are not read: what a page holds there, or the
// table names for them, does not matter. With a new row in the call, row length - 1 is taken from there and stored.
//
// Tracking adds to weights[b, g, t] the weights e^(s_t - lse) of the query heads that read KV head g. They need the whole row's
// lse, so the scores (4 bytes a head and key, against 4 * head_dim of key and value) go through the workspace to a second kernel.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../common.h"
#include "kernels.h"
#include "paged.cuh"

namespace pjrtx {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

struct AttendSpace {
  float* lse2;    // [batch, heads]: lse / ln 2
  float* scores;  // [batch, kv_heads, capacity, rep] in units of ln 2 (tracking only)
};

inline AttendSpace attend_space(const PagedView& c, int heads, void* workspace) {
  AttendSpace s;
  char* p = static_cast<char*>(workspace);
  s.lse2 = reinterpret_cast<float*>(p);
  s.scores = reinterpret_cast<float*>(p + ((uint64_t)c.batch_max * heads * 4 + 255) / 256 * 256);
  return s;
}

constexpr int kSimpleWarps = 8;

// One block per (query head, sequence), one key per warp and step.
template <typename T>
__global__ void __launch_bounds__(kSimpleWarps * 32) paged_attend_kernel(PagedView c, PagedAttend a, AttendSpace space) {
  constexpr int R = 8;  // 256 / 32
  __shared__ float acc[kSimpleWarps][32 * R];
  __shared__ float stat[kSimpleWarps][2];
  PJRTX_PDL_PROLOGUE();
  const int h = blockIdx.x, b = blockIdx.y, rep = a.heads / c.kv_heads, g = h / rep;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, D = c.head_dim;
  const int n = paged_length(c, b);
  if (h == 0 && threadIdx.x == 0) paged_check_length(c, b);
  const T* q = static_cast<const T*>(a.q) + b * a.q_batch_stride + h * a.q_head_stride;
  float qr[R], o[R], m = -INFINITY, l = 0.f;
  for (int i = 0; i < R; i++) {
    const int d = lane + 32 * i;
    qr[i] = d < D ? to_float(q[d]) * a.scale * kLog2e : 0.f;
    o[i] = 0.f;
  }
  for (int t = warp; t < n; t += kSimpleWarps) {
    const long long row = paged_row(c, b, t);
    if (row < 0) continue;
    const T* k = static_cast<const T*>(c.k) + row + g * c.head_stride;
    const T* v = static_cast<const T*>(c.v) + row + g * c.head_stride;
    if (a.k_new && t == n - 1) {
      const T* k_new = static_cast<const T*>(a.k_new) + b * a.new_batch_stride + g * a.new_head_stride;
      const T* v_new = static_cast<const T*>(a.v_new) + b * a.new_batch_stride + g * a.new_head_stride;
      if (h % rep == 0)
        for (int d = lane; d < D; d += 32) {
          const_cast<T*>(k)[d] = k_new[d];
          const_cast<T*>(v)[d] = v_new[d];
        }
      k = k_new;
      v = v_new;
    }
    float s = 0.f;
    for (int i = 0; i < R; i++)
      if (lane + 32 * i < D) s = fmaf(qr[i], to_float(k[lane + 32 * i]), s);
    for (int d = 16; d; d /= 2) s += __shfl_xor_sync(~0u, s, d);
    if (c.weights && lane == 0) space.scores[(((long long)b * c.kv_heads + g) * c.page_size * c.max_pages + t) * rep + h % rep] = s;
    const float to = max_nan(m, s), f = m == -INFINITY ? 0.f : exp2f(m - to), p = to == -INFINITY ? 0.f : exp2f(s - to);
    l = l * f + p;
    for (int i = 0; i < R; i++)
      if (lane + 32 * i < D) o[i] = fmaf(p, to_float(v[lane + 32 * i]), o[i] * f);
    m = to;
  }
  if (lane == 0) {
    stat[warp][0] = m;
    stat[warp][1] = l;
  }
  for (int i = 0; i < R; i++) acc[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float top = -INFINITY, total = 0.f;
  for (int w = 0; w < kSimpleWarps; w++) top = max_nan(top, stat[w][0]);
  for (int w = 0; w < kSimpleWarps; w++) total += stat[w][0] == -INFINITY ? 0.f : stat[w][1] * exp2f(stat[w][0] - top);
  const float inverse = total > 0.f ? 1.f / total : (total != total ? total : 0.f);
  T* out = static_cast<T*>(a.out) + b * a.out_batch_stride + h * a.out_head_stride;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float x = 0.f;
    for (int w = 0; w < kSimpleWarps; w++) x += stat[w][0] == -INFINITY ? 0.f : acc[w][d] * exp2f(stat[w][0] - top);
    out[d] = from_float<T>(x * inverse);
  }
  if (threadIdx.x == 0) {
    const float lse2 = total == 0.f ? -INFINITY : top + log2f(total);
    space.lse2[(long long)b * a.heads + h] = lse2;
    if (a.lse) a.lse[(long long)b * a.heads + h] = lse2 * kLn2;
  }
}

constexpr int kTrackThreads = 256;

__global__ void __launch_bounds__(kTrackThreads) paged_track_kernel(PagedView c, AttendSpace space, int heads, int appended) {
  PJRTX_PDL_PROLOGUE();
  const int g = blockIdx.y, b = blockIdx.z, rep = heads / c.kv_heads;
  const int n = paged_length(c, b);
  const long long base = ((long long)b * c.kv_heads + g) * c.page_size * c.max_pages;
  const float* lse2 = space.lse2 + (long long)b * heads + g * rep;
  for (int t = blockIdx.x * kTrackThreads + threadIdx.x; t < n; t += gridDim.x * kTrackThreads) {
    const float* s = space.scores + (base + t) * rep;
    float w = 0.f;
    for (int r = 0; r < rep; r++) w += lse2[r] == -INFINITY ? 0.f : exp2f(s[r] - lse2[r]);
    if (appended && t == n - 1) {
      c.weights[base + t] = w;
      c.positions[base + t] = c.tokens[b] - 1;
    } else {
      c.weights[base + t] += w;
    }
  }
}

template <typename T>
bool attend(const PagedView& c, const PagedAttend& a, const AttendSpace& space, bool pdl, cudaStream_t stream) {
  return launch_kernel(paged_attend_kernel<T>, dim3((unsigned)a.heads, (unsigned)c.batch), dim3(kSimpleWarps * 32), 0, stream, pdl, c, a,
                       space) == cudaSuccess;
}

}  // namespace

uint64_t paged_attend_workspace_bytes(const PagedView& c, int heads, bool track, int sm_count) {
  (void)sm_count;
  return ((uint64_t)c.batch_max * heads * 4 + 255) / 256 * 256 + (track ? (uint64_t)c.batch_max * heads * c.capacity() * 4 : 0);
}

int paged_attend_launch(const PagedView& c, const PagedAttend& a, int sm_count, bool pdl, cudaStream_t stream) {
  const AttendSpace space = attend_space(c, a.heads, a.workspace);
  const bool ok = c.dtype == kF32 ? attend<float>(c, a, space, pdl, stream) : c.dtype == kF16 ? attend<__half>(c, a, space, pdl, stream)
                                                                                             : attend<__nv_bfloat16>(c, a, space, pdl, stream);
  if (!ok) return 0;
  if (!c.weights) return 1;
  const long long pairs = (long long)c.batch * c.kv_heads;
  const long long blocks = std::max<long long>(1, std::min((c.capacity() + kTrackThreads - 1) / kTrackThreads, 8ll * sm_count / pairs + 1));
  return launch_kernel(paged_track_kernel, dim3((unsigned)blocks, (unsigned)c.kv_heads, (unsigned)c.batch), dim3(kTrackThreads), 0, stream, true,
                       c, space, a.heads, a.k_new != nullptr) == cudaSuccess ? 2 : 0;
}

}  // namespace pjrtx
