// Scoring a decoder's logits: log probability of a given token, entropy, likeliest tokens, and the gradient.
//
// With x = scale * logits, m = max x, S = sum e^(x - m) and T = sum e^(x - m) (x - m) over a row:
//   lse = m + ln S     log p(t) = x_t - lse     entropy = -sum p ln p = ln S - T / S
//   d logit_j = scale * ( g (delta_tj - p_j) - h p_j (ln p_j + entropy) ),   p_j = e^(x_j - lse)
// with g, h the gradients of the log probability and of the entropy. A logit of -inf has p = 0 and adds nothing to T.
//
// A row is read once: each thread keeps its own running (m, S, T) and rescales only when its maximum grows. The blocks of a
// cluster share a row where there are too few rows to fill the GPU and join through distributed shared memory.
//
// Top k: a chunk is what a warp reads with one 16-byte load a thread, and its maximum goes to shared memory on the way. In the
// order (value descending, id ascending) the k first elements lie in the k first chunks - an element of another chunk has k
// elements before it, the maxima of those - so afterwards only these k chunks are read again.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <utility>

#include "../common.h"
#include "kernels.h"
#include "paged.cuh"

namespace cg = cooperative_groups;

namespace pjrtx {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename T> struct Logit;
template <> struct Logit<float> {
  static constexpr int V = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
};
template <> struct Logit<__nv_bfloat16> {
  static constexpr int V = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint4 r;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    return r;
  }
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
};
template <> struct Logit<__half> {
  static constexpr int V = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 p = __half22float2(h[i]);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint4 r;
    __half2* h = reinterpret_cast<__half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    return r;
  }
  static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// A float in the order of unsigned integers: -0 as +0, NaN above all; 0 stands for "no element".
__device__ __forceinline__ unsigned order_key(float f) {
  if (f != f) return 0xffffffffu;
  const unsigned u = __float_as_uint(f == 0.f ? 0.f : f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(unsigned k) {
  return k == 0xffffffffu ? __uint_as_float(0x7fffffffu) : __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

// Running softmax statistics of raw logits; exponents count in units of ln 2 / scale. m = -inf: nothing but -inf so far.
struct Stats {
  float m, s, t;
};
// What (s, t) of maximum `m` become under the maximum `to` >= m.
__device__ __forceinline__ void restate(Stats& a, float to, float c) {
  if (a.m == to) return;
  const float d = a.m == -INFINITY ? -INFINITY : (a.m - to) * c;
  const float f = exp2_fast(d);
  a.t = f > 0.f ? f * (a.t + d * a.s) : (f != f ? f : 0.f);
  a.s *= f;
  a.m = to;
}
__device__ __forceinline__ Stats joined(Stats a, Stats b, float c) {
  const float m = max_nan(a.m, b.m);
  restate(a, m, c);
  restate(b, m, c);
  return {m, a.s + b.s, a.t + b.t};
}

// ---- forward -------------------------------------------------------------------------------------------------------

constexpr int kScoreThreads = 512, kScoreWarps = kScoreThreads / 32;
constexpr int kScoreUnroll = 4;      // 16-byte loads a thread has in flight
constexpr int kScoreCandidates = 512;
constexpr int kScoreClusterMax = 8;

struct ScoreShared {
  Stats stats[kScoreWarps];
  Stats cluster_stats[kScoreClusterMax];                             // of the rank-0 block
  unsigned long long cluster_top[kScoreClusterMax * kScoreTopMax];   // of the rank-0 block
  unsigned long long candidate[kScoreCandidates];
  int chunk[kScoreTopMax];
  int count[34];
  int n;
  unsigned threshold;
};

// Sum of one small count per thread over the block; nothing used `slot` since it was cleared.
__device__ __forceinline__ int block_count(int mine, int* slot) {
  mine = __reduce_add_sync(~0u, mine);
  if (threadIdx.x % 32 == 0 && mine) atomicAdd(slot, mine);
  __syncthreads();
  return *slot;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kScoreThreads) token_score_kernel(TokenScore a, int segment_chunks) {
  constexpr int V = Logit<T>::V;
  extern __shared__ unsigned chunk_key[];  // TOP: the maxima of this block's chunks
  __shared__ ScoreShared sh;
  PJRTX_PDL_PROLOGUE();
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  auto started = cluster.barrier_arrive();  // rank 0's shared memory is written once its block is known to run
  const long long row = blockIdx.x / ranks;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const T* logits = static_cast<const T*>(a.logits) + row * a.row_stride;
  // Vectors are 16-byte aligned: the row starts `shift` elements into the first one.
  const int shift = (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(T));
  const T* aligned = logits - shift;
  const int end = (int)a.vocab + shift;  // element positions [shift, end) of `aligned` are the row
  const int vectors = (end + V - 1) / V;
  const int chunks = (vectors + 31) / 32;
  const int chunk0 = min(chunks, rank * segment_chunks), chunk1 = min(chunks, chunk0 + segment_chunks);
  const float c = a.scale * kLog2e;

  auto load = [&](int v, float* f) {  // positions outside the row: -inf
    const int p = v * V;
    if (p >= shift && p + V <= end) {
      Logit<T>::unpack(*reinterpret_cast<const uint4*>(aligned + p), f);
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) f[i] = p + i >= shift && p + i < end ? Logit<T>::load(aligned + p + i) : -INFINITY;
    }
  };

  Stats mine = {-INFINITY, 0.f, 0.f};
  for (int k0 = chunk0 + warp * kScoreUnroll; k0 < chunk1; k0 += kScoreWarps * kScoreUnroll) {
    float f[kScoreUnroll][V];
    const bool whole = k0 + kScoreUnroll <= chunk1 && k0 * 32 * V >= shift && (k0 + kScoreUnroll) * 32 * V <= end;
    if (whole) {
      uint4 r[kScoreUnroll];
#pragma unroll
      for (int u = 0; u < kScoreUnroll; u++) r[u] = *reinterpret_cast<const uint4*>(aligned + ((k0 + u) * 32 + lane) * V);
#pragma unroll
      for (int u = 0; u < kScoreUnroll; u++) Logit<T>::unpack(r[u], f[u]);
    } else {
#pragma unroll
      for (int u = 0; u < kScoreUnroll; u++) {
        if (k0 + u < chunk1) {
          load((k0 + u) * 32 + lane, f[u]);
        } else {
#pragma unroll
          for (int i = 0; i < V; i++) f[u][i] = -INFINITY;
        }
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < kScoreUnroll; u++) {
      float best = f[u][0];
#pragma unroll
      for (int i = 1; i < V; i++) best = max_nan(best, f[u][i]);
      if (TOP) {
        const unsigned key = __reduce_max_sync(~0u, order_key(best));
        if (lane == 0 && k0 + u < chunk1) chunk_key[k0 + u - chunk0] = key;
      }
      top = max_nan(top, best);
    }
    if (!(top <= mine.m)) restate(mine, top, c);
    if (mine.m == -INFINITY) continue;
#pragma unroll
    for (int u = 0; u < kScoreUnroll; u++)
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float y = max_nan((f[u][i] - mine.m) * c, -200.f);  // 2^-200 is 0, and so is that times -200
        const float e = exp2_fast(y);
        mine.s += e;
        mine.t = fmaf(e, y, mine.t);
      }
  }
#pragma unroll
  for (int d = 16; d; d /= 2) {
    Stats o;
    o.m = __shfl_xor_sync(~0u, mine.m, d);
    o.s = __shfl_xor_sync(~0u, mine.s, d);
    o.t = __shfl_xor_sync(~0u, mine.t, d);
    mine = joined(mine, o, c);
  }
  if (lane == 0) sh.stats[warp] = mine;
  if (threadIdx.x < 34) sh.count[threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.n = 0;
  cluster.barrier_wait(std::move(started));
  __syncthreads();
  if (threadIdx.x == 0) {
    Stats all = sh.stats[0];
    for (int w = 1; w < kScoreWarps; w++) all = joined(all, sh.stats[w], c);
    cluster.map_shared_rank(&sh, 0)->cluster_stats[rank] = all;
  }

  if (TOP) {
    const int n = chunk1 - chunk0, k = a.top;
    // The k first chunks: the k-th largest maximum bit by bit, then those above it and the first ones at it.
    unsigned threshold = 0;
    if (n > k) {
      for (int bit = 31; bit >= 0; bit--) {
        const unsigned t = threshold | (1u << bit);
        int m = 0;
        for (int i = threadIdx.x; i < n; i += kScoreThreads) m += chunk_key[i] >= t;
        if (block_count(m, &sh.count[bit]) >= k) threshold = t;
      }
      for (int i = threadIdx.x; i < n; i += kScoreThreads)
        if (chunk_key[i] > threshold) sh.chunk[atomicAdd(&sh.n, 1)] = i;
      __syncthreads();
      // The first warp walks the rest in order; it stops at k.
      if (warp == 0) {
        int have = sh.n;
        for (int i0 = 0; i0 < n && have < k; i0 += 32) {
          const unsigned same = __ballot_sync(~0u, i0 + lane < n && chunk_key[i0 + lane] == threshold);
          const int at = have + __popc(same & ((1u << lane) - 1));
          if ((same >> lane & 1) && at < k) sh.chunk[at] = i0 + lane;
          have += __popc(same);
        }
      }
    } else if ((int)threadIdx.x < n) {
      sh.chunk[threadIdx.x] = threadIdx.x;
    }
    __syncthreads();
    if (threadIdx.x < 34) sh.count[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    // Their elements at or above the threshold: k of them at least (or all there are), usually few more.
    const int read = min(n, k);
    constexpr int R = kScoreTopMax / kScoreWarps;
    unsigned key[R][V];
    int found = 0;
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int j = warp + r * kScoreWarps;
      float f[V];
      const int v = j < read ? (chunk0 + sh.chunk[j]) * 32 + lane : 0;
      if (j < read) load(v, f);
#pragma unroll
      for (int i = 0; i < V; i++) {
        const int p = v * V + i;
        key[r][i] = j < read && p >= shift && p < end ? order_key(f[i]) : 0u;
        found += key[r][i] != 0u && key[r][i] >= threshold;
      }
    }
    int all = block_count(found, &sh.count[32]);
    unsigned id_limit = 0xffffffffu;  // of the elements at the threshold only those up to this position
    if (all > kScoreCandidates) {
      // Too many at or above it (long ties, or values that crowd into few chunks): the k-th largest element itself, and
      // of those equal to it the first positions.
      auto count = [&](auto&& is, int* slot) {
        int m = 0;
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
          for (int i = 0; i < V; i++) {
            const int j = warp + r * kScoreWarps;
            if (key[r][i] && j < read) m += is(key[r][i], (unsigned)(((chunk0 + sh.chunk[j]) * 32 + lane) * V + i));
          }
        return block_count(m, slot);
      };
      unsigned kth = 0;
      for (int bit = 31; bit >= 0; bit--) {
        const unsigned t = kth | (1u << bit);
        if (count([&](unsigned x, unsigned) { return x >= t; }, &sh.count[bit]) >= k) kth = t;
      }
      threshold = kth;
      __syncthreads();
      if (threadIdx.x < 34) sh.count[threadIdx.x] = 0;
      __syncthreads();
      const int above = count([&](unsigned x, unsigned) { return x > kth; }, &sh.count[33]);
      // The (k - above)-th smallest position among the equal ones: the largest limit with fewer than that many below it.
      unsigned limit = 0;
      for (int bit = 31; bit >= 0; bit--) {
        const unsigned t = limit | (1u << bit);
        if (count([&](unsigned x, unsigned p) { return x == kth && p < t; }, &sh.count[bit]) < k - above) limit = t;
      }
      id_limit = limit;
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int j = warp + r * kScoreWarps;
#pragma unroll
      for (int i = 0; i < V; i++) {
        if (j >= read || key[r][i] == 0u || key[r][i] < threshold) continue;
        const unsigned p = (unsigned)(((chunk0 + sh.chunk[j]) * 32 + lane) * V + i);
        if (key[r][i] == threshold && p > id_limit) continue;
        const int at = atomicAdd(&sh.n, 1);
        sh.candidate[at] = (unsigned long long)key[r][i] << 32 | (0xffffffffu - (p - (unsigned)shift));
      }
    }
    __syncthreads();
    const int have = sh.n;
    unsigned long long* to = cluster.map_shared_rank(&sh, 0)->cluster_top + rank * kScoreTopMax;
    if ((int)threadIdx.x < have) {
      const unsigned long long x = sh.candidate[threadIdx.x];
      int before = 0;
      for (int i = 0; i < have; i++) before += sh.candidate[i] > x;
      if (before < k) to[before] = x;
    }
    if ((int)threadIdx.x >= have && (int)threadIdx.x < k) to[threadIdx.x] = 0;
  }
  cluster.sync();
  if (rank != 0) return;
  if (warp == 0 || TOP) {
    Stats all = sh.cluster_stats[0];
    for (int r = 1; r < ranks; r++) all = joined(all, sh.cluster_stats[r], c);
    // Nothing but -inf: S = 0, lse = -inf, log probabilities -inf, entropy 0.
    const float log_s = logf(all.s);
    const bool none = all.m == -INFINITY;
    const float top = all.m * a.scale;
    if (threadIdx.x == 0) {
      const int token = a.tokens[row];
      float given = 0.f;
      if (token >= 0) {
        if (token < a.vocab) {
          given = none ? -INFINITY : (Logit<T>::load(logits + token) - all.m) * a.scale - log_s;
        } else {
          given = __uint_as_float(0x7fffffffu);
          report(a.error_flag, kErrorToken);
        }
      }
      a.log_probs[row] = given;
      if (a.entropy) a.entropy[row] = none ? 0.f : log_s - all.t * kLn2 / all.s;
      if (a.lse) a.lse[row] = none ? -INFINITY : top + log_s;
    }
    if (TOP) {
      const int k = a.top, n = ranks * k;
      if ((int)threadIdx.x < n) {
        const unsigned long long x = sh.cluster_top[threadIdx.x / k * kScoreTopMax + threadIdx.x % k];
        int before = 0;
        if (ranks == 1) {
          before = threadIdx.x;
        } else {
          for (int i = 0; i < n; i++) before += sh.cluster_top[i / k * kScoreTopMax + i % k] > x;
        }
        if (before < k && x) {
          const float value = key_value((unsigned)(x >> 32));
          if (a.top_ids) a.top_ids[row * k + before] = (int)(0xffffffffu - (unsigned)x);
          if (a.top_log_probs) a.top_log_probs[row * k + before] = none ? -INFINITY : (value - all.m) * a.scale - log_s;
        }
      }
    }
  }
}

// ---- gradient ------------------------------------------------------------------------------------------------------

constexpr int kGradThreads = 256;
constexpr int kGradUnroll = 4;

template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(kGradThreads) token_score_grad_kernel(TokenScoreGrad a, int blocks_per_row) {
  constexpr int V = Logit<T>::V;
  PJRTX_PDL_PROLOGUE();
  const long long row = blockIdx.x / blocks_per_row;
  const int part = (int)(blockIdx.x - row * blocks_per_row);
  const T* logits = static_cast<const T*>(a.logits) + row * a.row_stride;
  T* grad = static_cast<T*>(a.grad_logits) + row * a.grad_row_stride;
  const int token = a.tokens[row];
  if (part == 0 && threadIdx.x == 0 && token >= a.vocab) report(a.error_flag, kErrorToken);
  const float lse = a.lse[row];
  const float g = token >= 0 && a.grad_log_probs ? a.grad_log_probs[row] * a.scale : 0.f;
  const float h = ENTROPY ? a.grad_entropy[row] * a.scale : 0.f, entropy = ENTROPY ? a.entropy[row] : 0.f;
  const bool none = lse == -INFINITY;
  // entropy - lse in two numbers, so that ln p + entropy, which is small where it matters, is rounded once.
  const float base = entropy - lse, part_of = base - entropy, rest = (entropy - (base - part_of)) + (-lse - part_of);
  // d = [j = token] g - p (g + h (ln p + entropy)); p = 0 gives 0 also where ln p = -inf.
  auto gradient = [&](float x, int j) {
    const float log_p = fmaf(x, a.scale, -lse);
    const float p = none ? 0.f : exp2_fast(log_p * kLog2e);
    float d = g;
    if (ENTROPY) d = p == 0.f ? g : fmaf(h, fmaf(x, a.scale, base) + rest, g);
    d = -p * d;
    return j == token ? d + g : d;
  };
  const int shift = (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(T));
  if (shift == (int)((reinterpret_cast<uintptr_t>(grad) & 15) / sizeof(T))) {
    const T* from = logits - shift;
    T* to = grad - shift;
    const int end = (int)a.vocab + shift, vectors = (end + V - 1) / V;
    const int step = blocks_per_row * kGradThreads;
    for (int v0 = part * kGradThreads + (int)threadIdx.x; v0 < vectors; v0 += step * kGradUnroll) {
      uint4 r[kGradUnroll];
#pragma unroll
      for (int u = 0; u < kGradUnroll; u++) {
        const int p = (v0 + u * step) * V;
        if (p >= shift && p + V <= end) r[u] = *reinterpret_cast<const uint4*>(from + p);
      }
#pragma unroll
      for (int u = 0; u < kGradUnroll; u++) {
        const int p = (v0 + u * step) * V;
        if (p >= shift && p + V <= end) {
          float f[V];
          Logit<T>::unpack(r[u], f);
#pragma unroll
          for (int i = 0; i < V; i++) f[i] = gradient(f[i], p + i - shift);
          *reinterpret_cast<uint4*>(to + p) = Logit<T>::pack(f);
        } else {
          for (int i = max(p, shift); i < min(p + V, end); i++) Logit<T>::store(to + i, gradient(Logit<T>::load(from + i), i - shift));
        }
      }
    }
  } else {
    for (long long j = part * kGradThreads + (int)threadIdx.x; j < a.vocab; j += blocks_per_row * kGradThreads)
      Logit<T>::store(grad + j, gradient(Logit<T>::load(logits + j), (int)j));
  }
}

template <typename T>
int score_launch(const TokenScore& s, int sm_count, bool pdl, cudaStream_t stream) {
  const int chunks = (int)((s.vocab + Logit<T>::V - 1 + Logit<T>::V - 1) / Logit<T>::V + 31) / 32;
  // A cluster for each row: as many blocks as fill the GPU twice, none with less than a load of every thread.
  int ranks = 1;
  while (ranks < kScoreClusterMax && s.rows * ranks < 2 * sm_count && chunks > ranks * kScoreWarps) ranks *= 2;
  const int segment = (chunks + ranks - 1) / ranks;
  const bool top = s.top > 0;
  const size_t smem = top ? (size_t)segment * sizeof(unsigned) : 0;
  auto kernel = top ? token_score_kernel<T, true> : token_score_kernel<T, false>;
  if (smem > 32 * 1024 && !raise_smem_limit((const void*)kernel, 200 * 1024)) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(s.rows * ranks));
  cfg.blockDim = dim3(kScoreThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[3];
  cfg.numAttrs = fill_launch_attributes(attr, pdl);
  attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
  attr[cfg.numAttrs].val.clusterDim = {(unsigned)ranks, 1, 1};
  cfg.numAttrs++;
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kernel, s, segment) == cudaSuccess;
}

template <typename T>
int grad_launch(const TokenScoreGrad& s, int sm_count, bool pdl, cudaStream_t stream) {
  const long long vectors = (s.vocab + Logit<T>::V - 1) / Logit<T>::V + 1;
  const long long per_row = std::max<long long>(1, (vectors + kGradThreads * kGradUnroll - 1) / (kGradThreads * kGradUnroll));
  auto kernel = s.grad_entropy ? token_score_grad_kernel<T, true> : token_score_grad_kernel<T, false>;
  return launch_kernel(kernel, dim3((unsigned)(s.rows * per_row)), dim3(kGradThreads), 0, stream, pdl, s, (int)per_row) == cudaSuccess;
}

}  // namespace

int token_score_launch(const TokenScore& s, int sm_count, bool pdl, cudaStream_t stream) {
  switch (s.dtype) {
    case kF32: return score_launch<float>(s, sm_count, pdl, stream);
    case kF16: return score_launch<__half>(s, sm_count, pdl, stream);
    default: return score_launch<__nv_bfloat16>(s, sm_count, pdl, stream);
  }
}

int token_score_grad_launch(const TokenScoreGrad& s, int sm_count, bool pdl, cudaStream_t stream) {
  switch (s.dtype) {
    case kF32: return grad_launch<float>(s, sm_count, pdl, stream);
    case kF16: return grad_launch<__half>(s, sm_count, pdl, stream);
    default: return grad_launch<__nv_bfloat16>(s, sm_count, pdl, stream);
  }
}

}  // namespace pjrtx
