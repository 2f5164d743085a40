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
// Top k is a tournament of intervals. A chunk is 256 consecutive logits, a vector the 16 bytes of one load, and in the order
// (value descending, id ascending) the k first elements lie in the k intervals that come first by (maximum descending,
// position ascending): an element of any other interval has k elements before it, the maxima of those. So chunk maxima are left
// in shared memory on the way, and afterwards the k first chunks are read again, then the k first of their vectors.
//
// Bound by memory, and where the logits are 16 bits wide nearly as much by the exponents' instructions: 4.5 a logit (two at a time).
// 4096 rows of 128256 bf16 logits (1.05 GB) take 166 us without alternatives, 185 with five, 161 at the rate of a copy; one row,
// 0.26 MB, 8 us of latencies. The gradient reads and writes each logit once: 2048 rows of 128256 f32 315 us (2.1 GB, 6.7 TB/s).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <utility>

#include "../common.h"
#include "arith.cuh"
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
  // The largest element of `count` vectors.
  template <int N>
  static __device__ __forceinline__ float highest(const uint4* r) {
    float m = max_nan(max_nan(__uint_as_float(r[0].x), __uint_as_float(r[0].y)), max_nan(__uint_as_float(r[0].z), __uint_as_float(r[0].w)));
    if constexpr (N > 1) m = max_nan(m, highest<N - 1>(r + 1));
    return m;
  }
  template <int N>
  static __device__ __forceinline__ float lowest(const uint4* r) {
    float m = fminf(fminf(__uint_as_float(r[0].x), __uint_as_float(r[0].y)), fminf(__uint_as_float(r[0].z), __uint_as_float(r[0].w)));
    if constexpr (N > 1) m = fminf(m, lowest<N - 1>(r + 1));
    return m;
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
  template <int N>
  static __device__ __forceinline__ __nv_bfloat162 extreme(const uint4* r, bool high) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(r);
    __nv_bfloat162 m = h[0];
#pragma unroll
    for (int i = 1; i < 4 * N; i++) m = high ? __hmax2_nan(m, h[i]) : __hmin2(m, h[i]);
    return m;
  }
  template <int N>
  static __device__ __forceinline__ float highest(const uint4* r) {
    const float2 m = __bfloat1622float2(extreme<N>(r, true));
    return max_nan(m.x, m.y);
  }
  template <int N>
  static __device__ __forceinline__ float lowest(const uint4* r) {
    const float2 m = __bfloat1622float2(extreme<N>(r, false));
    return fminf(m.x, m.y);
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
  template <int N>
  static __device__ __forceinline__ __half2 extreme(const uint4* r, bool high) {
    const __half2* h = reinterpret_cast<const __half2*>(r);
    __half2 m = h[0];
#pragma unroll
    for (int i = 1; i < 4 * N; i++) m = high ? __hmax2_nan(m, h[i]) : __hmin2(m, h[i]);
    return m;
  }
  template <int N>
  static __device__ __forceinline__ float highest(const uint4* r) {
    const float2 m = __half22float2(extreme<N>(r, true));
    return max_nan(m.x, m.y);
  }
  template <int N>
  static __device__ __forceinline__ float lowest(const uint4* r) {
    const float2 m = __half22float2(extreme<N>(r, false));
    return fminf(m.x, m.y);
  }
  static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
};

// A float in the order of unsigned integers: -0 as +0, NaN above all; 0 stands for "no element".
__device__ __forceinline__ unsigned order_key(float f) {
  if (f != f) return 0xffffffffu;
  const unsigned u = __float_as_uint(f == 0.f ? 0.f : f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(unsigned k) {
  return k == 0xffffffffu ? __uint_as_float(0x7fffffffu) : __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

// Running softmax statistics: exponents count in units of ln 2 and relative to `reference(m)`, the product rounded once, so
// that the exponent of a logit is one fused multiply-add. m = -inf: nothing but -inf so far.
struct Stats {
  float m, s, t;
};
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }
// The exponent of x under the maximum m. Where m * c overflows (a row of the type's lowest value), the difference comes first.
__device__ __forceinline__ float exponent(float x, float m, float c) {
  const float r = m * c;
  return finite(r) ? fmaf(x, c, -r) : (x - m) * c;
}
// What (s, t) of maximum a.m become under the maximum `to` >= a.m.
__device__ __forceinline__ void restate(Stats& a, float to, float c) {
  if (a.m == to) return;
  const float r = to * c, q = a.m * c;
  const float d = a.m == -INFINITY ? -INFINITY : finite(r) ? q - r : (a.m - to) * c;
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

// Threads of a block. Small ones where there are rows enough to fill the GPU with them: eight share an SM, so that what one row's
// alternatives wait for is hidden by seven others (4096 rows of 128256 bf16 logits, 5 alternatives: 185 us, 193 with four blocks of
// 256); where a cluster has one row, larger ones (one row: 8.7 us, 10.3 with 128). One warp, up to 32 of them an SM, for a row of
// a few batches, where the others of a block would have none: 4000 rows of 1024 7.0 us, 13.3 with 128 threads (5 alternatives 14.3,
// 26.0), of 4000 12.4 (18.8), of 5000 14.5 (22.2); but 20 alternatives of 5000 f32 logits 73 us, not 59, and with few rows, which
// would have had a block of 256 each, 5 alternatives of 1500 logits 8.1 us, not 6.3.
constexpr int kScoreThreadsMany = 128, kScoreThreadsFew = 256, kScoreThreadsShort = 32, kScoreThreadsOfSm = 1024;
constexpr int kScoreVectors = 4;  // 16-byte loads of a batch; the next batch's are in flight while one is added up
constexpr int kChunk = 256;       // logits
constexpr int kScoreClusterMax = 8;

// An element or interval in the order of the tournament: value first, lower position first among equal ones. 0: none.
typedef unsigned long long Entry;
__device__ __forceinline__ Entry entry(unsigned key, unsigned position) { return (Entry)key << 32 | (0xffffffffu - position); }
__device__ __forceinline__ unsigned position_of(Entry e) { return 0xffffffffu - (unsigned)e; }

__device__ __forceinline__ Entry max_entry(Entry a, Entry b) { return a > b ? a : b; }

// Places of a warp's entries among each other, N a lane, the largest first.
template <int N, typename E>
__device__ __forceinline__ void places(const E (&x)[N], int (&place)[N]) {
#pragma unroll
  for (int i = 0; i < N; i++) {
    place[i] = 0;
#pragma unroll
    for (int j = 0; j < N; j++) place[i] += x[j] > x[i];
  }
#pragma unroll
  for (int d = 1; d < 32; d++)
#pragma unroll
    for (int j = 0; j < N; j++) {
      const E y = __shfl_xor_sync(~0u, x[j], d);
#pragma unroll
      for (int i = 0; i < N; i++) place[i] += y > x[i];
    }
}

// The first k of the entries get(0..n-1), n <= 32 N, to out; 0 where there are fewer.
template <int N, typename Get>
__device__ __forceinline__ void select_few(Get&& get, int n, int k, Entry* out) {
  const int lane = threadIdx.x % 32;
  Entry x[N];
  int place[N], have = 0;
#pragma unroll
  for (int i = 0; i < N; i++) {
    x[i] = i * 32 + lane < n ? get(i * 32 + lane) : 0;
    have += __popc(__ballot_sync(~0u, x[i] != 0));
  }
  places(x, place);
#pragma unroll
  for (int i = 0; i < N; i++)
    if (x[i] && place[i] < k) out[place[i]] = x[i];
  for (int i = have + lane; i < k; i += 32) out[i] = 0;
}

constexpr int kFew = 64;

// The same for any n. One warp; `spare` has room for kFew entries.
template <typename Get>
__device__ __forceinline__ void select(Get&& get, int n, int k, Entry* out, Entry* spare) {
  const int lane = threadIdx.x % 32;
  if (n <= 32) return select_few<1>(get, n, k, out);
  if (n <= kFew) return select_few<2>(get, n, k, out);
  int count = kFew + 1;
  if (k <= 32) {
    // The k-th largest of 64 groups' maxima (a lane has two) is a lower bound; about 64 ln(64 / (64 - k)) entries reach it.
    unsigned best[2] = {0, 0};
    for (int i = lane; i < n; i += 64) {
      best[0] = max(best[0], (unsigned)(get(i) >> 32));
      if (i + 32 < n) best[1] = max(best[1], (unsigned)(get(i + 32) >> 32));
    }
    int place[2];
    places(best, place);  // equal maxima share the first of their places
    const unsigned low = min(place[0] < k ? best[0] : ~0u, place[1] < k ? best[1] : ~0u);
    const unsigned bound = __reduce_min_sync(~0u, low);
    count = 0;
    for (int i0 = 0; i0 < n && count <= kFew; i0 += 32) {
      const Entry x = i0 + lane < n ? get(i0 + lane) : 0;
      const bool in = x != 0 && (unsigned)(x >> 32) >= bound;
      const unsigned all = __ballot_sync(~0u, in);
      const int at = count + __popc(all & ((1u << lane) - 1));
      if (in && at < kFew) spare[at] = x;
      count += __popc(all);
    }
    __syncwarp();
  }
  if (count <= 32) return select_few<1>([&](int i) { return spare[i]; }, count, k, out);
  if (count <= kFew) return select_few<2>([&](int i) { return spare[i]; }, count, k, out);
  Entry limit = ~0ull;  // many equal ones, or a long list: one by one
  for (int j = 0; j < k; j++) {
    Entry x = 0;
    for (int i = lane; i < n; i += 32) {
      const Entry y = get(i);
      if (y < limit) x = max_entry(x, y);
    }
    const unsigned key = __reduce_max_sync(~0u, (unsigned)(x >> 32));
    const unsigned low = __reduce_max_sync(~0u, (unsigned)(x >> 32) == key ? (unsigned)x : 0u);
    limit = (Entry)key << 32 | low;
    if (lane == 0) out[j] = limit;
  }
}

template <int THREADS>
struct ScoreShared {
  static constexpr int kRanks = THREADS == kScoreThreadsShort ? 1 : kScoreClusterMax;
  Stats stats[THREADS / 32];
  Stats cluster_stats[kRanks];               // of the rank-0 block
  Entry cluster_top[kRanks * kScoreTopMax];  // of the rank-0 block
  Entry chosen[kScoreTopMax], spare[kFew];
  int n;
};

// Entries that the chosen chunks' vectors or the chosen vectors' elements take.
template <int V>
constexpr __host__ __device__ int score_room(int top, int chunks) {
  const int vectors = (top < chunks ? top : chunks) * (kChunk / V);
  return vectors > top * V ? vectors : top * V;
}

__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, kScoreThreadsOfSm / THREADS) token_score_kernel(TokenScore a, int segment_chunks) {
  constexpr int kScoreWarps = THREADS / 32;
  constexpr int V = Logit<T>::V;
  constexpr int kVectorsOfChunk = kChunk / (32 * V);              // 16-byte loads a thread has of a chunk
  constexpr int kChunks = kScoreVectors / kVectorsOfChunk;        // chunks of a batch
  extern __shared__ float chunk_max[];  // TOP: of this block's chunks
  Entry* list = reinterpret_cast<Entry*>(chunk_max + (segment_chunks + 1) / 2 * 2);  // TOP: of vectors, or elements, of the chosen ones
  __shared__ ScoreShared<THREADS> sh;
  PJRTX_PDL_PROLOGUE();
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  auto started = cluster.barrier_arrive();  // rank 0's shared memory is written once its block is known to run
  const long long row = blockIdx.x / ranks;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const T* logits = static_cast<const T*>(a.logits) + row * a.row_stride;
  // Vectors are 16-byte aligned: the row is elements [shift, end) of `aligned`.
  const int shift = (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(T));
  const T* aligned = logits - shift;
  const int end = (int)a.vocab + shift;
  const int chunks = (end + kChunk - 1) / kChunk;
  const int chunk0 = min(chunks, rank * segment_chunks), chunk1 = min(chunks, chunk0 + segment_chunks);
  const float c = a.scale * kLog2e;

  auto load = [&](int p) {  // the vector at element p; -inf outside the row
    if (p >= shift && p + V <= end) return *reinterpret_cast<const uint4*>(aligned + p);
    float f[V];
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = p + i >= shift && p + i < end ? Logit<T>::load(aligned + p + i) : -INFINITY;
    return Logit<T>::pack(f);
  };
  auto load_batch = [&](int k0, uint4 (&r)[kScoreVectors]) {
    const int p = k0 * kChunk + lane * V;
    if (k0 * kChunk >= shift && (k0 + kChunks) * kChunk <= end && k0 + kChunks <= chunk1) {
#pragma unroll
      for (int u = 0; u < kScoreVectors; u++) r[u] = *reinterpret_cast<const uint4*>(aligned + p + u * 32 * V);
    } else {
      const int stop = min(end, chunk1 * kChunk);
#pragma unroll
      for (int u = 0; u < kScoreVectors; u++) {
        if (p + u * 32 * V < stop) {
          r[u] = load(p + u * 32 * V);
        } else {
          float f[V];
#pragma unroll
          for (int i = 0; i < V; i++) f[i] = -INFINITY;
          r[u] = Logit<T>::pack(f);
        }
      }
    }
  };

  float m = -INFINITY, reference = -INFINITY;
  Pair s = pair_of(0.f, 0.f), t = pair_of(0.f, 0.f);
  uint4 next[kScoreVectors];
  const int step = kScoreWarps * kChunks;
  int k0 = chunk0 + warp * kChunks;
  if (k0 < chunk1) load_batch(k0, next);
  for (; k0 < chunk1; k0 += step) {
    uint4 r[kScoreVectors];
#pragma unroll
    for (int u = 0; u < kScoreVectors; u++) r[u] = next[u];
    if (k0 + step < chunk1) load_batch(k0 + step, next);
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kChunks; j++) {
      float high = Logit<T>::template highest<kVectorsOfChunk>(r + j * kVectorsOfChunk);
      if (TOP) {
        high = warp_max(high);
        if (lane == 0 && k0 + j < chunk1) chunk_max[k0 + j - chunk0] = high;
      }
      top = max_nan(top, high);
    }
    if (!(top <= m)) {
      const float2 s2 = pair_split(s), t2 = pair_split(t);
      Stats x = {m, s2.x, t2.x}, y = {m, s2.y, t2.y};
      restate(x, top, c);
      restate(y, top, c);
      s = pair_of(x.s, y.s);
      t = pair_of(x.t, y.t);
      m = top;
      reference = m * c;
    }
    // Every exponent is finite unless a logit is -inf (or near the lowest number there is).
    if (finite(reference) && fmaf(Logit<T>::template lowest<kScoreVectors>(r), c, -reference) > -INFINITY) {
      const Pair c2 = pair_of(c, c), from = pair_of(-reference, -reference);
#pragma unroll
      for (int u = 0; u < kScoreVectors; u++) {
        float f[V];
        Logit<T>::unpack(r[u], f);
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const Pair y = pair_fma(pair_of(f[i], f[i + 1]), c2, from);
          const float2 y2 = pair_split(y);
          const Pair e = pair_of(exp2_fast(y2.x), exp2_fast(y2.y));
          s = pair_add(s, e);
          t = pair_fma(e, y, t);
        }
      }
    } else if (m != -INFINITY) {
      float2 s2 = pair_split(s), t2 = pair_split(t);
#pragma unroll
      for (int u = 0; u < kScoreVectors; u++) {
        float f[V];
        Logit<T>::unpack(r[u], f);
#pragma unroll
        for (int i = 0; i < V; i++) {
          const float y = max_nan(exponent(f[i], m, c), -200.f);  // 2^-200 is 0, and so is that times -200
          const float e = exp2_fast(y);
          s2.x += e;
          t2.x = fmaf(e, y, t2.x);
        }
      }
      s = pair_of(s2.x, s2.y);
      t = pair_of(t2.x, t2.y);
    }
  }
  const float2 s2 = pair_split(s), t2 = pair_split(t);
  Stats mine = {m, s2.x + s2.y, t2.x + t2.y};
#pragma unroll
  for (int d = 16; d; d /= 2) {
    Stats o;
    o.m = __shfl_xor_sync(~0u, mine.m, d);
    o.s = __shfl_xor_sync(~0u, mine.s, d);
    o.t = __shfl_xor_sync(~0u, mine.t, d);
    mine = joined(mine, o, c);
  }
  if (lane == 0) sh.stats[warp] = mine;
  if (threadIdx.x == 0) sh.n = 0;
  cluster.barrier_wait(std::move(started));
  __syncthreads();
  if (warp == kScoreWarps - 1) {
    Stats all = lane < kScoreWarps ? sh.stats[lane] : Stats{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int d = kScoreWarps / 2; d; d /= 2) {
      Stats o;
      o.m = __shfl_xor_sync(~0u, all.m, d);
      o.s = __shfl_xor_sync(~0u, all.s, d);
      o.t = __shfl_xor_sync(~0u, all.t, d);
      all = joined(all, o, c);
    }
    if (lane == 0) cluster.map_shared_rank(&sh, 0)->cluster_stats[rank] = all;
  }

  if (TOP) {
    const int k = a.top, n = chunk1 - chunk0;
    if (warp == 0) select([&](int i) { return entry(order_key(chunk_max[i]), (unsigned)i); }, n, k, sh.chosen, sh.spare);
    __syncthreads();
    // What reaches the last of their maxima: elements at once where they are few, else vectors first and then theirs.
    const unsigned bound = n < k ? 0u : (unsigned)(sh.chosen[k - 1] >> 32);
    const int room = score_room<V>(k, segment_chunks);
    auto gather = [&](bool elements) {
      for (int j = warp; j < k && sh.chosen[j] != 0; j += kScoreWarps) {
        const int chunk = chunk0 + (int)position_of(sh.chosen[j]);
#pragma unroll
        for (int u = 0; u < kVectorsOfChunk; u++) {
          const int p = chunk * kChunk + (u * 32 + lane) * V;
          if (p >= end || p + V <= shift) continue;
          const uint4 r = load(p);
          const unsigned key = order_key(Logit<T>::template highest<1>(&r));
          if (key < bound) continue;
          if (!elements) {
            list[atomicAdd(&sh.n, 1)] = entry(key, (unsigned)p);
            continue;
          }
          float f[V];
          Logit<T>::unpack(r, f);
#pragma unroll
          for (int i = 0; i < V; i++) {
            const unsigned x = order_key(f[i]);
            if (x < bound || p + i < shift || p + i >= end) continue;
            const int at = atomicAdd(&sh.n, 1);
            if (at < room) list[at] = entry(x, (unsigned)(p + i - shift));
          }
        }
      }
    };
    const bool by_vectors = n < k && min(end, chunk1 * kChunk) - chunk0 * kChunk > room;  // fewer chunks than places: no bound
    if (!by_vectors) {
      gather(true);
      __syncthreads();
    }
    if (by_vectors || sh.n > room) {  // or long ties
      __syncthreads();
      if (threadIdx.x == 0) sh.n = 0;
      __syncthreads();
      gather(false);
      __syncthreads();
      const int vectors = sh.n;
      __syncthreads();
      if (threadIdx.x == 0) sh.n = 0;
      if (warp == 0) select([&](int i) { return list[i]; }, vectors, k, sh.chosen, sh.spare);
      __syncthreads();
      const unsigned limit = vectors < k ? 0u : (unsigned)(sh.chosen[k - 1] >> 32);
      for (int j = threadIdx.x; j < k && sh.chosen[j] != 0; j += THREADS) {
        const int p = (int)position_of(sh.chosen[j]);
        float f[V];
        Logit<T>::unpack(load(p), f);
#pragma unroll
        for (int i = 0; i < V; i++) {
          const unsigned key = order_key(f[i]);
          if (p + i >= shift && p + i < end && key >= limit) list[atomicAdd(&sh.n, 1)] = entry(key, (unsigned)(p + i - shift));
        }
      }
      __syncthreads();
    }
    if (warp == 0) select([&](int i) { return list[i]; }, sh.n, k, cluster.map_shared_rank(&sh, 0)->cluster_top + rank * k, sh.spare);
  }
  cluster.sync();
  if (rank != 0 || warp != 0) return;
  Stats all = sh.cluster_stats[0];
  for (int r = 1; r < ranks; r++) all = joined(all, sh.cluster_stats[r], c);
  // ln of the sum of e^(x - m): S counts from the rounded product m c. Nothing but -inf: S = 0, log probabilities and lse -inf.
  const float from = all.m * c, log_s = finite(from) ? logf(all.s) - fmaf(all.m, c, -from) * kLn2 : logf(all.s);
  const bool none = all.m == -INFINITY;
  if (lane == 0) {
    const int token = a.tokens[row];
    float given = 0.f;
    if (token >= 0) {
      if (token < a.vocab) {
        given = none ? -INFINITY : (Logit<T>::load(logits + token) - all.m) * a.scale - log_s;
      } else {
        given = __uint_as_float(0x7fffffffu);
        report(a.error_words, kErrorToken);
      }
    }
    a.log_probs[row] = given;
    if (a.entropy) a.entropy[row] = none ? 0.f : logf(all.s) - all.t * kLn2 / all.s;
    if (a.lse) a.lse[row] = none ? -INFINITY : all.m * a.scale + log_s;
  }
  if (TOP) {
    const int k = a.top;
    if (ranks > 1) select([&](int i) { return sh.cluster_top[i]; }, ranks * k, k, sh.chosen, sh.spare);
    __syncwarp();
    const Entry* best = ranks > 1 ? sh.chosen : sh.cluster_top;
    for (int j = lane; j < k; j += 32) {
      const float value = key_value((unsigned)(best[j] >> 32));
      if (a.top_ids) a.top_ids[row * k + j] = (int)position_of(best[j]);
      if (a.top_log_probs) a.top_log_probs[row * k + j] = none ? -INFINITY : (value - all.m) * a.scale - log_s;
    }
  }
}

// ---- gradient ------------------------------------------------------------------------------------------------------

// Four vectors a thread in flight, eight blocks an SM, both sides past the caches (nothing is read twice): 3111 rows of 128256 bf16
// logits with an entropy term 253 us, floor 244; with the caches and one logit at a time 317.
constexpr int kGradThreads = 128;
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
  if (part == 0 && threadIdx.x == 0 && token >= a.vocab) report(a.error_words, kErrorToken);
  const float lse = a.lse[row];
  const float g = token >= 0 && a.grad_log_probs ? a.grad_log_probs[row] * a.scale : 0.f;
  const float h = ENTROPY ? a.grad_entropy[row] * a.scale : 0.f, entropy = ENTROPY ? a.entropy[row] : 0.f;
  const bool none = lse == -INFINITY;  // nothing but -inf in the row: p = 0 everywhere
  // entropy - lse in two numbers, so that ln p + entropy, which is small where it matters, is rounded once.
  const float base = entropy - lse, part_of = base - entropy, rest = (entropy - (base - part_of)) + (-lse - part_of);
  // -p (g + h (ln p + entropy)), two logits at a time; what the token's own logit gets besides is added by the thread that has it.
  const Pair scale2 = pair_of(a.scale, a.scale), from2 = pair_of(none ? 0.f : -lse, none ? 0.f : -lse), log2e2 = pair_of(kLog2e, kLog2e);
  const Pair base2 = pair_of(base, base), rest2 = pair_of(rest, rest), g2 = pair_of(-g, -g), h2 = pair_of(-h, -h);
  auto gradient = [&](float& x0, float& x1) {
    const Pair x = pair_of(x0, x1);
    const float2 y = pair_split(pair_mul(pair_fma(x, scale2, from2), log2e2));
    const Pair p = pair_of(exp2_fast(y.x), exp2_fast(y.y));
    Pair d = g2;
    if (ENTROPY) {
      const float2 t = pair_split(pair_add(pair_fma(x, scale2, base2), rest2));
      // Finite, for p = 0 to make it 0; where p > 0, ln p is above -88 and the entropy is not negative.
      d = pair_fma(h2, pair_of(max_nan(t.x, -128.f), max_nan(t.y, -128.f)), g2);
    }
    const float2 r = pair_split(pair_mul(p, d));
    x0 = r.x;
    x1 = r.y;
  };
  auto single = [&](float x, int j) {
    float unused = 0.f;
    gradient(x, unused);
    return (none ? 0.f : x) + (j == token ? g : 0.f);
  };
  const int shift = (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(T));
  if (shift == (int)((reinterpret_cast<uintptr_t>(grad) & 15) / sizeof(T)) && !none) {
    const T* from = logits - shift;
    T* to = grad - shift;
    const int end = (int)a.vocab + shift, vectors = (end + V - 1) / V, own = token + shift;
    const int step = blocks_per_row * kGradThreads;
    for (int v0 = part * kGradThreads + (int)threadIdx.x; v0 < vectors; v0 += step * kGradUnroll) {
      uint4 r[kGradUnroll];
#pragma unroll
      for (int u = 0; u < kGradUnroll; u++) {
        const int p = (v0 + u * step) * V;
        if (p >= shift && p + V <= end) r[u] = __ldcs(reinterpret_cast<const uint4*>(from + p));
      }
#pragma unroll
      for (int u = 0; u < kGradUnroll; u++) {
        const int p = (v0 + u * step) * V;
        if (p >= shift && p + V <= end) {
          float f[V];
          Logit<T>::unpack(r[u], f);
#pragma unroll
          for (int i = 0; i < V; i += 2) gradient(f[i], f[i + 1]);
          if (own >= p && own < p + V) {
#pragma unroll
            for (int i = 0; i < V; i++)
              if (p + i == own) f[i] += g;
          }
          __stcs(reinterpret_cast<uint4*>(to + p), Logit<T>::pack(f));
        } else {
          for (int i = max(p, shift); i < min(p + V, end); i++) Logit<T>::store(to + i, single(Logit<T>::load(from + i), i - shift));
        }
      }
    }
  } else {
    for (long long j = part * kGradThreads + (int)threadIdx.x; j < a.vocab; j += blocks_per_row * kGradThreads)
      Logit<T>::store(grad + j, single(Logit<T>::load(logits + j), (int)j));
  }
}

template <typename T, int THREADS>
int score_launch_of(const TokenScore& s, int sm_count, bool pdl, cudaStream_t stream) {
  const int chunks = (int)((s.vocab + Logit<T>::V - 1 + kChunk - 1) / kChunk);
  // A cluster for each row: as many blocks as fit the GPU at once, none with less than a batch for every warp. A few more than fit
  // wait for the others to end: 150 rows of 32000 7.5 us by three blocks, 9.0 by four (600 of 592; with 20 alternatives 12.5 and
  // 17.4). Only long rows gain by it: 300 of 128256 23.2 us by two, 28.9 by one.
  const int batch_chunks = THREADS * kScoreVectors * Logit<T>::V / kChunk;
  const long long slots = (long long)kScoreThreadsOfSm / THREADS * sm_count;
  long long ranks = std::max<long long>(1, slots / s.rows);
  if ((ranks + 1) * s.rows <= slots + slots / 16 && chunks / (ranks + 1) >= 200) ranks++;
  ranks = std::min({ranks, (long long)ScoreShared<THREADS>::kRanks, (chunks + batch_chunks - 1ll) / batch_chunks});
  const int segment = (int)((chunks + ranks - 1) / ranks);
  const bool top = s.top > 0;
  const size_t smem = top ? score_room<Logit<T>::V>(s.top, segment) * sizeof(Entry) + (size_t)(segment + 1) / 2 * sizeof(Entry) : 0;
  auto kernel = top ? token_score_kernel<T, true, THREADS> : token_score_kernel<T, false, THREADS>;
  if (smem > 32 * 1024 && !raise_smem_limit((const void*)kernel, 200 * 1024)) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(s.rows * ranks));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[3];
  cfg.numAttrs = fill_launch_attributes(attr, pdl);
  if (ranks > 1) {  // a cluster of one starts slower: 4000 rows of 1024 17.5 us, without 13.3
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim = {(unsigned)ranks, 1, 1};
    cfg.numAttrs++;
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kernel, s, segment) == cudaSuccess;
}

template <typename T>
int score_launch(const TokenScore& s, int sm_count, bool pdl, cudaStream_t stream) {
  const long long chunks = (s.vocab + Logit<T>::V - 1 + kChunk - 1) / kChunk;
  if (chunks <= (s.rows * kScoreThreadsFew < (long long)kScoreThreadsOfSm * sm_count ? 5 : s.top > 8 ? 16 : 24))
    return score_launch_of<T, kScoreThreadsShort>(s, sm_count, pdl, stream);
  return s.rows * kScoreThreadsMany >= (long long)kScoreThreadsOfSm * sm_count ? score_launch_of<T, kScoreThreadsMany>(s, sm_count, pdl, stream)
                                                                               : score_launch_of<T, kScoreThreadsFew>(s, sm_count, pdl, stream);
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
