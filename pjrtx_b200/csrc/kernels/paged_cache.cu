// Writing into a paged key-value cache and cutting it back.
//
// append: row t of the new ones of sequence b becomes row lengths[b] - counts[b] + t of its pages. Pure copying: every row is
// read once and written once, 16 bytes a thread, the threads of a warp on neighbouring pieces of one row.
//
// evict: of the n > keep rows of a (sequence, KV head) those stay that come first by (protected, weight descending, row
// ascending), a row being protected when its token is among the first `sinks` or the last `recent`. Attention does not depend
// on the order of its rows, so nothing is compacted: the i-th kept row at or beyond `keep` moves into the i-th dropped place
// before it, and only those rows are read and written. The token of each row is kept beside it in `positions`.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../common.h"
#include "kernels.h"
#include "paged.cuh"

namespace pjrtx {

namespace {

// ---- append --------------------------------------------------------------------------------------------------------

constexpr int kAppendThreads = 256;

__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(PagedView c, PagedAppend a, int pieces, int esize) {
  PJRTX_PDL_PROLOGUE();
  const int b = blockIdx.y;
  const int length = paged_length(c, b);
  int count = a.counts ? a.counts[b] : (int)a.rows;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    paged_check_length(c, b);
    if (count < 0 || count > a.rows || count > length) report(c.error_flag, kErrorLength);
  }
  count = max(0, min(count, min((int)a.rows, length)));
  const int first = length - count;
  const int per_row = c.kv_heads * pieces;  // 16-byte pieces of a row, all heads
  const long long total = (long long)count * per_row;
  const long long step = (long long)gridDim.x * kAppendThreads;
  for (long long i = (long long)blockIdx.x * kAppendThreads + threadIdx.x; i < total; i += step) {
    const int t = (int)(i / per_row), r = (int)(i - (long long)t * per_row);
    const int g = r / pieces, piece = r - g * pieces;
    const long long row = paged_row(c, b, first + t);
    if (row < 0) continue;
    const long long from = (b * a.batch_stride + t * a.row_stride + g * a.head_stride) * esize + piece * 16;
    const long long to = (row + g * c.head_stride) * esize + piece * 16;
    const uint4 k = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.k_new) + from);
    const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.v_new) + from);
    *reinterpret_cast<uint4*>(static_cast<char*>(c.k) + to) = k;
    *reinterpret_cast<uint4*>(static_cast<char*>(c.v) + to) = v;
  }
  if (!c.weights) return;
  const int token = c.tokens[b] - count;
  const long long capacity = (long long)c.page_size * c.max_pages;
  for (long long i = (long long)blockIdx.x * kAppendThreads + threadIdx.x; i < (long long)count * c.kv_heads; i += step) {
    const int g = (int)(i / count), t = (int)(i - (long long)g * count);
    const long long at = ((long long)b * c.kv_heads + g) * capacity + first + t;
    c.weights[at] = 0.f;
    c.positions[at] = token + t;
  }
}

// ---- evict ---------------------------------------------------------------------------------------------------------

constexpr int kSelectThreads = 1024, kSelectWarps = kSelectThreads / 32;
constexpr int kMoveThreads = 256;

// Weights in the order of unsigned integers: -0 as +0, NaN above all numbers, protected rows above NaN.
__device__ __forceinline__ unsigned weight_key(float w, bool is_protected) {
  if (is_protected) return 0xffffffffu;
  if (w != w) return 0xfffffffeu;
  const unsigned u = __float_as_uint(w == 0.f ? 0.f : w);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Copies the K and V rows of slot `from` to slot `to` of KV head g, one 16-byte piece of each per thread.
__device__ __forceinline__ void move_row(const PagedView& c, int b, int g, int from, int to, int piece, int esize) {
  const long long s = paged_row(c, b, from), d = paged_row(c, b, to);
  if (s < 0 || d < 0) return;
  const long long sa = (s + g * c.head_stride) * esize + piece * 16, da = (d + g * c.head_stride) * esize + piece * 16;
  const uint4 k = *reinterpret_cast<const uint4*>(static_cast<const char*>(c.k) + sa);
  const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const char*>(c.v) + sa);
  *reinterpret_cast<uint4*>(static_cast<char*>(c.k) + da) = k;
  *reinterpret_cast<uint4*>(static_cast<char*>(c.v) + da) = v;
}

// Workspace of evict: per sequence an arrival counter, per (sequence, KV head) the number of moves, then the moves.
struct EvictSpace {
  unsigned* arrivals;  // [batch]
  int* moves;          // [batch * kv_heads]
  int2* list;          // [batch * kv_heads][list_max] (from, to)
  long long list_max;
};

__host__ __device__ inline long long evict_list_max(const PagedView& c) { return (long long)c.page_size * c.max_pages / 2 + 1; }

// Places go by the largest batch, so that the counters stay where they are.
inline EvictSpace evict_space(const PagedView& c, void* workspace) {
  EvictSpace s;
  const uint64_t head = ((uint64_t)c.batch_max * 4 + 255) / 256 * 256, counts = ((uint64_t)c.batch_max * c.kv_heads * 4 + 255) / 256 * 256;
  char* p = static_cast<char*>(workspace);
  s.arrivals = reinterpret_cast<unsigned*>(p);
  s.moves = reinterpret_cast<int*>(p + head);
  s.list = reinterpret_cast<int2*>(p + head + counts);
  s.list_max = evict_list_max(c);
  return s;
}

// Block-wide exclusive prefix over the warps of one value per warp; `total` gets the sum. All threads call it.
__device__ __forceinline__ int warp_prefix(int value, int* buffer, int* total) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  __syncthreads();
  if (lane == 0) buffer[warp] = value;
  __syncthreads();
  int v = buffer[lane < kSelectWarps ? lane : 0], sum = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int o = __shfl_up_sync(~0u, sum, d);
    if (lane >= d) sum += o;
  }
  *total = __shfl_sync(~0u, sum, 31);
  return __shfl_sync(~0u, sum - v, warp);
}

// One block per (sequence, KV head). The threshold - the keep-th largest key - is found two bits at a time by counting the keys
// at or above three candidates; a warp owns a contiguous range of rows, so ranks within it are ballots and one prefix over
// the warps orders the rest.
__global__ void __launch_bounds__(kSelectThreads) paged_evict_select_kernel(PagedView c, PagedEvict e, EvictSpace space, int pieces,
                                                                            int esize, int keys_in_smem, int move_here) {
  extern __shared__ unsigned keys[];
  __shared__ int buffer[kSelectWarps];
  __shared__ int counts[16][4];
  __shared__ int last;
  PJRTX_PDL_PROLOGUE();
  const int g = blockIdx.x, b = blockIdx.y;
  const int pair = b * c.kv_heads + g;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int capacity = c.page_size * c.max_pages;
  const int n = paged_length(c, b), keep = e.keep;
  const long long base = (long long)pair * capacity;
  const float* weights = c.weights + base;
  const int* positions = c.positions + base;
  float* weights_out = e.weights_out + base;
  int* positions_out = e.positions_out + base;
  const int left = min(n, keep);
  if (threadIdx.x == 0) paged_check_length(c, b);
  int moves = 0;
  if (n > keep) {
    const int newest = c.tokens[b] - e.recent;
    auto key_of = [&](int t) {
      const int p = positions[t];
      return weight_key(weights[t], p < e.sinks || p >= newest);
    };
    if (threadIdx.x < 64) counts[threadIdx.x / 4][threadIdx.x % 4] = 0;
    if (keys_in_smem)
      for (int t = threadIdx.x; t < n; t += kSelectThreads) keys[t] = key_of(t);
    auto key_at = [&](int t) { return keys_in_smem ? keys[t] : key_of(t); };
    __syncthreads();
    unsigned threshold = 0;
    for (int step = 0; step < 16; step++) {
      const int shift = 30 - 2 * step;
      const unsigned c1 = threshold | (1u << shift), c2 = threshold | (2u << shift), c3 = threshold | (3u << shift);
      int n1 = 0, n2 = 0, n3 = 0;
      for (int t = threadIdx.x; t < n; t += kSelectThreads) {
        const unsigned k = key_at(t);
        n1 += k >= c1;
        n2 += k >= c2;
        n3 += k >= c3;
      }
      n1 = __reduce_add_sync(~0u, n1);
      n2 = __reduce_add_sync(~0u, n2);
      n3 = __reduce_add_sync(~0u, n3);
      if (lane == 0) {
        atomicAdd(&counts[step][1], n1);
        atomicAdd(&counts[step][2], n2);
        atomicAdd(&counts[step][3], n3);
      }
      __syncthreads();
      threshold = counts[step][3] >= keep ? c3 : counts[step][2] >= keep ? c2 : counts[step][1] >= keep ? c1 : threshold;
    }
    // Rows above the threshold stay, and of those at it the first ones.
    const int range = ((n + kSelectWarps - 1) / kSelectWarps + 31) / 32 * 32;
    const int begin = min(n, warp * range), end = min(n, begin + range);
    int above = 0, equal = 0;
    for (int t0 = begin; t0 < end; t0 += 32) {
      const unsigned k = t0 + lane < end ? key_at(t0 + lane) : 0u;
      const bool in = t0 + lane < end;
      above += __popc(__ballot_sync(~0u, in && k > threshold));
      equal += __popc(__ballot_sync(~0u, in && k == threshold));
    }
    int all_above, ignored;
    warp_prefix(above, buffer, &all_above);
    const int equal_before = warp_prefix(equal, buffer, &ignored);
    const int equal_kept = keep - all_above;
    auto walk = [&](auto&& row) {  // row(t, kept, ballot of dropped rows before `keep`, ballot of kept rows from `keep` on)
      int rank = equal_before;
      for (int t0 = begin; t0 < end; t0 += 32) {
        const int t = t0 + lane;
        const bool in = t < end;
        const unsigned k = in ? key_at(t) : 0u;
        const unsigned same = __ballot_sync(~0u, in && k == threshold);
        const bool kept = in && (k > threshold || (k == threshold && rank + __popc(same & ((1u << lane) - 1)) < equal_kept));
        rank += __popc(same);
        const unsigned hole = __ballot_sync(~0u, in && !kept && t < keep), source = __ballot_sync(~0u, kept && t >= keep);
        row(t, kept, hole, source);
      }
    };
    int holes = 0, sources = 0;
    walk([&](int, bool, unsigned hole, unsigned source) {
      holes += __popc(hole);
      sources += __popc(source);
    });
    int hole_at = warp_prefix(holes, buffer, &moves);
    int source_at = warp_prefix(sources, buffer, &ignored);
    int2* list = space.list + pair * space.list_max;
    walk([&](int t, bool kept, unsigned hole, unsigned source) {
      const unsigned before = (1u << lane) - 1;
      if (hole >> lane & 1) list[hole_at + __popc(hole & before)].y = t;
      if (source >> lane & 1) list[source_at + __popc(source & before)].x = t;
      if (kept && t < keep) {
        const float w = weights[t];
        const int p = positions[t];
        weights_out[t] = w;
        positions_out[t] = p;
      }
      hole_at += __popc(hole);
      source_at += __popc(source);
    });
    __syncthreads();
    for (int i = threadIdx.x; i < moves; i += kSelectThreads) {
      const int2 m = list[i];
      const float w = weights[m.x];
      const int p = positions[m.x];
      weights_out[m.y] = w;
      positions_out[m.y] = p;
    }
    if (move_here)
      for (long long i = threadIdx.x; i < (long long)moves * pieces; i += kSelectThreads) {
        const int2 m = list[i / pieces];
        move_row(c, b, g, m.x, m.y, (int)(i % pieces), esize);
      }
    __syncthreads();
  } else {
    for (int t = threadIdx.x; t < n; t += kSelectThreads) {
      const float w = weights[t];
      const int p = positions[t];
      weights_out[t] = w;
      positions_out[t] = p;
    }
  }
  for (int t = left + threadIdx.x; t < capacity; t += kSelectThreads) {
    weights_out[t] = 0.f;
    positions_out[t] = -1;
  }
  // The new length may take the old one's place, so it is written when every KV head's block has read that.
  if (threadIdx.x == 0) {
    space.moves[pair] = moves;
    __threadfence();
    last = atomicInc(&space.arrivals[b], (unsigned)c.kv_heads - 1) == (unsigned)c.kv_heads - 1;
    if (last) e.lengths_out[b] = left;
  }
}

// The rows of all moves, a group of `pieces` threads a row.
__global__ void __launch_bounds__(kMoveThreads) paged_evict_move_kernel(PagedView c, EvictSpace space, int pieces, int esize) {
  PJRTX_PDL_PROLOGUE();
  const int g = blockIdx.y, b = blockIdx.z;
  const int pair = b * c.kv_heads + g;
  const long long total = (long long)space.moves[pair] * pieces;
  const int2* list = space.list + pair * space.list_max;
  for (long long i = (long long)blockIdx.x * kMoveThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kMoveThreads) {
    const int2 m = list[i / pieces];
    move_row(c, b, g, m.x, m.y, (int)(i % pieces), esize);
  }
}

}  // namespace

int paged_append_launch(const PagedView& c, const PagedAppend& a, bool pdl, cudaStream_t stream) {
  const int esize = (int)dtype_size(c.dtype), pieces = c.head_dim * esize / 16;
  const long long work = a.rows * c.kv_heads * pieces;
  const long long blocks = std::min<long long>((work + kAppendThreads - 1) / kAppendThreads, 1024);
  return launch_kernel(paged_append_kernel, dim3((unsigned)std::max<long long>(blocks, 1), (unsigned)c.batch), dim3(kAppendThreads), 0,
                       stream, pdl, c, a, pieces, esize) == cudaSuccess;
}

uint64_t paged_evict_workspace_bytes(const PagedView& c) {
  const uint64_t head = ((uint64_t)c.batch_max * 4 + 255) / 256 * 256, counts = ((uint64_t)c.batch_max * c.kv_heads * 4 + 255) / 256 * 256;
  return head + counts + (uint64_t)c.batch_max * c.kv_heads * evict_list_max(c) * sizeof(int2);
}

int paged_evict_launch(const PagedView& c, const PagedEvict& e, int sm_count, bool pdl, cudaStream_t stream) {
  const int esize = (int)dtype_size(c.dtype), pieces = c.head_dim * esize / 16;
  const EvictSpace space = evict_space(c, e.workspace);
  const long long capacity = c.capacity();
  constexpr int kKeyBytesMax = 192 * 1024;
  const int in_smem = capacity * 4 <= kKeyBytesMax;
  if (!raise_smem_limit((const void*)paged_evict_select_kernel, kKeyBytesMax)) return 0;
  const long long moves_max = std::min<long long>(e.keep, capacity - e.keep);
  const int move_here = moves_max <= 64;
  if (launch_kernel(paged_evict_select_kernel, dim3((unsigned)c.kv_heads, (unsigned)c.batch), dim3(kSelectThreads),
                    in_smem ? (size_t)capacity * 4 : 0, stream, pdl, c, e, space, pieces, esize, in_smem, move_here) != cudaSuccess)
    return 0;
  if (move_here || moves_max <= 0) return 1;
  const long long pairs = (long long)c.batch * c.kv_heads;
  const long long blocks = std::max<long long>(1, std::min((moves_max * pieces + kMoveThreads - 1) / kMoveThreads, 8ll * sm_count / pairs + 1));
  if (launch_kernel(paged_evict_move_kernel, dim3((unsigned)blocks, (unsigned)c.kv_heads, (unsigned)c.batch), dim3(kMoveThreads), 0, stream,
                    true, c, space, pieces, esize) != cudaSuccess)
    return 0;
  return 2;
}

}  // namespace pjrtx
