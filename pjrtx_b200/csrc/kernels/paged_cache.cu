// Writing into a paged key-value cache and cutting it back.
//
// append: row t of the new ones of sequence b becomes row lengths[b] - counts[b] + t of its pages. Pure copying: every row is
// read once and written once, 16 bytes a thread, the threads of a warp on neighbouring pieces of one row. Bound by memory: 319 MB
// in 52.7 us (floor 48.7); 4 prompts up to 2048 rows of 8 heads of 128 in bf16, 51 MB, in 11.2.
//
// evict: of the n > keep rows of a (sequence, KV head) those stay that come first by (protected, weight descending, row
// ascending), a row being protected when its token is among the first `sinks` or the last `recent`. Attention does not depend
// on the order of its rows, so nothing is compacted: the i-th kept row at or beyond `keep` moves into the i-th dropped place
// before it, and only those rows are read and written. The token of each row is kept beside it in `positions`. Bound by what a
// block waits for until the moves are known (8 pairs of 2049 rows, one over: 9.2 us in all), then by rows of 256 bytes in no order:
// 128 pairs up to 4096 rows cut to 2048 (73 MB) 27.7 us, 14 of them moving.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../common.h"
#include "kernels.h"
#include "paged.cuh"

namespace pjrtx {

namespace {

// ---- append --------------------------------------------------------------------------------------------------------

// One piece of a key and of its value in flight a thread, and at most 64 blocks an SM for all sequences, which go on to further
// pieces: up to 8177 rows of 57 sequences, 2 heads of 64 in bf16 (319 MB), 52.7 us, with 16 an SM 55.7, with a block for every 256 pieces 58.8 (floor 48.7).
constexpr int kAppendThreads = 256;

__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(PagedView c, PagedAppend a, int pieces, int esize) {
  PJRTX_PDL_PROLOGUE();
  const int b = blockIdx.y;
  const int length = paged_length(c, b);
  int count = a.counts ? a.counts[b] : (int)a.rows;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    paged_check_length(c, b);
    if (count < 0 || count > a.rows || count > length) report(c.error_words, kErrorLength);
  }
  count = max(0, min(count, min((int)a.rows, length)));
  const int first = length - count;
  const int per_row = c.kv_heads * pieces;  // 16-byte pieces of a row, all heads
  const long long total = (long long)count * per_row;
  const long long step = (long long)gridDim.x * kAppendThreads;
  for (long long i = (long long)blockIdx.x * kAppendThreads + threadIdx.x; i < total; i += step) {
    const int t = total >> 31 ? (int)(i / per_row) : (int)((unsigned)i / (unsigned)per_row), r = (int)(i - (long long)t * per_row);
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
// Up to so many moves a pair its own block makes them: a second launch takes longer (87 at most: 12.7 us against 13.6).
constexpr int kMoveHere = 256;
constexpr int kMoveBatch = 512;

// Weights in the order of unsigned integers: -0 as +0, NaN above all numbers, protected rows above NaN.
__device__ __forceinline__ unsigned weight_key(float w, bool is_protected) {
  if (is_protected) return 0xffffffffu;
  if (w != w) return 0xfffffffeu;
  const unsigned u = __float_as_uint(w == 0.f ? 0.f : w);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Where a row moves from and to, as byte offsets of its KV head's elements in either pool; to < 0: one of the two has no page.
struct Move {
  long long from, to;
};

// 32 rows: which of them stay, and how many dropped rows before `keep` and kept rows from `keep` on there are before them.
struct Word {
  unsigned kept;
  int holes, sources;
};

// Workspace of evict: per sequence an arrival counter, per (sequence, KV head) the number of moves, then the moves.
struct EvictSpace {
  unsigned* arrivals;  // [batch]
  int* moves;          // [batch * kv_heads]
  Move* list;          // [batch * kv_heads][list_max]
  Word* words;         // [batch * kv_heads][words_max], where shared memory does not hold them
  long long list_max, words_max;
};

// Rows whose keys, and their words, a block has in shared memory.
constexpr long long kRowsInShared = 40 * 1024;

struct EvictLayout {
  uint64_t moves, list, words, bytes;
  long long list_max, words_max;
};

// Places go by the largest batch, so that the counters stay where they are.
inline EvictLayout evict_layout(const PagedView& c) {
  EvictLayout l;
  const uint64_t pairs = (uint64_t)c.batch_max * c.kv_heads;
  l.list_max = c.capacity() / 2 + 1;
  l.words_max = c.capacity() > kRowsInShared ? c.capacity() / 32 + 1 : 0;
  l.moves = ((uint64_t)c.batch_max * 4 + 255) / 256 * 256;
  l.list = l.moves + (pairs * 4 + 255) / 256 * 256;
  l.words = l.list + pairs * l.list_max * sizeof(Move);
  l.bytes = l.words + pairs * l.words_max * sizeof(Word);
  return l;
}

inline EvictSpace evict_space(const PagedView& c, void* workspace) {
  const EvictLayout l = evict_layout(c);
  char* p = static_cast<char*>(workspace);
  return {reinterpret_cast<unsigned*>(p), reinterpret_cast<int*>(p + l.moves), reinterpret_cast<Move*>(p + l.list),
          reinterpret_cast<Word*>(p + l.words), l.list_max, l.words_max};
}

// Copies the rows of moves 0..count-1, `lanes` (a power of two) threads a row, kMoveUnroll rows of each in flight.
constexpr int kMoveUnroll = 4;
__device__ __forceinline__ void move_rows(const PagedView& c, const Move* list, int count, int pieces, int lanes, int first, int step) {
  const int piece = threadIdx.x & (lanes - 1);
  if (piece >= pieces) return;
  for (int i0 = first; i0 < count; i0 += step * kMoveUnroll) {
    Move m[kMoveUnroll];
    uint4 k[kMoveUnroll], v[kMoveUnroll];
#pragma unroll
    for (int u = 0; u < kMoveUnroll; u++) {
      m[u].to = -1;
      if (i0 + u * step < count) m[u] = list[i0 + u * step];
    }
#pragma unroll
    for (int u = 0; u < kMoveUnroll; u++)
      if (m[u].to >= 0) {
        k[u] = *reinterpret_cast<const uint4*>(static_cast<const char*>(c.k) + m[u].from + piece * 16);
        v[u] = *reinterpret_cast<const uint4*>(static_cast<const char*>(c.v) + m[u].from + piece * 16);
      }
#pragma unroll
    for (int u = 0; u < kMoveUnroll; u++)
      if (m[u].to >= 0) {
        *reinterpret_cast<uint4*>(static_cast<char*>(c.k) + m[u].to + piece * 16) = k[u];
        *reinterpret_cast<uint4*>(static_cast<char*>(c.v) + m[u].to + piece * 16) = v[u];
      }
  }
}

// Exclusive sums of two values over the threads of the block, and the totals. One barrier; `step` alternates between calls, so
// that a buffer is written again only behind the next one.
struct Sums {
  int2 buffer[2][kSelectWarps];
};
struct Before {
  int a, b, all_a, all_b;
};
__device__ __forceinline__ Before block_before(Sums& s, int& step, int a, int b) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int x = a, y = b;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int u = __shfl_up_sync(~0u, x, d), v = __shfl_up_sync(~0u, y, d);
    if (lane >= d) {
      x += u;
      y += v;
    }
  }
  int2* buffer = s.buffer[step++ & 1];
  if (lane == 31) buffer[warp] = make_int2(x, y);
  __syncthreads();
  const int2 v = buffer[lane];
  Before r;
  r.all_a = __reduce_add_sync(~0u, v.x);
  r.all_b = __reduce_add_sync(~0u, v.y);
  r.a = x - a + __reduce_add_sync(~0u, lane < warp ? v.x : 0);
  r.b = y - b + __reduce_add_sync(~0u, lane < warp ? v.y : 0);
  return r;
}
static_assert(kSelectWarps == 32, "a lane for every warp");

constexpr int kDigitBits = 11;

struct SelectShared {
  union {
    int histogram[1 << kDigitBits];
    Move moves[kMoveBatch];  // when the threshold is known
  };
  Sums sums;
  int digit, need;
};

// One block per (sequence, KV head). The threshold - the keep-th largest key - comes from three histograms of 11, 11 and 10 bits,
// each over the keys that share the digits found so far. Then every 32 rows become a word of bits, the words' counts are added
// up by a thread each, and the rows that move are listed by a warp a word.
__global__ void __launch_bounds__(kSelectThreads) paged_evict_select_kernel(PagedView c, PagedEvict e, EvictSpace space, int pieces,
                                                                            int lanes, int esize, int in_shared, int move_here) {
  extern __shared__ unsigned keys[];
  __shared__ SelectShared sh;
  for (int i = threadIdx.x; i < 1 << kDigitBits; i += kSelectThreads) sh.histogram[i] = 0;
  __syncthreads();
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
    auto key_of = [&](float w, int p) { return weight_key(w, p < e.sinks || p >= newest); };
    auto key_at = [&](int t) { return in_shared ? keys[t] : key_of(weights[t], positions[t]); };
    if (in_shared) {
      constexpr int U = 8;
      for (int t0 = threadIdx.x; t0 < n; t0 += U * kSelectThreads) {
        float w[U];
        int p[U];
#pragma unroll
        for (int u = 0; u < U; u++)
          if (t0 + u * kSelectThreads < n) {
            w[u] = weights[t0 + u * kSelectThreads];
            p[u] = positions[t0 + u * kSelectThreads];
          }
#pragma unroll
        for (int u = 0; u < U; u++)
          if (t0 + u * kSelectThreads < n) {
            const unsigned k = key_of(w[u], p[u]);
            keys[t0 + u * kSelectThreads] = k;
            atomicAdd(&sh.histogram[k >> (32 - kDigitBits)], 1);
          }
      }
    }
    unsigned threshold = 0;  // its digits so far
    int need = keep, step = 0;  // how many of the keys that share them stay
    for (int shift = 32, bits = kDigitBits; shift > 0;) {
      bits = min(kDigitBits, shift);
      shift -= bits;
      const int size = 1 << bits;
      const bool first_digit = shift + bits == 32;
      if (!first_digit || !in_shared) {
#pragma unroll 4
        for (int t = threadIdx.x; t < n; t += kSelectThreads) {
          const unsigned k = key_at(t);
          if (first_digit || k >> (shift + bits) == threshold) atomicAdd(&sh.histogram[k >> shift & (size - 1)], 1);
        }
      }
      __syncthreads();
      const int high = size - 1 - 2 * (int)threadIdx.x;  // two digits a thread, the largest ones first
      int at_high = 0, at_low = 0;
      if (high > 0) {
        at_high = sh.histogram[high];
        at_low = sh.histogram[high - 1];
        sh.histogram[high] = sh.histogram[high - 1] = 0;  // for the next digit
      }
      const int before = block_before(sh.sums, step, at_high + at_low, 0).a;
      if (before < need && need <= before + at_high + at_low) {
        const bool first = need <= before + at_high;
        sh.digit = first ? high : high - 1;
        sh.need = need - before - (first ? 0 : at_high);
      }
      __syncthreads();
      threshold = threshold << bits | (unsigned)sh.digit;
      need = sh.need;
    }
    // Rows above the threshold stay, and of those at it the first `need`.
    const int words = (n + 31) / 32;
    Word* word = in_shared ? reinterpret_cast<Word*>(keys + (capacity + 3) / 4 * 4) : space.words + pair * space.words_max;
#pragma unroll 4
    for (int i = warp; i < words; i += kSelectWarps) {
      const int t = i * 32 + lane;
      const unsigned k = t < n ? key_at(t) : 0u;
      const unsigned above = __ballot_sync(~0u, t < n && k > threshold), equal = __ballot_sync(~0u, t < n && k == threshold);
      if (lane == 0) {
        word[i].kept = above;
        word[i].holes = (int)equal;
      }
    }
    __syncthreads();
    int equals = 0, holes = 0, sources = 0;  // of the words so far
    for (int i0 = 0; i0 < words; i0 += kSelectThreads) {
      const int i = i0 + (int)threadIdx.x;
      unsigned kept = 0, equal = 0;
      if (i < words) {
        kept = word[i].kept;
        equal = (unsigned)word[i].holes;
      }
      const Before same = block_before(sh.sums, step, __popc(equal), 0);
      int room = need - equals - same.a;
      for (; equal && room > 0; room--) {
        kept |= equal & -equal;
        equal &= equal - 1;
      }
      const int first = i * 32;
      const unsigned in = first >= n ? 0u : n - first >= 32 ? ~0u : (1u << (n - first)) - 1;
      const unsigned front = first >= keep ? 0u : keep - first >= 32 ? ~0u : (1u << (keep - first)) - 1;
      const Before listed = block_before(sh.sums, step, __popc(~kept & in & front), __popc(kept & ~front));
      if (i < words) word[i] = {kept, holes + listed.a, sources + listed.b};
      equals += same.all_a;
      holes += listed.all_a;
      sources += listed.all_b;
    }
    moves = holes;
    __syncthreads();
    Move* list = space.list + pair * space.list_max;
#pragma unroll 2
    for (int i = warp; i < words; i += kSelectWarps) {  // rows first, their places in the pools behind the barrier
      const Word x = word[i];
      const int t = i * 32 + lane;
      const bool kept = x.kept >> lane & 1, front = t < keep;
      const unsigned hole = __ballot_sync(~0u, t < n && !kept && front), source = __ballot_sync(~0u, kept && !front);
      const unsigned before = (1u << lane) - 1;
      if (hole >> lane & 1) list[x.holes + __popc(hole & before)].to = t;
      if (source >> lane & 1) list[x.sources + __popc(source & before)].from = t;
      if (kept && front) {
        if (weights_out != weights) weights_out[t] = weights[t];
        if (positions_out != positions) positions_out[t] = positions[t];
      }
    }
    __syncthreads();
    for (int i0 = 0; i0 < moves; i0 += kMoveBatch) {
      const int i = i0 + (int)threadIdx.x;
      if ((int)threadIdx.x < kMoveBatch && i < moves) {
        Move m = list[i];
        const float w = weights[m.from];
        const int p = positions[m.from];
        const long long from = paged_row(c, b, (int)m.from), to = paged_row(c, b, (int)m.to);
        weights_out[m.to] = w;
        positions_out[m.to] = p;
        m.from = (from + g * c.head_stride) * esize;
        m.to = from < 0 || to < 0 ? -1 : (to + g * c.head_stride) * esize;
        if (move_here) sh.moves[threadIdx.x] = m;
        else list[i] = m;
      }
      if (move_here) {
        __syncthreads();
        move_rows(c, sh.moves, min(kMoveBatch, moves - i0), pieces, lanes, (int)threadIdx.x / lanes, kSelectThreads / lanes);
        __syncthreads();
      }
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
    if (atomicInc(&space.arrivals[b], (unsigned)c.kv_heads - 1) == (unsigned)c.kv_heads - 1) e.lengths_out[b] = left;
  }
}

// The rows of all moves. It lets the next kernel of the stream start only as it ends: blocks that wait would take its place.
__global__ void __launch_bounds__(kMoveThreads) paged_evict_move_kernel(PagedView c, EvictSpace space, int pieces, int lanes) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int pair = blockIdx.z * c.kv_heads + blockIdx.y;
  const int rows = kMoveThreads / lanes;
  move_rows(c, space.list + pair * space.list_max, space.moves[pair], pieces, lanes, blockIdx.x * rows + threadIdx.x / lanes, gridDim.x * rows);
}

}  // namespace

int paged_append_launch(const PagedView& c, const PagedAppend& a, int sm_count, bool pdl, cudaStream_t stream) {
  const int esize = (int)dtype_size(c.dtype), pieces = c.head_dim * esize / 16;
  const long long work = a.rows * c.kv_heads * pieces;
  const long long blocks = std::min((work + kAppendThreads - 1) / kAppendThreads, (64ll * sm_count + c.batch - 1) / c.batch);
  return launch_kernel(paged_append_kernel, dim3((unsigned)blocks, (unsigned)c.batch), dim3(kAppendThreads), 0,
                       stream, pdl, c, a, pieces, esize) == cudaSuccess;
}

WorkspaceSize paged_evict_workspace(const PagedView& c) {
  const EvictLayout l = evict_layout(c);
  return {l.bytes, l.moves};
}

int paged_evict_launch(const PagedView& c, const PagedEvict& e, int sm_count, bool pdl, cudaStream_t stream) {
  const int esize = (int)dtype_size(c.dtype), pieces = c.head_dim * esize / 16;
  int lanes = 1;
  while (lanes < pieces) lanes *= 2;
  const EvictSpace space = evict_space(c, e.workspace);
  const long long capacity = c.capacity(), pairs = (long long)c.batch * c.kv_heads;
  const int in_shared = capacity <= kRowsInShared;
  const size_t smem = in_shared ? (size_t)(capacity + 3) / 4 * 16 + (size_t)(capacity / 32 + 1) * sizeof(Word) : 0;
  if (!raise_smem_limit((const void*)paged_evict_select_kernel, (int)(kRowsInShared * 4 + (kRowsInShared / 32 + 1) * sizeof(Word)))) return 0;
  const long long moves_max = std::min<long long>(e.keep, capacity - e.keep);
  const int move_here = moves_max <= kMoveHere;
  if (launch_kernel(paged_evict_select_kernel, dim3((unsigned)c.kv_heads, (unsigned)c.batch), dim3(kSelectThreads),
                    smem, stream, pdl, c, e, space, pieces, lanes, esize, in_shared, move_here) != cudaSuccess)
    return 0;
  if (move_here || moves_max <= 0) return 1;
  const long long blocks = std::max<long long>(1, std::min((moves_max * lanes + kMoveThreads - 1) / kMoveThreads, 8ll * sm_count / pairs + 1));
  if (launch_kernel(paged_evict_move_kernel, dim3((unsigned)blocks, (unsigned)c.kv_heads, (unsigned)c.batch), dim3(kMoveThreads), 0, stream,
                    true, c, space, pieces, lanes) != cudaSuccess)
    return 0;
  return 2;
}

}  // namespace pjrtx
