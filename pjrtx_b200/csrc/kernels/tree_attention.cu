// Attention of a tree of drafted tokens per sequence over a paged cache: node i sees the cached rows, its ancestors and itself.
//
// Cached rows and nodes are one axis of keys, rows 0..length - 1 and behind them nodes 0..count - 1, cut into tiles; which source a key
// comes from is known where it is fetched, and what a row sees are the keys below `length` and a word of bits from there on. A tile of
// query rows is some nodes of a sequence times the query heads of a KV head: row x is head x % heads of node x / heads. So each cached row
// is read once for all nodes and heads that share it, which is what the operator is for: one node at a time would read it once for each.
//
// Bound by the cached rows' bytes until a row is read for some 250 query rows (16 bits: 4 operations an element and query row). 16-bit types go
// to the tensor cores (umma_tree.cuh), f32 to the CUDA cores (row_attention.cuh).
#include <algorithm>

#include "../common.h"
#include "kernels.h"
#include "paged.cuh"
#include "row_attention.cuh"
#include "tree.cuh"

namespace pjrtx {

namespace {

// ---- division of the work ------------------------------------------------------------------------------------------
// A segment is a (sequence, KV head, tile of query rows), a unit a tile of its keys. Segments have numbers for their units and, behind
// them, for kSegmentCost more: what ending one and going on with the next takes. The numbers are cut into equal shares, one for each
// block; lengths are device data, so each block adds them up itself. Where several blocks share a segment, each leaves (sums, max, total)
// in its slot of the workspace, and a second kernel joins them in block order.
// kSegmentCost, in units, by 16 sequences of up to 4096 rows and 16 nodes, 32 of up to 2048 and 4, one of 65536 and 32 (bf16, 32 heads of 128 over 8) and
// 16 of up to 2000 and 8 in f32: 0 takes 63, 77, 82 us; 2 59, 64, 72 and 171; 3 57, 62, 69 and 179; 4 57, 67, 70 and 187; 6 56, 69, 68 and 201.

constexpr int kSegmentCost = 2;
constexpr int kJoinWarps = 16;

// What the query rows of a segment are.
struct Segment {
  int b, node0, nodes, g, h0, heads;  // nodes and heads of the tile
  __device__ __forceinline__ bool place(int across, int row, int* node, int* head) const {  // `across`: heads of a full tile
    *node = node0 + row / across;
    *head = row % across;
    return row / across < nodes && *head < heads;
  }
};

// A segment that ends in another block than it begins in: written by the block it begins in, first >= last where there is none.
struct Cut {
  Segment seg;
  int first, last;
};

struct TreeArgs {
  PagedView c;
  PagedTree a;
  int rep, heads, groups;  // query heads of a KV head; those of a tile; tiles that share a node
  int nodes;               // of a tile
  int tile_keys;
  int slot_rows, dims;     // of a part's sums in the workspace: [dims][rows], then the rows' maxima and totals
  unsigned reciprocal;     // floor(2^32 / page_size), at most 2^32 - 1
  int blocks;
  Cut* cuts;               // [blocks]
  float* parts;            // [blocks][2][slot_rows * (dims + 2)]
};

struct Sequence {
  int length, count, tiles, segments;  // cached rows, nodes; units of a segment; segments
};

__device__ __forceinline__ Sequence sequence_of(const TreeArgs& p, int b, bool check = false) {
  Sequence s;
  const int count = p.a.counts ? p.a.counts[b] : p.a.nodes;
  s.length = paged_length(p.c, b);
  if (check) {
    paged_check_length(p.c, b);
    if (count < 0 || count > p.a.nodes) report(p.c.error_words, kErrorLength);
  }
  s.count = max(0, min(count, p.a.nodes));
  s.tiles = s.count ? (s.length + s.count + p.tile_keys - 1) / p.tile_keys : 0;
  s.segments = p.c.kv_heads * p.groups * ((s.count + p.nodes - 1) / p.nodes);
  return s;
}

struct Cursor {
  int b, group, tile;  // group: the segment's number in its sequence, ((tile of nodes) * KV heads + KV head) * groups + group of heads
  Sequence s;
};

// What this block works on: the units among numbers [begin, begin + size), the first of them at `first` of these.
struct Share {
  long long begin, quota, size, first;  // first >= size: none
  Cursor at;
};

__device__ __forceinline__ long long numbers_of(const Sequence& s) { return s.tiles ? (long long)s.segments * (s.tiles + kSegmentCost) : 0; }

// On to the next segment. A call, since many places do it and none often.
__device__ __noinline__ Cursor next_segment(const TreeArgs& p, Cursor u) {
  u.tile = 0;
  if (++u.group < u.s.segments) return u;
  u.group = 0;
  do {
    u.b++;
    u.s = sequence_of(p, u.b);
  } while (u.s.tiles == 0);
  return u;
}

__device__ __forceinline__ void advance(const TreeArgs& p, Cursor& u) {
  if (++u.tile >= u.s.tiles) u = next_segment(p, u);
}

// The next unit of a share; false at its end.
__device__ __forceinline__ bool next_unit(const TreeArgs& p, Cursor& u, long long& at, long long size) {
  const long long to = at + (u.tile + 1 < u.s.tiles ? 1 : 1 + kSegmentCost);
  if (to >= size) return false;
  at = to;
  advance(p, u);
  return true;
}

template <int THREADS>
struct ShareSpace {
  long long sums[THREADS / 32], first;
  Cursor at;
};

// Called by all threads.
template <int THREADS>
__device__ __forceinline__ Share share_of_block(const TreeArgs& p, ShareSpace<THREADS>& space) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int per_thread = (p.c.batch + THREADS - 1) / THREADS;
  const int first = min(p.c.batch, (int)threadIdx.x * per_thread), last = min(p.c.batch, first + per_thread);
  long long mine = 0;
  for (int b = first; b < last; b++) mine += numbers_of(sequence_of(p, b, blockIdx.x == 0));
  long long sum = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long o = __shfl_up_sync(~0u, sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 31) space.sums[warp] = sum;
  __syncthreads();
  long long before = sum - mine, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; w++) {
    if (w < warp) before += space.sums[w];
    total += space.sums[w];
  }
  Share s;
  s.quota = max(1ll, (total + gridDim.x - 1) / gridDim.x);
  s.begin = min(total, blockIdx.x * s.quota);
  s.size = min(total - s.begin, s.quota);
  if (s.size > 0 && before <= s.begin && s.begin < before + mine) {
    long long rest = s.begin - before;
    Cursor u;
    u.b = first;
    for (;; u.b++) {
      u.s = sequence_of(p, u.b);
      if (rest < numbers_of(u.s)) break;
      rest -= numbers_of(u.s);
    }
    u.group = (int)(rest / (u.s.tiles + kSegmentCost));
    u.tile = (int)(rest % (u.s.tiles + kSegmentCost));
    long long at = 0;
    if (u.tile >= u.s.tiles) {  // behind a segment's units: the share begins with the next one
      at = u.s.tiles + kSegmentCost - u.tile;
      if (at < s.size) advance(p, u);
    }
    space.at = u;
    space.first = at;
  }
  __syncthreads();
  s.at = space.at;
  s.first = s.size > 0 ? space.first : 0;
  return s;
}

__device__ __noinline__ Segment segment_of(const TreeArgs& p, int b, int group, int count) {
  Segment s;
  s.b = b;
  const int across = p.c.kv_heads * p.groups, r = group % across;
  s.node0 = group / across * p.nodes;
  s.nodes = min(p.nodes, count - s.node0);
  s.g = r / p.groups;
  s.h0 = r % p.groups * p.heads;
  s.heads = min(p.heads, p.rep - s.h0);
  return s;
}

__device__ __forceinline__ long long query_at(const TreeArgs& p, const Segment& s, int node, int head) {
  return s.b * p.a.q_batch_stride + node * p.a.q_node_stride + (long long)(s.g * p.rep + s.h0 + head) * p.a.q_head_stride;
}
__device__ __forceinline__ long long out_at(const TreeArgs& p, const Segment& s, int node, int head) {
  return s.b * p.a.out_batch_stride + node * p.a.out_node_stride + (long long)(s.g * p.rep + s.h0 + head) * p.a.out_head_stride;
}
__device__ __forceinline__ long long lse_at(const TreeArgs& p, const Segment& s, int node, int head) {
  return ((long long)s.b * p.a.nodes + node) * p.a.heads + s.g * p.rep + s.h0 + head;
}

// Column of the page table that row t is in.
__device__ __forceinline__ int column_of(const TreeArgs& p, int t) {
  const int column = (int)__umulhi((unsigned)t, p.reciprocal);  // the quotient or one less
  return t - column * p.c.page_size >= p.c.page_size ? column + 1 : column;
}

// Element offset of cached row t of sequence b in either pool (KV head 0), -1 where the table names no page.
__device__ __forceinline__ long long cached_row(const TreeArgs& p, int b, int t) {
  const int column = column_of(p, t), page = p.c.table[b * p.c.table_stride + column];
  if (page < 0 || page >= p.c.num_pages) {
    report(p.c.error_words, kErrorPageId);
    return -1;
  }
  return page * p.c.page_stride + (t - column * p.c.page_size) * p.c.row_stride;
}

// The slot of this block's part of a segment that other blocks share, and the cut that the join goes by; null where none does. Slot 1
// of a block holds the segment that begins in it, slot 0 the one that began before.
__device__ __forceinline__ float* part_of(const TreeArgs& p, const Share& share, const Cursor& u, const Segment& seg, long long segment) {
  const long long first = segment / share.quota, last = (segment + u.s.tiles - 1) / share.quota;
  if (first == last) return nullptr;
  if (threadIdx.x == 0 && blockIdx.x == first) p.cuts[blockIdx.x] = {seg, (int)first, (int)last};
  return p.parts + ((long long)blockIdx.x * 2 + (blockIdx.x == first ? 1 : 0)) * p.slot_rows * (p.dims + 2);
}

__device__ __forceinline__ void store_statistics(const TreeArgs& p, float* part, int row, float m, float total) {
  part[(long long)p.slot_rows * p.dims + row] = m;
  part[(long long)p.slot_rows * (p.dims + 1) + row] = total;
}

}  // namespace
}  // namespace pjrtx

#include "umma_tree.cuh"

namespace pjrtx {
namespace {

// ---- on the CUDA cores ---------------------------------------------------------------------------------------------

template <int D, int R>
__global__ void __launch_bounds__(rows::kThreads) tree_rows_kernel(const __grid_constant__ TreeArgs p) {
  PJRTX_PDL_PROLOGUE();
  using namespace rows;
  using Space = Shared<D, R>;
  extern __shared__ __align__(16) char smem[];
  __shared__ ShareSpace<kThreads> space;
  __shared__ unsigned long long ancestors[kTreeNodesMax];
  Space& s = *reinterpret_cast<Space*>(smem);
  if (threadIdx.x == 0) p.cuts[blockIdx.x] = {};
  const Share share = share_of_block(p, space);
  if (share.first >= share.size) return;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const float* any = static_cast<const float*>(p.a.q);
  Cursor now = share.at;
  long long at = share.first;
  int stage = 0;
  for (bool more = true; more;) {
    const Segment seg = segment_of(p, now.b, now.group, now.s.count);
    const Cursor here = now;
    const int keys = here.s.length + here.s.count;
    auto request = [&](int tile, int to) {
      constexpr int kOfWarp = Space::kKeys / 8;
      const int t = tile * Space::kKeys + warp * kOfWarp + lane;
      const float *k = nullptr, *v = nullptr;
      if (lane < kOfWarp && t < here.s.length) {
        const long long row = cached_row(p, seg.b, t);
        if (row >= 0) {
          k = static_cast<const float*>(p.c.k) + row + seg.g * p.c.head_stride;
          v = static_cast<const float*>(p.c.v) + row + seg.g * p.c.head_stride;
        }
      } else if (lane < kOfWarp && t < keys) {
        const long long row = seg.b * p.a.new_batch_stride + (t - here.s.length) * p.a.new_node_stride + seg.g * p.a.new_head_stride;
        k = static_cast<const float*>(p.a.k_new) + row;
        v = static_cast<const float*>(p.a.v_new) + row;
      }
      request_rows<D, Space::kKeys>(s.k[to & 1], k, p.c.head_dim, any);
      request_rows<D, Space::kKeys>(s.v[to & 1], v, p.c.head_dim, any);
    };
    __syncthreads();  // the segment before has been read
    if (warp == 0) {
      const Ancestors above = tree_ancestors(p.a.parents + (long long)seg.b * p.a.nodes, here.s.count, p.c.error_words);
      ancestors[lane] = above.low;
      ancestors[lane + 32] = above.high;
    }
    {
      constexpr int kOfWarp = Space::kRows / 8;
      int node, head;
      const float* q = nullptr;
      if (lane < kOfWarp && seg.place(p.heads, warp * kOfWarp + lane, &node, &head)) q = any + query_at(p, seg, node, head);
      request_rows<D, Space::kRows>(s.q, q, p.c.head_dim, any);
    }
    request(now.tile, stage);
    __syncthreads();
    Sight sight[R];
    Sums<D, R> sum;
    sum.clear();
#pragma unroll
    for (int i = 0; i < R; i++) {
      int node, head;
      sight[i] = {0, 0ull};
      if (seg.place(p.heads, ty * R + i, &node, &head)) sight[i] = {here.s.length, ancestors[node]};
    }
    const long long segment = share.begin + at - here.tile;  // number of its first unit
    for (bool same = true; same; stage++) {
      const int tile = now.tile;
      more = next_unit(p, now, at, share.size);
      same = more && now.group == here.group && now.b == here.b;
      block_of_keys<false, D, R>(s, sum, sight, stage, tile * Space::kKeys, keys, keys, here.s.length, p.a.scale * kLog2e, [&] {
        if (same) request(now.tile, stage + 1);
      });
    }
    if (float* part = part_of(p, share, here, seg, segment)) {
#pragma unroll
      for (int c = 0; c < D / 64; c++)
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
          for (int i = 0; i < R; i++) {
            const float2 o = pair_split(sum.o[i][c][e / 2]);
            part[(c * 64 + tx * 4 + e) * p.slot_rows + ty * R + i] = e % 2 ? o.y : o.x;
          }
#pragma unroll
      for (int i = 0; i < R; i++)
        if (tx == 0) store_statistics(p, part, ty * R + i, sum.m[i], sum.l[i]);
      continue;
    }
#pragma unroll
    for (int i = 0; i < R; i++) {
      int node, head;
      if (!seg.place(p.heads, ty * R + i, &node, &head)) continue;
      const float inverse = inverse_of(sum.l[i]);
      float* out = static_cast<float*>(p.a.out) + out_at(p, seg, node, head);
#pragma unroll
      for (int c = 0; c < D / 64; c++) {
        const float2 x = pair_split(sum.o[i][c][0]), y = pair_split(sum.o[i][c][1]);
        const int d = c * 64 + tx * 4;
        if (d < p.c.head_dim) store4(out + d, make_float4(x.x * inverse, x.y * inverse, y.x * inverse, y.y * inverse));
      }
      if (tx == 0 && p.a.lse) p.a.lse[lse_at(p, seg, node, head)] = lse_of(sum.m[i], sum.l[i]);
    }
  }
}

// ---- parts of a segment ---------------------------------------------------------------------------------------------

// A block has 32 rows of a cut segment, a lane a row, a warp eight dimensions and every `splits`-th part, in an order that does not depend on
// which is first. Many segments are cut once or twice and take the parts one after the other; where few blocks have a place, more warps share a row's
// parts, and blocks go by the cuts that there are (looking for one takes 1 us): so where a segment has four blocks and more. Without that, one sequence of
// 65536 rows and 32 nodes takes 90 us, not 75, and one of 517 rows and 8 nodes 16.4, not 14.2; with it from one block a segment on, 16 of up to 4096
// rows and 16 nodes 80, not 60. Loops are not unrolled: every launch fetches its instructions anew, and 16 dimensions a warp with unrolled loops
// took 8 us for each part behind the first.
constexpr int kJoinDims = 8;

// The n-th cut there is, -1: none. Called by all threads.
__device__ __forceinline__ int cut_of(const TreeArgs& p, int n) {
  __shared__ int found, counts[kJoinWarps];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (threadIdx.x == 0) found = -1;
  int before = 0;
  for (int i0 = 0; i0 < p.blocks && before <= n; i0 += kJoinWarps * 32) {
    const int i = i0 + threadIdx.x;
    const bool valid = i < p.blocks && p.cuts[i].first < p.cuts[i].last;
    const unsigned mask = __ballot_sync(~0u, valid);
    if (lane == 0) counts[warp] = __popc(mask);
    __syncthreads();
    int at = before + __popc(mask & ((1u << lane) - 1));
#pragma unroll 1
    for (int w = 0; w < kJoinWarps; w++) {
      if (w < warp) at += counts[w];
      before += counts[w];
    }
    if (valid && at == n) found = i;
    __syncthreads();
  }
  return found;
}

// Sums of a row relative to m, with more of them.
__device__ __forceinline__ void join(float& m, float& total, float (&x)[kJoinDims], float m_new, float mass, const float (&y)[kJoinDims]) {
  if (m_new == -INFINITY && mass == 0.f) return;
  const float top = fmaxf(m, m_new), shift = top == -INFINITY ? 0.f : top;
  const float was = m == top ? 1.f : exp2_fast(m - shift), is = m_new == top ? 1.f : exp2_fast(m_new - shift);
  total = fmaf(total, was, mass * is);
#pragma unroll
  for (int e = 0; e < kJoinDims; e++) x[e] = fmaf(x[e], was, y[e] * is);
  m = top;
}

template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) tree_join_kernel(const __grid_constant__ TreeArgs p, int splits, int look) {
  PJRTX_PDL_PROLOGUE();
  __shared__ float parts[kJoinWarps][kJoinDims + 2][32];
  __shared__ __align__(16) float results[32][kJoinWarps * kJoinDims + 4];
  const int at = look ? cut_of(p, blockIdx.x) : (int)blockIdx.x;
  if (at < 0) return;
  const Cut cut = p.cuts[at];
  if (cut.first >= cut.last) return;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, row0 = blockIdx.y * 32, chunks = kJoinWarps / splits;
  const int first = blockIdx.z * chunks * kJoinDims, mine = warp / splits * kJoinDims, d0 = first + mine;  // dimensions: the block's, the warp's
  const Segment& seg = cut.seg;
  int node, head;
  const bool there = seg.place(p.heads, row0 + lane, &node, &head);
  if (!__any_sync(~0u, there)) return;  // the same rows in every warp
  float m = -INFINITY, total = 0.f, x[kJoinDims], y[kJoinDims];
#pragma unroll
  for (int e = 0; e < kJoinDims; e++) x[e] = 0.f;
  if (there && d0 < p.dims) {
#pragma unroll 1
    for (int i = warp % splits; i <= cut.last - cut.first; i += splits) {
      const float* from = p.parts + ((long long)(cut.first + i) * 2 + (i ? 0 : 1)) * p.slot_rows * (p.dims + 2) + row0 + lane;
      const float m_new = from[p.slot_rows * p.dims], mass = from[p.slot_rows * (p.dims + 1)];
#pragma unroll
      for (int e = 0; e < kJoinDims; e++) y[e] = from[(d0 + e) * p.slot_rows];
      join(m, total, x, m_new, mass, y);
    }
  }
  if (splits > 1) {
    parts[warp][kJoinDims][lane] = m;
    parts[warp][kJoinDims + 1][lane] = total;
#pragma unroll
    for (int e = 0; e < kJoinDims; e++) parts[warp][e][lane] = x[e];
    __syncthreads();
    if (warp % splits == 0) {
#pragma unroll 1
      for (int w = warp + 1; w < warp + splits; w++) {
#pragma unroll
        for (int e = 0; e < kJoinDims; e++) y[e] = parts[w][e][lane];
        join(m, total, x, parts[w][kJoinDims][lane], parts[w][kJoinDims + 1][lane], y);
      }
    }
  }
  if (warp % splits == 0) {
    const float inverse = rows::inverse_of(total);
#pragma unroll
    for (int e = 0; e < kJoinDims; e++) results[lane][mine + e] = x[e] * inverse;
    if (p.a.lse && there && d0 == 0) p.a.lse[lse_at(p, seg, node, head)] = rows::lse_of(m, total);
  }
  __syncthreads();
  const int pieces = chunks * kJoinDims / 4;
#pragma unroll 1
  for (int i = threadIdx.x; i < 32 * pieces; i += kJoinWarps * 32) {
    const int r = i / pieces, d = i % pieces * 4;
    if (first + d < p.c.head_dim && seg.place(p.heads, row0 + r, &node, &head))
      rows::store4(static_cast<T*>(p.a.out) + out_at(p, seg, node, head) + first + d, *reinterpret_cast<const float4*>(&results[r][d]));
  }
}

// ---- launches ------------------------------------------------------------------------------------------------------

// Which kernel a shape runs on.
struct TreePlan {
  int dims, rows, keys;  // of a row, of a tile of queries, of a tile of keys
  int threads, per_sm;   // threads of a block, blocks an SM
  size_t smem;
};

// f(kernel, plan) for calls with `wanted` query rows a sequence and KV head at most: two tiles read the keys once for up to 256 of them, and in
// f32 no more rows are computed than there are, up to 64.
template <typename F>
auto with_kernel(int dtype, int head_dim, long long wanted, F&& f) {
#define PJRTX_TREE_ROWS(D, R) return f(tree_rows_kernel<D, R>, TreePlan{D, 16 * R, rows::keys_of(D), rows::kThreads, D == 64 ? 2 : 1, sizeof(rows::Shared<D, R>)})
#define PJRTX_TREE_ROWS_OF(D)              \
  {                                        \
    if (wanted <= 16) PJRTX_TREE_ROWS(D, 1); \
    if (wanted <= 32) PJRTX_TREE_ROWS(D, 2); \
    PJRTX_TREE_ROWS(D, 4);                 \
  }
#define PJRTX_TREE_UMMA(BF16, D, TILES) \
  return f(umma::umma_tree_kernel<BF16, D, TILES>, \
           TreePlan{D, TILES * umma::kAttnRows, umma::tree_keys(D), umma::tree_threads(TILES), 1, umma::tree_smem(D, TILES)})
#define PJRTX_TREE_UMMA_OF(BF16)                                                     \
  if (head_dim > 128) PJRTX_TREE_UMMA(BF16, 256, 1);                                 \
  if (head_dim > 64 && wanted > umma::kAttnRows) PJRTX_TREE_UMMA(BF16, 128, 2);        \
  if (head_dim > 64) PJRTX_TREE_UMMA(BF16, 128, 1);                                  \
  if (wanted > umma::kAttnRows) PJRTX_TREE_UMMA(BF16, 64, 2);                          \
  PJRTX_TREE_UMMA(BF16, 64, 1)
  if (dtype == kF32) {
    if (head_dim <= 64) PJRTX_TREE_ROWS_OF(64)
    if (head_dim <= 128) PJRTX_TREE_ROWS_OF(128)
    PJRTX_TREE_ROWS_OF(256)
  }
  if (dtype == kF16) { PJRTX_TREE_UMMA_OF(false); }
  PJRTX_TREE_UMMA_OF(true);
#undef PJRTX_TREE_UMMA_OF
#undef PJRTX_TREE_UMMA
#undef PJRTX_TREE_ROWS_OF
#undef PJRTX_TREE_ROWS
}

// The tensor-core kernels take the scale apart.
bool start(void (*kernel)(const TreeArgs), const TreeArgs& p, const TreePlan& plan, bool pdl, cudaStream_t stream) {
  return launch_kernel(kernel, dim3((unsigned)p.blocks), dim3((unsigned)plan.threads), plan.smem, stream, pdl, p) == cudaSuccess;
}
bool start(void (*kernel)(const umma::TreeKernelArgs, const CUtensorMap, const CUtensorMap), const TreeArgs& p, const TreePlan& plan, bool pdl, cudaStream_t stream) {
  const float scale = p.a.scale;
  umma::TreeKernelArgs a;
  a.p = p;
  a.scale_log2 = scale == 0.f ? 1.f : (scale < 0.f ? -scale : scale) * rows::kLog2e;
  a.sign = scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f;
  a.timeout_ns = wait_timeout_ns();
  a.box = umma::tree_box(plan.keys, p.c.page_size);
  CUtensorMap kmap{}, vmap{};
  if (a.box) {
    const PagedView& c = p.c;
    const long long extents[4] = {c.head_dim, c.page_size, c.kv_heads, c.num_pages}, strides[3] = {c.row_stride, c.head_stride, c.page_stride};
    const int box[4] = {64, a.box, 1, 1};
    if (!umma::encode_map(&kmap, c.k, c.dtype == kF16, 4, extents, strides, box) || !umma::encode_map(&vmap, c.v, c.dtype == kF16, 4, extents, strides, box))
      return false;
  }
  return launch_kernel(kernel, dim3((unsigned)p.blocks), dim3((unsigned)plan.threads), plan.smem, stream, pdl, a, kmap, vmap) == cudaSuccess;
}

uint64_t round256(uint64_t n) { return (n + 255) / 256 * 256; }

}  // namespace

uint64_t paged_tree_workspace(const PagedView& c, int heads, int nodes, int sm_count) {
  return with_kernel(c.dtype, c.head_dim, (long long)nodes * (heads / c.kv_heads), [&](auto, const TreePlan& plan) {
    const uint64_t blocks = (uint64_t)sm_count * plan.per_sm;
    return round256(blocks * sizeof(Cut)) + blocks * 2 * plan.rows * (plan.dims + 2) * 4;
  });
}

int paged_tree_launch(const PagedView& c, const PagedTree& a, int sm_count, bool pdl, cudaStream_t stream) {
  TreeArgs p;
  p.c = c;
  p.a = a;
  p.rep = a.heads / c.kv_heads;
  p.reciprocal = (unsigned)std::min<uint64_t>((1ull << 32) / c.page_size, 0xffffffffu);
  char* space = static_cast<char*>(a.workspace);
  p.cuts = reinterpret_cast<Cut*>(space);
  long long segments = 0;
  const bool ok = with_kernel(c.dtype, c.head_dim, (long long)a.nodes * p.rep, [&](auto kernel, const TreePlan& plan) {
    p.heads = std::min(p.rep, plan.rows);
    p.groups = (p.rep + p.heads - 1) / p.heads;
    p.nodes = plan.rows / p.heads;
    p.tile_keys = plan.keys;
    p.slot_rows = plan.rows;
    p.dims = plan.dims;
    if (!raise_smem_limit((const void*)kernel, (int)plan.smem)) return false;
    segments = (long long)c.batch * c.kv_heads * p.groups * ((a.nodes + p.nodes - 1) / p.nodes);
    const long long numbers = segments * ((c.capacity() + a.nodes + p.tile_keys - 1) / p.tile_keys + kSegmentCost);
    p.blocks = (int)std::min<long long>(numbers, (long long)sm_count * plan.per_sm);
    p.parts = reinterpret_cast<float*>(space + round256((uint64_t)sm_count * plan.per_sm * sizeof(Cut)));
    return start(kernel, p, plan, pdl, stream);
  });
  if (!ok) return 0;
  const int groups = (std::min(p.slot_rows, std::min(p.nodes, a.nodes) * p.heads) + 31) / 32;
  const int look = segments * 4 <= p.blocks, splits = look ? 8 : 1, across = kJoinWarps / splits * kJoinDims;
  const dim3 grid((unsigned)(look ? segments : p.blocks), (unsigned)groups, (unsigned)((c.head_dim + across - 1) / across));
  auto join = c.dtype == kF32 ? tree_join_kernel<float> : c.dtype == kF16 ? tree_join_kernel<__half> : tree_join_kernel<__nv_bfloat16>;
  return launch_kernel(join, grid, dim3(kJoinWarps * 32), 0, stream, true, p, splits, look) == cudaSuccess ? 2 : 0;
}

}  // namespace pjrtx
