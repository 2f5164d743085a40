// Page tables and slots of a paged key-value cache, built where the lengths are: on the device.
//
// assign: need = ceil(length / page_size). Surplus pages go onto the stack of free ones, ordered by (sequence, column), entries that name no
// page of the pool left out; then the i-th page wanted, in the same order, is the i-th from the top, for the sequences whose running sum of wants
// fits what is there. Both orders are prefix sums over the batch, so the result does not depend on who is first.
//
// path: a drafted token is accepted when it lies on the way from the leaf to its root; its row is the number of those before it.
//
// All of it is a few hundred KB at most (a table of 512 x 256 pages and its copy: 1 MB), so what counts is the number of trips to memory
// in a row: one launch of one cluster, whose blocks pass sums and pages to each other between cluster barriers, and loops that have several
// loads under way. 32 sequences that grow by a row take 7.8 us, 512 that get new prompts of up to 4096 tokens, with the slots of all of these
// (377 000, by a kernel of their own), 23.0, of which counting the surplus pages first is 1.7; 4096 sequences of 64 pages 55. Before that count, one load
// after the other took 27.3, not 20.8, eight at a time 20.4 and 59, not 49, with 4096 sequences; blocks of 1024 threads 10.5, 21.1 and 38. Path slots of 256 trees of 64 nodes take 2.5 us, with the
// ancestors in six rounds of doubling and not by up to 63 steps of a chain.
#include <cooperative_groups.h>

#include <utility>

#include "../common.h"
#include "kernels.h"
#include "paged.cuh"
#include "tree.cuh"

namespace pjrtx {

namespace {

constexpr int kBlocks = 8, kThreads = 512, kWarps = kThreads / 32;

// What a sequence has and is to have, in pages. A length or count that the table cannot hold: `ok` is 0 and need is what it has.
struct Want {
  int held, need, ok;
};

__device__ __forceinline__ Want want_of(const PagedAssign& a, int b, bool stack_ok) {
  const int held = a.held[b], length = a.lengths[b];
  Want w;
  const bool known = held >= 0 && held <= a.max_pages;
  w.held = known ? held : 0;
  const long long need = length < 0 ? -1 : ((long long)length + a.page_size - 1) / a.page_size;
  w.ok = known && need >= 0 && need <= a.max_pages;
  w.need = w.ok && stack_ok ? (int)need : w.held;
  return w;
}

// Sum over the block's threads before this one, and of all; called by all threads.
__device__ __forceinline__ long long block_prefix(long long x, long long* warp_sums, long long* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  long long sum = x;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long o = __shfl_up_sync(~0u, sum, d);
    if (lane >= d) sum += o;
  }
  __syncthreads();  // the sums of the call before have been read
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; w++) {
    if (w < warp) before += warp_sums[w];
    all += warp_sums[w];
  }
  *total = all;
  return before + sum - x;
}

struct Sums {
  long long give, take, granted;
};

// For i = first, first + step, .. before last: from(i) for several of them, whose loads are then under way together, before to(i, what it gave).
template <typename From, typename To>
__device__ __forceinline__ void in_batches(long long first, long long last, int step, From from, To to) {
  constexpr int kBatch = 4;
  for (long long i0 = first; i0 < last; i0 += (long long)kBatch * step) {
    int x[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; u++) {
      const long long i = i0 + u * step;
      x[u] = i < last ? from(i) : 0;
    }
#pragma unroll
    for (int u = 0; u < kBatch; u++) {
      const long long i = i0 + u * step;
      if (i < last) to(i, x[u]);
    }
  }
}

// Slot of a packed token, once tables and page counts are written: the sequence by bisection, the row from its end.
__device__ __forceinline__ int slot_of(const PagedAssign& a, long long t) {
  if (a.batch == 0 || t < a.starts[0] || t >= a.starts[a.batch]) return -1;
  int lo = 0, hi = a.batch;  // starts[lo] <= t < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int length = a.lengths[lo], held = __ldcg(a.held_out + lo);
  const long long row = length - (a.starts[lo + 1] - t);
  if (row < 0 || length > (long long)a.page_size * a.max_pages) {
    report(a.error_words, kErrorLength);
    return -1;
  }
  if ((long long)held * a.page_size < length) return -1;
  const int column = (int)row / a.page_size, page = __ldcg(a.table_out + lo * a.table_out_stride + column);
  if (page < 0 || page >= a.num_pages) {
    report(a.error_words, kErrorPageId);
    return -1;
  }
  return page * a.page_size + ((int)row - column * a.page_size);
}

// Sequences are divided among the blocks in chunks; a warp has a sequence at a time, its lanes the pages. `offsets`: shared memory of
// two numbers a sequence of the chunk. Sums have 64 bits: lengths may ask for more pages than there are.
__global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kThreads) paged_assign_kernel(const __grid_constant__ PagedAssign a, int slots) {
  PJRTX_PDL_PROLOGUE();
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ longlong2 offsets[];
  __shared__ Sums sums[kBlocks];  // of every block of the cluster
  __shared__ long long warp_sums[kWarps];
  const int rank = (int)cluster.block_rank(), lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int chunk = (a.batch + kBlocks - 1) / kBlocks, first = min(a.batch, rank * chunk), last = min(a.batch, first + chunk);
  const int had = *a.free_count;
  const bool stack_ok = had >= 0 && had <= a.num_pages;
  const int free_count = stack_ok ? had : 0;
  if (!stack_ok && rank == 0 && threadIdx.x == 0) report(a.error_words, kErrorLength);
  auto started = cluster.barrier_arrive();  // the other blocks' shared memory is written once they are known to run

  // What each sequence has to give and wants.
  bool gives = false;
  for (int b = first + threadIdx.x; b < last; b += kThreads) {
    const Want w = want_of(a, b, stack_ok);
    if (!w.ok) report(a.error_words, kErrorLength);
    offsets[b - first] = make_longlong2(max(0, w.held - w.need), max(0, w.need - w.held));
    gives = gives || w.held > w.need;
  }
  // Of surplus entries, those that name a page: the others go nowhere, or another sequence would get them.
  if (__syncthreads_or(gives)) {
    for (int b = first + warp; b < last; b += kWarps) {
      const int surplus = (int)offsets[b - first].x;
      if (surplus == 0) continue;
      const int* from = a.table + b * a.table_stride + want_of(a, b, stack_ok).need;
      int pages = 0;
      in_batches(lane, surplus, 32, [&](long long j) { return from[j]; }, [&](long long, int page) { pages += page >= 0 && page < a.num_pages; });
      pages = __reduce_add_sync(~0u, pages);
      if (lane == 0) offsets[b - first].x = pages;
      if (lane == 0 && pages < surplus) report(a.error_words, kErrorPageId);
    }
    __syncthreads();
  }
  // How many pages the sequences before have to give and want.
  long long give = 0, take = 0;
  for (int b0 = first; b0 < last; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    const longlong2 mine = b < last ? offsets[b - first] : make_longlong2(0, 0);
    long long given, taken;
    const long long give_at = give + block_prefix(mine.x, warp_sums, &given);
    const long long take_at = take + block_prefix(mine.y, warp_sums, &taken);
    if (b < last) offsets[b - first] = make_longlong2(give_at, take_at);
    give += given;
    take += taken;
  }
  cluster.barrier_wait(std::move(started));
  if (threadIdx.x < kBlocks) *cluster.map_shared_rank(&sums[rank], threadIdx.x) = Sums{give, take, 0};
  cluster.sync();
  long long give_before = 0, take_before = 0, returned = 0;
#pragma unroll
  for (int r = 0; r < kBlocks; r++) {
    if (r < rank) {
      give_before += sums[r].give;
      take_before += sums[r].take;
    }
    returned += sums[r].give;
  }
  // More pages than the pool has come back only where a page was held twice; what does not fit the stack is dropped.
  const int there = (int)min((long long)a.num_pages, free_count + returned);
  if (free_count + returned > a.num_pages && rank == 0 && threadIdx.x == 0) report(a.error_words, kErrorLength);

  // Surplus pages onto the stack, and how many pages this block's sequences get.
  long long granted = 0;
  for (int b = first + warp; b < last; b += kWarps) {
    const Want w = want_of(a, b, stack_ok);
    const longlong2 at = offsets[b - first];
    const int* surplus = a.table + b * a.table_stride + w.need;
    long long top = free_count + give_before + at.x;
    for (int j0 = 0; j0 < w.held - w.need; j0 += 128) {
      int page[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int j = j0 + u * 32 + lane;
        page[u] = j < w.held - w.need ? surplus[j] : -1;
      }
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const bool valid = page[u] >= 0 && page[u] < a.num_pages;
        const unsigned pages = __ballot_sync(~0u, valid);
        const long long to = top + __popc(pages & ((1u << lane) - 1));
        if (valid && to < a.num_pages) a.free_pages_out[to] = page[u];
        top += __popc(pages);
      }
    }
    const int wanted = w.need - w.held;
    if (wanted > 0 && take_before + at.y + wanted <= there) granted += wanted;
  }
  __syncthreads();
  if (lane == 0) warp_sums[warp] = granted;
  __syncthreads();
  granted = 0;
#pragma unroll
  for (int w = 0; w < kWarps; w++) granted += warp_sums[w];
  if (threadIdx.x < kBlocks) cluster.map_shared_rank(&sums[rank], threadIdx.x)->granted = granted;
  cluster.sync();  // the stack has what came back, too
  int count = there;
#pragma unroll
  for (int r = 0; r < kBlocks; r++) count -= (int)sums[r].granted;
  if (rank == 0 && threadIdx.x == 0) *a.free_count_out = stack_ok ? count : had;

  // The new tables. A popped place of the stack is cleared by whoever popped it.
  const bool copy_table = a.table != a.table_out, copy_stack = a.free_pages != a.free_pages_out;
  for (int b = first + warp; b < last; b += kWarps) {
    const Want w = want_of(a, b, stack_ok);
    const longlong2 at = offsets[b - first];
    const int wanted = w.need - w.held;
    const bool served = wanted <= 0 || take_before + at.y + wanted <= there;
    const int held = served ? w.need : w.held;
    const int* from = a.table + b * a.table_stride;
    int* to = a.table_out + b * a.table_out_stride;
    const int c0 = copy_table ? 0 : min(w.held, held), c1 = copy_table ? a.max_pages : max(w.held, held);
    const long long top = there - 1 - (take_before + at.y) + w.held;  // where column 0 would come from
    in_batches(
        c0 + lane, c1, 32,
        [&](long long c) {
          if (c >= w.held && c < held) return __ldcg((top - c < free_count ? a.free_pages : a.free_pages_out) + (top - c));
          return c >= held && c < w.held ? -1 : from[c];
        },
        [&](long long c, int page) {
          if (c >= w.held && c < held) {
            a.free_pages_out[top - c] = -1;
            if (page < 0 || page >= a.num_pages) report(a.error_words, kErrorPageId);
          }
          to[c] = page;
        });
    __syncwarp();  // in place: all lanes have read what the sequence had
    if (lane == 0) a.held_out[b] = w.ok ? held : a.held[b];
  }
  if (copy_stack)
    in_batches(
        rank * kThreads + threadIdx.x, a.num_pages, kBlocks * kThreads, [&](long long i) { return a.free_pages[i]; },
        [&](long long i, int page) {
          if (i < min(count, free_count) || i >= there) a.free_pages_out[i] = page;
        });
  if (!slots) return;
  cluster.sync();
  for (long long t = rank * kThreads + threadIdx.x; t < a.tokens; t += kBlocks * kThreads) a.slots[t] = slot_of(a, t);
}

// The same for more tokens than the cluster has threads. A second kernel costs the call its launch and next to nothing on the device: 8 sequences with 8
// tokens 7.0 us, not 6.7, 256 with 2048 in all 9.1 either way; a second and a fourth round of the cluster cost 8 192 tokens of 256 sequences 10.8, not 9.2,
// and 16 384 14.0, not 9.2.
constexpr int kSlotThreads = 256;
constexpr long long kSlotsHere = kBlocks * kThreads;

__global__ void __launch_bounds__(kSlotThreads) paged_slots_kernel(const __grid_constant__ PagedAssign a) {
  PJRTX_PDL_PROLOGUE();
  const long long t = (long long)blockIdx.x * kSlotThreads + threadIdx.x;
  if (t < a.tokens) a.slots[t] = slot_of(a, t);
}

constexpr int kPathThreads = 128;

// A warp a sequence, a lane two nodes.
__global__ void __launch_bounds__(kPathThreads) paged_path_kernel(const PagedPath a) {
  PJRTX_PDL_PROLOGUE();
  const int b = (blockIdx.x * kPathThreads + threadIdx.x) / 32, lane = threadIdx.x % 32;
  if (b >= a.batch) return;
  const int length = a.lengths[b], leaf = a.leaves[b];
  const int known = leaf < 0 || leaf >= a.nodes ? 0 : leaf + 1;  // a way goes to lower nodes
  const Ancestors above = tree_ancestors(a.parents + (long long)b * a.nodes, known, a.error_words);
  unsigned long long path = tree_of_node(above, max(0, min(leaf, kTreeNodesMax - 1)));
  const int rows = __popcll(path);
  if (leaf < 0) path = 0;
  if (leaf >= a.nodes || length < 0 || (path && length + (long long)rows > (long long)a.page_size * a.max_pages)) {
    if (lane == 0) report(a.error_words, kErrorLength);
    path = 0;
  }
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int node = lane + u * 32;
    if (node >= a.nodes) continue;
    int slot = -1;
    if (path >> node & 1) {
      const int row = length + __popcll(path & ((1ull << node) - 1)), column = row / a.page_size;
      const int page = a.table[b * a.table_stride + column];
      const long long at = (long long)page * a.page_size + (row - column * a.page_size);
      if (page >= 0 && at <= INT32_MAX) slot = (int)at;
      else report(a.error_words, kErrorPageId);
    }
    a.slots[(long long)b * a.nodes + node] = slot;
  }
  if (lane == 0) a.lengths_out[b] = length + __popcll(path);
}

}  // namespace

int paged_assign_launch(const PagedAssign& a, bool pdl, cudaStream_t stream) {
  const size_t smem = (size_t)((a.batch + kBlocks - 1) / kBlocks) * sizeof(longlong2);
  constexpr size_t kMost = (65535 + kBlocks - 1) / kBlocks * sizeof(longlong2);
  if (!raise_smem_limit((const void*)paged_assign_kernel, (int)kMost)) return 0;
  const bool here = a.tokens <= kSlotsHere;
  if (launch_kernel(paged_assign_kernel, dim3(kBlocks), dim3(kThreads), smem, stream, pdl, a, (int)(here && a.tokens > 0)) != cudaSuccess) return 0;
  if (here) return 1;
  return launch_kernel(paged_slots_kernel, dim3((unsigned)((a.tokens + kSlotThreads - 1) / kSlotThreads)), dim3(kSlotThreads), 0, stream, true, a) == cudaSuccess
             ? 2
             : 0;
}

int paged_path_launch(const PagedPath& a, bool pdl, cudaStream_t stream) {
  constexpr int kPerBlock = kPathThreads / 32;
  return launch_kernel(paged_path_kernel, dim3((unsigned)((a.batch + kPerBlock - 1) / kPerBlock)), dim3(kPathThreads), 0, stream, pdl, a) == cudaSuccess;
}

}  // namespace pjrtx
