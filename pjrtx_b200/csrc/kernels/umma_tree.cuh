// Attention of trees of drafted tokens in 16 bits on the 5th-generation tensor cores (formulas, tiles and shares: tree_attention.cu).
//
// A block of threads goes through its share as one row of steps, a step being a block of keys of a segment, and nothing drains between
// segments: rows of the next one are fetched while the last ones of this are at work.
//   loader warps   four; queries of a segment, then keys and values of the steps into a ring of shared-memory slots, in the 128-byte
//                  swizzle that the tensor core reads. Blocks of cached rows come by tensor-map copies of a page's rows, where pages are
//                  8, 16 or a multiple of 32 rows; the last rows, nodes, and pages of other sizes by cp.async, a row at a time,
//                  each thread's copies counting themselves in on the slot's barrier when they have landed
//   MMA warp       S = Q . K^T, O += P . V with P in tensor memory. With one tile of 128 query rows the scores have two buffers, so
//                  that those of the next step are there when the softmax warps are done; with two tiles these take turns (blocks of
//                  64 keys, for which two buffers fit: 211 us, not 171, where 64 nodes of 64 heads see 65536 rows)
//   softmax warps  four a tile, a query row a thread; those whose rows are not there only count along
//
// Bound by memory up to two tiles, nearly: 128 keys of 128 elements are 64 KB of keys and values, 2650 cycles as measured in the middle of a long share
// (7 TB/s over all SMs), and take 1024 cycles of exponentials and, with two numbers a probability, 1536 of the tensor core for each tile. Around that stand
// 6 to 7 us of launch, shares, page ids and first rows, and 5 to 10 of the join: 16 sequences of up to 4096 rows, 16 nodes of 32 heads over 8, pages of 16
// rows 56 to 59 us (184 MB, 3.2 TB/s), one sequence of 65536 rows and 32 nodes 70 to 78, 517 rows and 8 nodes 14.1. 65536 rows and 64 nodes of 64 heads over
// 8, four tiles a KV head that read every row twice, 196 to 210 us: 137 GFLOP, of which half count twice, at 1.0 PFLOP/s, bound by two tiles' exponentials
// and their instructions taking turns with the tensor core; there is one buffer of scores a tile.
//
// Registers: the 14 warps of a block with two tiles are four on two of the SM's sub-partitions, so 128 a thread, and 64 bytes are spilled with rows of
// 128 elements (none with 64); ten warps with one tile take 162 to 168 and spill none.
//
// Hidden nodes have probability 0, and 0 times infinity or NaN is NaN on the tensor core. So a node with such a value is cleared in shared
// memory (one more warp, the cleaner, looks at the nodes' values where they have landed), and rows that see it add their probability times its values
// when they take their results out. The same product makes NaN of an infinite cached value where one of its probability's numbers is 0: a warp with a result
// that is not finite looks at that result's columns of the cached rows, and which infinities and NaN these have says what it is. Rounding and the lazily
// followed maximum: umma_rows.cuh.
#pragma once

#include "umma_rows.cuh"

namespace pjrtx {
namespace umma {

constexpr int kTreeLoaders = 4;
constexpr int kOddRing = 16, kCleanRing = 16;  // longer than a cleaner can be ahead, which has the slots
__host__ __device__ constexpr int tree_keys(int hd) { return hd == 256 ? 64 : 128; }
__host__ __device__ constexpr int tree_slot_bytes(int hd) { return tree_keys(hd) * hd * 2; }
__host__ __device__ constexpr int tree_query_buffers(int hd, int tiles) { return tiles == 1 && hd <= 128 ? 2 : 1; }
__host__ __device__ constexpr int tree_query_bytes(int hd, int tiles) { return tree_query_buffers(hd, tiles) * tiles * kAttnRows * hd * 2; }
constexpr int kTreeOther = 2048 + 1024;  // barriers and shares, and what aligning to 1024 bytes takes
// As many slots as fit, up to ten: more do not bring the rows any sooner.
__host__ __device__ constexpr int tree_slots(int hd, int tiles) {
  const int fit = (227 * 1024 - kTreeOther - tree_query_bytes(hd, tiles)) / tree_slot_bytes(hd);
  return fit < 10 ? fit : 10;
}
__host__ __device__ constexpr size_t tree_smem(int hd, int tiles) {
  const size_t bytes = (size_t)tree_query_bytes(hd, tiles) + (size_t)tree_slots(hd, tiles) * tree_slot_bytes(hd) + kTreeOther;
  const size_t least = least_smem(512);
  return bytes < least ? least : bytes;
}
// Four softmax warps a tile, the loaders, the warp that issues, the cleaner.
__host__ __device__ constexpr int tree_threads(int tiles) { return 128 * tiles + 32 * (kTreeLoaders + 2); }

struct TreeKernelArgs {
  TreeArgs p;
  float scale_log2, sign;  // scale: |scale| * log2(e), 1 where it is zero, and its sign, by which scores are multiplied first
  unsigned long long timeout_ns;
  int box;  // rows of a page that a tensor-map copy takes, a multiple of eight; 0: rows are copied one by one
};

// Rows of a box: as many as a page has, at most a loader's part of a block; 0 where blocks are not made of such.
inline int tree_box(int keys, int page_size) {
  const int most = keys / kTreeLoaders;
  const int box = page_size < most ? page_size : most;
  return box % 8 == 0 && most % box == 0 && page_size % box == 0 ? box : 0;
}

__device__ __forceinline__ void row_copy16(uint32_t to, unsigned long long from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
// A whole warp's wait. One for all places: see the loops of the loaders.
__device__ __noinline__ bool warp_wait(uint64_t* bar, unsigned parity, unsigned long long deadline, volatile int* abort) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, WaitBudget{deadline, abort})) != 0;
}

// Of keys key0 + 32 w .. + 31, those that a row sees.
__device__ __forceinline__ unsigned seen_word(int key0, int length, unsigned long long bits) {
  const int below = length - key0;  // cached rows among them and behind
  if (below >= 32) return ~0u;
  if (below > 0) return ((1u << below) - 1) | (unsigned)(bits << below);
  return below > -64 ? (unsigned)(bits >> -below) : 0u;
}

// Probability of a node for one query row, as the softmax warps have it.
template <bool BF16>
__device__ __noinline__ float node_probability(const TreeKernelArgs& a, const unsigned short* q, const unsigned short* k, float shift) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  float s = 0.f;
  for (int d = 0; d < a.p.c.head_dim; d += 8) {
    float x[8], y[8];
    rows::unpack16<T>(*reinterpret_cast<const uint4*>(q + d), x);
    rows::unpack16<T>(*reinterpret_cast<const uint4*>(k + d), y);
#pragma unroll
    for (int e = 0; e < 8; e++) s = fmaf(x[e], y[e], s);
  }
  return exp2_approx(fmaf(s * a.sign, a.scale_log2, shift));
}

// Of cached rows [first, end) of a sequence, for a whole warp.
template <bool BF16>
__device__ __noinline__ OddColumns cached_odd_columns(const TreeArgs& p, int b, int g, int c, int first, int end) {
  OddColumns all = {0, 0, 0};
  for (int t = first + threadIdx.x % 32; t < end; t += 32) {
    const long long row = cached_row(p, b, t);
    if (row < 0) continue;
    const long long at = row + g * p.c.head_stride;
    all.add(odd_columns<BF16>(static_cast<const unsigned short*>(p.c.k) + at, static_cast<const unsigned short*>(p.c.v) + at, c, p.c.head_dim));
  }
  __syncwarp();
  all.join_lanes();
  return all;
}

template <bool BF16, int HD, int TILES>
__global__ void __launch_bounds__(tree_threads(TILES), 1) umma_tree_kernel(const __grid_constant__ TreeKernelArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  constexpr int kThreads = tree_threads(TILES), kKeys = tree_keys(HD), kSlots = tree_slots(HD, TILES);
  constexpr int kBuffers = TILES == 1 ? 2 : 1;  // of scores, a tile
  constexpr int kQueries = tree_query_buffers(HD, TILES);
  constexpr uint32_t kQueryBytes = TILES * kAttnRows * HD * 2, kTileBytes = kAttnRows * HD * 2, kSlotBytes = kKeys * HD * 2;
  constexpr uint32_t kQueryBlock = kAttnRows * 128, kKeyBlock = kKeys * 128;  // bytes of 64 elements of all rows
  constexpr uint32_t kTmemCols = 512;
  static_assert(TILES * (kBuffers * kKeys + HD) <= kTmemCols && kSlots >= 4, "");
  struct Barriers {
    uint64_t q_full[kQueries], q_empty[kQueries], slot_full[kSlots], slot_empty[kSlots];
    uint64_t s_full[TILES][kBuffers];   // the step's scores are in tensor memory, and the products two uses back are done
    uint64_t p_ready[TILES][kBuffers];  // its probabilities are
    uint64_t clean[kCleanRing];         // nodes with values that are infinite or NaN have been cleared in the slot
    uint64_t odd_ready[kOddRing];       // of a segment
    uint64_t drained;                   // no product is under way
    unsigned long long odd[kOddRing];   // which nodes these are
    uint32_t tmem;
    int abort;
    ShareSpace<kThreads> share;
  };
  static_assert(sizeof(Barriers) <= kTreeOther - 1024, "");
  extern __shared__ unsigned char smem_dyn[];
  const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
  unsigned char* base_ptr = smem_dyn + (base - smem_u32(smem_dyn));
  const uint32_t ring = base + kQueries * kQueryBytes;
  Barriers& bar = *reinterpret_cast<Barriers*>(base_ptr + kQueries * kQueryBytes + kSlots * kSlotBytes);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kFirstLoader = 4 * TILES, kMmaWarp = kFirstLoader + kTreeLoaders;
  const TreeArgs& p = a.p;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kQueries; i++) {
      mbar_init(&bar.q_full[i], kTreeLoaders * 32);
      mbar_init(&bar.q_empty[i], 1);
    }
    for (int i = 0; i < kSlots; i++) {
      mbar_init(&bar.slot_full[i], kTreeLoaders * 32);
      mbar_init(&bar.slot_empty[i], 2);  // the products, and the cleaner: it sees every use of a slot, or could take one for another
    }
    for (int t = 0; t < TILES; t++)
      for (int i = 0; i < kBuffers; i++) {
        mbar_init(&bar.s_full[t][i], 1);
        mbar_init(&bar.p_ready[t][i], 4);
      }
    for (int i = 0; i < kCleanRing; i++) mbar_init(&bar.clean[i], 1);
    for (int i = 0; i < kOddRing; i++) mbar_init(&bar.odd_ready[i], 1);
    mbar_init(&bar.drained, 1);
    bar.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar.tmem)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // Tensor memory is asked for before the kernel in front has ended: no block of threads that holds some fits the SM beside this one.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (threadIdx.x == 0) p.cuts[blockIdx.x] = {};
  const Share share = share_of_block(p, bar.share);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem_base = bar.tmem;
  const bool work = share.first < share.size;
  auto s_col = [&](int t, int buffer) { return tmem_base + (uint32_t)((t * kBuffers + buffer) * kKeys); };
  auto o_col = [&](int t) { return tmem_base + (uint32_t)(TILES * kBuffers * kKeys + t * HD); };
  auto budget = budget_from_now(a.timeout_ns, &bar.abort);  // renewed with every segment
  auto renew = [&]() { budget = budget_from_now(a.timeout_ns, &bar.abort); };
  auto wait = [&](uint64_t* b, unsigned parity) { return warp_wait(b, parity, budget.deadline, budget.abort); };
  auto has_nodes = [&](const Cursor& u) { return (u.tile + 1) * kKeys > u.s.length; };

  if (warp >= kFirstLoader && warp < kMmaWarp) {
    const int lw = warp - kFirstLoader;
    const bool leader = elect_one();
    constexpr int kPieces = HD / 8, kAcross = 32 / kPieces, kRowsOfWarp = kKeys / kTreeLoaders;
    static_assert(kRowsOfWarp <= 32, "");
    // Counts this thread in once its copies so far have landed.
    auto arrive_when_landed = [&](uint64_t* b) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(b)) : "memory"); };
    // Page id of row `lane` of this warp's part of a block, fetched a step before it is looked at, or, for blocks of nothing but cached
    // rows whose pages are made of boxes, of box `lane`.
    auto first_key = [&](const Cursor& u) { return u.tile * kKeys + lw * kRowsOfWarp; };
    auto whole = [&](const Cursor& u) { return a.box > 0 && first_key(u) + kRowsOfWarp <= u.s.length; };
    auto fetch = [&](const Cursor& u) {
      const int t = first_key(u) + lane * (whole(u) ? a.box : 1);
      return t < min(u.s.length, first_key(u) + kRowsOfWarp) ? p.c.table[u.b * p.c.table_stride + column_of(p, t)] : 0;
    };
    // Address of the key of row `lane`: bit 0 marks a node, 0 stands for none.
    auto locate = [&](const Cursor& u, int g, int page) -> unsigned long long {
      const int t = first_key(u) + lane;
      if (lane >= kRowsOfWarp) return 0ull;
      if (t < u.s.length) {
        if (page < 0 || page >= p.c.num_pages) {
          report(p.c.error_words, kErrorPageId);
          return 0ull;
        }
        return (unsigned long long)(static_cast<const unsigned short*>(p.c.k) + page * p.c.page_stride +
                                    (t - column_of(p, t) * p.c.page_size) * p.c.row_stride + g * p.c.head_stride);
      }
      const int node = t - u.s.length;
      if (node >= u.s.count) return 0ull;
      return (unsigned long long)(static_cast<const unsigned short*>(p.a.k_new) + u.b * p.a.new_batch_stride + node * p.a.new_node_stride +
                                  g * p.a.new_head_stride) | 1ull;
    };
    const unsigned long long apart = (unsigned long long)p.c.v - (unsigned long long)p.c.k;
    const unsigned long long apart_new = (unsigned long long)p.a.v_new - (unsigned long long)p.a.k_new;
    const int piece = lane % kPieces;
    const bool inside = piece * 8 < p.c.head_dim;
    int slot = 0;
    unsigned phase = 0;
    long long used = 0;
    auto take_slot = [&](uint32_t* at) {  // false: given up
      if (used >= kSlots && !wait(&bar.slot_empty[slot], phase ^ 1)) return false;
      used++;
      *at = ring + (uint32_t)slot * kSlotBytes;
      return true;
    };
    auto advance_slot = [&]() {
      if (++slot == kSlots) {
        slot = 0;
        phase ^= 1;
      }
    };
    // Where this lane's piece of row `row` of a slot goes.
    auto place = [&](uint32_t at, int row) { return at + (uint32_t)(piece / 8) * kKeyBlock + (uint32_t)row * 128u + (uint32_t)(((piece & 7) ^ (row & 7)) << 4); };
    // The warp's rows one by one, `row` being the address of row `lane`, 0: none. The loops are not unrolled: the code of all roles runs side by
    // side, and what does not fit the instruction cache costs more than it saves (5.1 of a warp's 10 cycles an instruction before).
    auto copy_rows = [&](unsigned long long row, uint32_t at, int row0, const void* any) {
#pragma unroll 2
      for (int j = 0; j < kRowsOfWarp / kAcross; j++) {
        const int r = j * kAcross + lane / kPieces;
        const unsigned long long from = __shfl_sync(~0u, row, r);
        row_copy16(place(at, row0 + r), from && inside ? from + piece * 16 : (unsigned long long)any, from && inside);
      }
    };
    // A page outside the pool: a box of nothing, which the copy fills with zeros.
    auto load_boxes = [&](const CUtensorMap* map, const Cursor& u, int g, int pages, uint32_t at) {
      if (leader) mbar_expect_tx(&bar.slot_full[slot], kRowsOfWarp * HD * 2);
      __syncwarp();
      const uint32_t to = at + (uint32_t)(lw * kRowsOfWarp) * 128u;
      const int t = first_key(u), row = t - column_of(p, t) * p.c.page_size;  // 0 where a page has no more than a box
#pragma unroll 1
      for (int i = 0; i * a.box < kRowsOfWarp; i++) {
        const int page = __shfl_sync(~0u, pages, i);
        const bool valid = page >= 0 && page < p.c.num_pages;
        if (leader) {
          if (!valid) report(p.c.error_words, kErrorPageId);
#pragma unroll
          for (int c = 0; c < HD / 64; c++)
            tma_load_4d(to + (uint32_t)c * kKeyBlock + (uint32_t)(i * a.box) * 128u, map, c * 64, row, g, valid ? page : (int)p.c.num_pages,
                        &bar.slot_full[slot]);
        }
      }
      __syncwarp();
      if (!leader) mbar_arrive(&bar.slot_full[slot]);
      advance_slot();
    };
    // Keys, or values.
    auto load_block = [&](bool values, const Cursor& u, int g, int pages) {
      uint32_t at;
      if (!take_slot(&at)) return false;
      if (whole(u)) {
        load_boxes(values ? &vmap : &kmap, u, g, pages, at);
        return true;
      }
      unsigned long long row = locate(u, g, pages);
      if (row) row = (row & ~1ull) + (values ? row & 1 ? apart_new : apart : 0);
      copy_rows(row, at, lw * kRowsOfWarp, p.c.k);
      arrive_when_landed(&bar.slot_full[slot]);
      advance_slot();
      return true;
    };
    auto load_queries = [&](const Segment& seg, long long number) {
      const int buffer = (int)(number % kQueries);
      if (number >= kQueries && !wait(&bar.q_empty[buffer], (unsigned)(number / kQueries - 1) & 1u)) return false;
      const uint32_t at = base + buffer * kQueryBytes;
      constexpr int kEach = TILES * kAttnRows / kTreeLoaders;
#pragma unroll 1
      for (int i = 0; i < kEach; i += 32) {
        const int r0 = lw * kEach + i, tile = r0 / kAttnRows;
        int node, head;
        unsigned long long row = 0;
        if (seg.place(p.heads, r0 + lane, &node, &head))
          row = (unsigned long long)(static_cast<const unsigned short*>(p.a.q) + query_at(p, seg, node, head));
#pragma unroll 2
        for (int j = 0; j < 32 / kAcross; j++) {
          const int r = r0 % kAttnRows + j * kAcross + lane / kPieces;
          const unsigned long long from = __shfl_sync(~0u, row, j * kAcross + lane / kPieces);
          row_copy16(at + tile * kTileBytes + (uint32_t)(piece / 8) * kQueryBlock + (uint32_t)r * 128u + (uint32_t)(((piece & 7) ^ (r & 7)) << 4),
                     from && inside ? from + piece * 16 : (unsigned long long)p.a.q, from && inside);
        }
      }
      arrive_when_landed(&bar.q_full[buffer]);
      return true;
    };
    if (work) {
      // Keys run `kBuffers` steps ahead of the values, as the products do.
      Cursor key_at = share.at, value_at = share.at;
      long long key_number = share.first, value_number = share.first, segments = 0;
      bool keys_left = true, ok = true, fresh = true;
      int pages[kBuffers + 1];  // of the steps whose values are still to come
      int g = segment_of(p, key_at.b, key_at.group, key_at.s.count).g, value_g = g;
      int next = fetch(key_at);
      auto step_keys = [&](int into) {
        if (fresh) {
          renew();
          ok = load_queries(segment_of(p, key_at.b, key_at.group, key_at.s.count), segments++);
          if (!ok) return;
        }
        pages[into] = next;
        ok = load_block(false, key_at, g, next);
        const int b = key_at.b, group = key_at.group;
        keys_left = next_unit(p, key_at, key_number, share.size);
        fresh = key_at.b != b || key_at.group != group;
        if (keys_left) {
          if (fresh) g = segment_of(p, key_at.b, key_at.group, key_at.s.count).g;
          next = fetch(key_at);
        }
      };
      int ahead = 0;
#pragma unroll
      for (int i = 0; i < kBuffers; i++)
        if (ok && keys_left) {
          step_keys(i);
          ahead++;
        }
      while (ok && ahead > 0) {
        ok = load_block(true, value_at, value_g, pages[0]);
        if (!ok) break;
        const int b = value_at.b, group = value_at.group;
        if (next_unit(p, value_at, value_number, share.size) && (value_at.b != b || value_at.group != group))
          value_g = segment_of(p, value_at.b, value_at.group, value_at.s.count).g;
#pragma unroll
        for (int i = 0; i + 1 < kBuffers; i++) pages[i] = pages[i + 1];
        ahead--;
        if (keys_left) {
          step_keys(kBuffers - 1);
          ahead++;
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      const unsigned long long until = global_timer_ns() + kLandNs;
      for (long long u = used - 1; u >= 0 && u >= used - kSlots; u--) wait_landed(&bar.slot_full[u % kSlots], (unsigned)(u / kSlots) & 1u, until);
    }
  } else if (warp == kMmaWarp) {
    const bool leader = elect_one();
    // N = keys with K as a K-major B operand; N = HD with V as an MN-major one (bit 16).
    const uint32_t idesc_s = instr_desc(BF16, kKeys, 0);
    const uint32_t idesc_o = instr_desc(BF16, HD, 0) | 1u << 16;
    const uint64_t q_first = smem_desc(base, 16, 1024), k_first = smem_desc(ring, 16, 1024), v_first = smem_desc(ring, kKeyBlock, 1024);
    int slot = 0;
    unsigned phase = 0;
    auto next_slot = [&]() {
      if (++slot == kSlots) {
        slot = 0;
        phase ^= 1;
      }
    };
    if (work) {
      Cursor ahead = share.at, now = share.at;
      long long ahead_number = share.first, number = share.first, ahead_step = 0, ahead_segment = 0;
      bool left = true, fresh = true, ok = true;
      int k_slot = 0;
      // Scores of step `ahead`: `scores_wait` before, `scores` for every tile, `scores_done` behind.
      auto scores_wait = [&]() {
        if (fresh) {
          renew();
          ok = ok && wait(&bar.q_full[ahead_segment % kQueries], (unsigned)(ahead_segment / kQueries) & 1u);
        }
        k_slot = slot;
        ok = ok && wait(&bar.slot_full[slot], phase);
        next_slot();
      };
      auto scores = [&](int t) {
        const uint64_t q = desc_advance(q_first, (uint32_t)(ahead_segment % kQueries) * kQueryBytes + t * kTileBytes);
        const uint64_t k = desc_advance(k_first, (uint32_t)k_slot * kSlotBytes);
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk++)
          mma_f16(s_col(t, (int)(ahead_step % kBuffers)), desc_advance(q, (uint32_t)(kk >> 2) * kQueryBlock + (uint32_t)(kk & 3) * 32u),
                  desc_advance(k, (uint32_t)(kk >> 2) * kKeyBlock + (uint32_t)(kk & 3) * 32u), idesc_s, kk ? 1u : 0u);
      };
      auto scores_done = [&]() {
        if (leader) mma_commit(&bar.slot_empty[k_slot]);
        const Cursor here = ahead;
        left = next_unit(p, ahead, ahead_number, share.size);
        fresh = !left || ahead.b != here.b || ahead.group != here.group;
        if (fresh) {
          if (leader) mma_commit(&bar.q_empty[ahead_segment % kQueries]);
          ahead_segment++;
        }
        ahead_step++;
        __syncwarp();
      };
#pragma unroll
      for (int i = 0; i < kBuffers; i++)
        if (ok && left) {
          scores_wait();
          if (!ok) break;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the copies are seen by the threads' own accesses first
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (leader)
            for (int t = 0; t < TILES; t++) {
              scores(t);
              mma_commit(&bar.s_full[t][i]);
            }
          __syncwarp();
          scores_done();
        }
      bool first = true;
      long long checked = 0;
      for (long long step = 0; ok; step++) {
        const int buffer = (int)(step % kBuffers), v_slot = slot;
        ok = wait(&bar.slot_full[slot], phase);
        next_slot();
        const bool more = left;
        if (more) scores_wait();
        if (has_nodes(now)) {
          ok = ok && wait(&bar.clean[checked % kCleanRing], (unsigned)(checked / kCleanRing) & 1u);
          checked++;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
#pragma unroll
        for (int t = 0; t < TILES; t++) {
          ok = ok && wait(&bar.p_ready[t][buffer], (unsigned)(step / kBuffers) & 1u);
          if (!ok) continue;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (leader) {
            const uint64_t v = desc_advance(v_first, (uint32_t)v_slot * kSlotBytes);
#pragma unroll
            for (int kk = 0; kk < kKeys / 16; kk++)
              mma_values(o_col(t), s_col(t, buffer) + (uint32_t)kk * 16u, desc_advance(v, (uint32_t)kk * 2048u), idesc_o, (!first || kk) ? 1u : 0u);
            if (more) scores(t);
            mma_commit(&bar.s_full[t][buffer]);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (leader) mma_commit(&bar.slot_empty[v_slot]);
        __syncwarp();
        if (more) scores_done();
        const Cursor here = now;
        if (!next_unit(p, now, number, share.size)) break;
        first = now.b != here.b || now.group != here.group;
      }
      if (leader) {
        if (!ok) report(p.c.error_words, kErrorWait);
        mma_commit(&bar.drained);
        wait_landed(&bar.drained, 0, global_timer_ns() + kLandNs);
      }
      __syncwarp();
    }
  } else if (warp == kMmaWarp + 1) {
    // The cleaner: looks at the values of nodes where they have landed.
    Cursor now = share.at;
    long long number = share.first, used = 0, checked = 0, segments = 0;
    unsigned long long odd = 0;
    bool left = work, more_keys = true, fresh = true;
    // Slots in the order in which they are used: `kBuffers` steps of keys, then a step's values and the keys `kBuffers` further on.
    Cursor ahead = share.at;
    long long ahead_number = share.first;
    bool ok = true;
    auto next_use = [&]() {
      const int slot = (int)(used % kSlots);
      ok = ok && wait(&bar.slot_full[slot], (unsigned)(used / kSlots) & 1u);
      used++;
      return slot;
    };
    auto pass = [&](int slot) {
      if (ok && lane == 0) mbar_arrive(&bar.slot_empty[slot]);
    };
    auto pass_keys = [&]() {
      pass(next_use());
      more_keys = next_unit(p, ahead, ahead_number, share.size);
    };
    for (int i = 0; i < kBuffers && left && more_keys; i++) pass_keys();
    while (left && ok) {
      if (fresh) renew();
      const int slot = next_use();
      if (ok && has_nodes(now)) {
        const int from = max(0, now.s.length - now.tile * kKeys), to = min(kKeys, now.s.length + now.s.count - now.tile * kKeys);
        unsigned char* rows0 = base_ptr + kQueries * kQueryBytes + slot * kSlotBytes;
        constexpr int kPieces = HD / 8, kAcross = 32 / kPieces;
        const int piece = lane % kPieces;
#pragma unroll 4
        for (int r0 = from; r0 < to; r0 += kAcross) {
          const int r = r0 + lane / kPieces;
          uint4* const at = reinterpret_cast<uint4*>(rows0 + (piece / 8) * kKeyBlock + r * 128 + (((piece & 7) ^ (r & 7)) << 4));
          bool bad = false;
          if (r < to) {
            const uint4 x = *at;
            bad = odd_pair<BF16>(x.x) || odd_pair<BF16>(x.y) || odd_pair<BF16>(x.z) || odd_pair<BF16>(x.w);
          }
          // Whether any lane of the row has found one.
          if (__ballot_sync(~0u, bad) >> (lane / kPieces * kPieces) & (unsigned)((1ull << kPieces) - 1)) {
            *at = make_uint4(0, 0, 0, 0);
            odd |= 1ull << (now.tile * kKeys + r - now.s.length);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.clean[checked % kCleanRing]);
        checked++;
      }
      pass(slot);
      if (more_keys) pass_keys();
      const int b = now.b, group = now.group;
      left = next_unit(p, now, number, share.size);
      fresh = !left || now.b != b || now.group != group;
      if (fresh) {
        odd |= __shfl_xor_sync(~0u, odd, 16);  // lanes of different rows
        odd |= __shfl_xor_sync(~0u, odd, 8);
        if (lane == 0) {
          bar.odd[segments % kOddRing] = odd;
          mbar_arrive(&bar.odd_ready[segments % kOddRing]);
        }
        segments++;
        odd = 0;
      }
    }
  } else if (warp < kFirstLoader) {
    const int t = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_addr = o_col(t) + lanes;
    const int row = t * kAttnRows + (warp & 3) * 32 + lane;
    Cursor now = share.at;
    long long number = share.first, step = 0, segments = 0;
    bool ok = true;
    for (bool more = work; more && ok; segments++) {
      renew();
      const Cursor here = now;
      const Segment seg = segment_of(p, here.b, here.group, here.s.count);
      const long long segment = share.begin + number - here.tile;  // number of its first unit
      int node, head;
      const bool there = seg.place(p.heads, row, &node, &head);
      const bool active = __any_sync(0xffffffffu, there);
      unsigned long long bits = 0;
      if (active) {
        const Ancestors above = tree_ancestors(p.a.parents + (long long)seg.b * p.a.nodes, here.s.count, p.c.error_words);
        bits = tree_of_node(above, there ? node : 0);
        if (!there) bits = 0;
      }
      float m_used = -INFINITY, sum = 0.f;
      int buffer = 0, tile_end = here.tile;
      for (bool first = true;; first = false, step++) {
        buffer = (int)(step % kBuffers);
        const uint32_t s_addr = s_col(t, buffer) + lanes;
        ok = wait(&bar.s_full[t][buffer], (unsigned)(step / kBuffers) & 1u);
        if (!ok) break;
        if (active) {
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          // The scores are read twice, in pieces, and the loops are not unrolled: that takes some 200 cycles, and the code is a fifth as
          // long. Where some are hidden or the scale is not positive, they go back as they are to be.
          const int key0 = now.tile * kKeys;
          const bool special = a.sign != 1.f || key0 + kKeys > here.s.length;
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, m_block = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < kKeys; c += 64) {
            float s[64];
            tmem_load_32(s_addr + c, s);
            tmem_load_32(s_addr + c + 32, s + 32);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            if (special) {
#pragma unroll
              for (int h = 0; h < 64; h += 32) {
                const unsigned seen = there ? seen_word(key0 + c + h, here.s.length, bits) : 0u;
#pragma unroll
                for (int e = 0; e < 32; e++) s[h + e] = seen >> e & 1 ? s[h + e] * a.sign : -INFINITY;
                tmem_store_32(s_addr + c + h, s + h);
              }
            }
            m_block = max_of<64>(s, mx);
          }
          m_block *= a.scale_log2;
          if (special) asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          if (__any_sync(0xffffffffu, m_block > m_used + Probability<BF16>::kGrow)) {
            const float top = fmaxf(m_used, m_block), corr = top == m_used ? 1.f : exp2_approx(m_used - top);  // 0 the first time
            m_used = top;
            sum *= corr;
            if (!first) {
              // With two buffers the product of the step before may still be adding to the results.
              if (kBuffers == 2) ok = wait(&bar.s_full[t][buffer ^ 1], (unsigned)((step - 1) / 2 + 1) & 1u);
              if (!ok) break;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
              for (int c = 0; c < HD; c += 32) {
                float o[32];
                tmem_load_32(o_addr + c, o);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] *= corr;
                tmem_store_32(o_addr + c, o);
              }
            }
          }
          const float shift = m_used == -INFINITY ? 0.f : Probability<BF16>::kLift - m_used;
          Pair part[2] = {0, 0};
          // One piece after the other: a second one on its way while the first is at work takes registers and code, and was slower (16 sequences of up to
          // 4096 rows and 16 nodes 62 us, not 59, 32 of up to 2048 and 40 nodes 107, not 101), as were pieces of 16 (60 and 105).
#pragma unroll 1
          for (int c = 0; c < kKeys; c += 32) {
            float s[32];
            tmem_load_32(s_addr + c, s);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            store_probabilities<BF16>(s, a.scale_log2, shift, part, s_addr + c);
          }
          const float2 block = pair_split(pair_add(part[0], part[1]));
          sum += block.x + block.y;
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.p_ready[t][buffer]);
        tile_end++;
        more = next_unit(p, now, number, share.size);
        if (!more || now.b != here.b || now.group != here.group) break;
      }
      // The results, once the last product is done.
      ok = ok && wait(&bar.s_full[t][buffer], (unsigned)(step / kBuffers + 1) & 1u) &&
           wait(&bar.odd_ready[segments % kOddRing], (unsigned)(segments / kOddRing) & 1u);
      step++;
      if (!ok) break;
      float* part = part_of(p, share, here, seg, segment);
      if (!active) continue;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned long long odd = bar.odd[segments % kOddRing] & bits;
      const float m = m_used - Probability<BF16>::kLift;  // what the sums are relative to
      const float shift = m_used == -INFINITY ? 0.f : -m;
      const float inverse = part ? 1.f : rows::inverse_of(sum);
      const long long fresh = seg.b * p.a.new_batch_stride + seg.g * p.a.new_head_stride;
      unsigned short* out = static_cast<unsigned short*>(p.a.out) + (there ? out_at(p, seg, node, head) : 0);
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        float o[32];
        tmem_load_32(o_addr + c, o);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        Pair nan = 0;
#pragma unroll
        for (int e = 0; e < 32; e += 2) nan = pair_fma(pair_of(o[e], o[e + 1]), 0, nan);
        const float2 sums = pair_split(nan);
        // Not where the sum is NaN, as every result then is.
        if (__any_sync(0xffffffffu, there && sums.x + sums.y != 0.f && sum == sum)) {
          OddColumns seen = cached_odd_columns<BF16>(p, seg.b, seg.g, c, here.tile * kKeys, min(tile_end * kKeys, here.s.length));
          if (sum == 0.f) seen = {seen.any(), 0, 0};
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (seen.any() >> e & 1) o[e] = seen.of(e);
        }
        if (!there) continue;
        for (unsigned long long left = odd; left; left &= left - 1) {
          using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
          const long long at = fresh + (__ffsll(left) - 1) * p.a.new_node_stride;
          const float w = node_probability<BF16>(a, static_cast<const unsigned short*>(p.a.q) + query_at(p, seg, node, head),
                                                 static_cast<const unsigned short*>(p.a.k_new) + at, shift);
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (c + e < p.c.head_dim) o[e] = fmaf(w, (float)(static_cast<const T*>(p.a.v_new) + at)[c + e], o[e]);
        }
        if (part) {
#pragma unroll
          for (int e = 0; e < 32; e++) part[(c + e) * p.slot_rows + row] = o[e];
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            if (c + e < p.c.head_dim)
              *reinterpret_cast<uint4*>(out + c + e) =
                  make_uint4(pack_pair<BF16>(o[e] * inverse, o[e + 1] * inverse), pack_pair<BF16>(o[e + 2] * inverse, o[e + 3] * inverse),
                             pack_pair<BF16>(o[e + 4] * inverse, o[e + 5] * inverse), pack_pair<BF16>(o[e + 6] * inverse, o[e + 7] * inverse));
        }
      }
      if (!there) continue;
      if (part) store_statistics(p, part, row, m, sum);
      else if (p.a.lse) p.a.lse[lse_at(p, seg, node, head)] = sum == 0.f ? -INFINITY : fmaf(m, rows::kLn2, logf(sum));
    }
    if (!ok && lane == 0) report(p.c.error_words, kErrorWait);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
}

}  // namespace umma
}  // namespace pjrtx
