// Attention of trees of drafted tokens in 16 bits on the 5th-generation tensor cores (formulas, tiles and shares: tree_attention.cu).
//
// A block of threads goes through its share as one row of steps, a step being a block of keys of a segment, and nothing drains between
// segments: rows of the next one are fetched while the last ones of this are at work.
//   loader warps   two; queries of a segment, then keys and values of the steps into a ring of shared-memory slots, by cp.async: a row
//                  of a page is the longest run that is contiguous whatever the layout. Rows are written in the 128-byte swizzle that the
//                  tensor core reads, and handed over some slots later, when they have landed
//   MMA warp       S = Q . K^T, O += P . V with P in tensor memory. With one tile of 128 query rows the scores have two buffers, so
//                  that those of the next step are there when the softmax warps are done; with two tiles these take turns
//   softmax warps  four a tile, a query row a thread; those whose rows are not there only count along
//
// Bound by memory up to two tiles: 128 keys of 128 elements are 64 KB of keys and values, 2800 cycles of this SM's share of the memory, and
// take 1024 cycles of tensor core and of exponentials for each tile.
//
// Hidden nodes have probability 0, and 0 times infinity or NaN is NaN on the tensor core. So a node with such a value goes into shared memory
// as zeros, and rows that see it add their probability times its values when they take their results out. Rounding and the lazily
// followed maximum: umma_rows.cuh.
#pragma once

#include "umma_rows.cuh"

namespace pjrtx {
namespace umma {

constexpr int kTreeLoaders = 2, kOddRing = 16;
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
// Four softmax warps a tile, the loaders, the warp that issues, and one that has nothing to do: eight or twelve, which divide the registers evenly.
__host__ __device__ constexpr int tree_threads(int tiles) { return 128 * tiles + 128; }

struct TreeKernelArgs {
  TreeArgs p;
  float scale_log2, sign;  // scale: |scale| * log2(e), 1 where it is zero, and its sign, by which scores are multiplied first
  unsigned long long timeout_ns;
};

__device__ __forceinline__ void row_copy16(uint32_t to, unsigned long long from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void row_copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

template <bool BF16, int HD, int TILES>
__global__ void __launch_bounds__(tree_threads(TILES), 1) umma_tree_kernel(const __grid_constant__ TreeKernelArgs a) {
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
    uint64_t odd_ready[kOddRing];       // of a segment
    unsigned long long odd[kOddRing][kTreeLoaders];  // nodes with values that are infinite or NaN
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
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const TreeArgs& p = a.p;
  if (threadIdx.x == 0) p.cuts[blockIdx.x] = {0, 0, 0, 0};
  check_sequences(p);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kQueries; i++) {
      mbar_init(&bar.q_full[i], kTreeLoaders);
      mbar_init(&bar.q_empty[i], 1);
    }
    for (int i = 0; i < kSlots; i++) {
      mbar_init(&bar.slot_full[i], kTreeLoaders);
      mbar_init(&bar.slot_empty[i], 1);
    }
    for (int t = 0; t < TILES; t++)
      for (int i = 0; i < kBuffers; i++) {
        mbar_init(&bar.s_full[t][i], 1);
        mbar_init(&bar.p_ready[t][i], 4);
      }
    for (int i = 0; i < kOddRing; i++) mbar_init(&bar.odd_ready[i], kTreeLoaders);
    bar.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar.tmem)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const Share share = share_of_block(p, bar.share);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem_base = bar.tmem;
  const bool work = share.first < share.size;
  auto s_col = [&](int t, int buffer) { return tmem_base + (uint32_t)((t * kBuffers + buffer) * kKeys); };
  auto o_col = [&](int t) { return tmem_base + (uint32_t)(TILES * kBuffers * kKeys + t * HD); };
  WaitBudget budget{global_timer_ns() + a.timeout_ns, &bar.abort};  // renewed with every segment
  auto renew = [&]() { budget.deadline = global_timer_ns() + a.timeout_ns; };
  auto wait = [&](uint64_t* b, unsigned parity) { return __all_sync(0xffffffffu, mbar_wait(b, parity, budget)) != 0; };

  if (warp >= kFirstLoader && warp < kMmaWarp) {
    const int lw = warp - kFirstLoader;
    constexpr int kLag = kSlots - 2;  // copies under way, in groups
    constexpr int kPieces = HD / 8, kAcross = 32 / kPieces, kRowsOfWarp = kKeys / kTreeLoaders, kRowsOfLane = kRowsOfWarp / 32;
    uint32_t pending[kLag];  // barriers of the groups that have not been handed over, the oldest first
#pragma unroll
    for (int i = 0; i < kLag; i++) pending[i] = 0;
    auto hand_over = [&](uint32_t b) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (b && lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(b) : "memory");
    };
    auto commit = [&](uint64_t* b) {
      asm volatile("cp.async.commit_group;" ::: "memory");
      row_copies_wait<kLag>();
      hand_over(pending[0]);
#pragma unroll
      for (int i = 0; i + 1 < kLag; i++) pending[i] = pending[i + 1];
      pending[kLag - 1] = smem_u32(b);
    };
    auto drain = [&]() {
      row_copies_wait<0>();
#pragma unroll
      for (int i = 0; i < kLag; i++) {
        hand_over(pending[i]);
        pending[i] = 0;
      }
    };
    // Address of the key of row `lane` of the warp's i-th 32 in the step's block: bit 0 marks a node, 0 stands for none.
    auto locate_row = [&](const Cursor& u, int g, int i) -> unsigned long long {
      const int t = u.tile * kKeys + lw * kRowsOfWarp + i * 32 + lane;
      if (t < u.s.length) {
        const long long row = cached_row(p, u.b, t);
        return row < 0 ? 0ull : (unsigned long long)(static_cast<const unsigned short*>(p.c.k) + row + g * p.c.head_stride);
      }
      const int node = t - u.s.length;
      if (node >= u.s.count) return 0ull;
      return (unsigned long long)(static_cast<const unsigned short*>(p.a.k_new) + u.b * p.a.new_batch_stride + node * p.a.new_node_stride +
                                  g * p.a.new_head_stride) | 1ull;
    };
    struct Keys {
      unsigned long long at[kRowsOfLane];
    };
    auto locate = [&](const Cursor& u, int g) {
      Keys k;
#pragma unroll
      for (int i = 0; i < kRowsOfLane; i++) k.at[i] = locate_row(u, g, i);
      return k;
    };
    const unsigned long long apart = (unsigned long long)p.c.v - (unsigned long long)p.c.k;
    const unsigned long long apart_new = (unsigned long long)p.a.v_new - (unsigned long long)p.a.k_new;
    const int piece = lane % kPieces;
    const bool inside = piece * 8 < p.c.head_dim;
    int slot = 0;
    unsigned phase = 0;
    long long used = 0;
    auto take_slot = [&](uint32_t* at) {  // false: given up
      if (used++ >= kSlots && !wait(&bar.slot_empty[slot], phase ^ 1)) return false;
      *at = ring + (uint32_t)slot * kSlotBytes;
      return true;
    };
    auto next_slot = [&]() {
      commit(&bar.slot_full[slot]);
      if (++slot == kSlots) {
        slot = 0;
        phase ^= 1;
      }
    };
    auto place = [&](uint32_t at, int row) { return at + (uint32_t)(piece / 8) * kKeyBlock + (uint32_t)row * 128u + (uint32_t)(((piece & 7) ^ (row & 7)) << 4); };
    auto load_keys = [&](const Keys& key) {
      uint32_t at;
      if (!take_slot(&at)) return false;
#pragma unroll
      for (int i = 0; i < kRowsOfLane; i++)
#pragma unroll 4
        for (int j = 0; j < 32 / kAcross; j++) {
          const int r = j * kAcross + lane / kPieces;
          const unsigned long long from = __shfl_sync(~0u, key.at[i], r) & ~1ull;
          row_copy16(place(at, lw * kRowsOfWarp + i * 32 + r), from && inside ? from + piece * 16 : (unsigned long long)p.c.k, from && inside);
        }
      next_slot();
      return true;
    };
    unsigned long long odd = 0;
    auto load_values = [&](const Keys& key, const Cursor& u) {
      uint32_t at;
      if (!take_slot(&at)) return false;
#pragma unroll
      for (int i = 0; i < kRowsOfLane; i++) {
        const bool nodes = __any_sync(~0u, key.at[i] & 1);
#pragma unroll 4
        for (int j = 0; j < 32 / kAcross; j++) {
          const int r = j * kAcross + lane / kPieces, row = lw * kRowsOfWarp + i * 32 + r;
          unsigned long long from = __shfl_sync(~0u, key.at[i], r);
          const bool node = from & 1, there = from && inside;
          from = (from & ~1ull) + (node ? apart_new : apart) + piece * 16;
          if (!nodes) {
            row_copy16(place(at, row), there ? from : (unsigned long long)p.c.v, there);
            continue;
          }
          uint4 x = make_uint4(0, 0, 0, 0);
          if (there) x = *reinterpret_cast<const uint4*>(from);
          const bool bad = node && (odd_pair<BF16>(x.x) || odd_pair<BF16>(x.y) || odd_pair<BF16>(x.z) || odd_pair<BF16>(x.w));
          // Whether any lane of the row has found one.
          const unsigned found = __ballot_sync(~0u, bad) >> (lane / kPieces * kPieces) & (unsigned)((1ull << kPieces) - 1);
          if (found) {
            x = make_uint4(0, 0, 0, 0);
            odd |= 1ull << (u.tile * kKeys + row - u.s.length);
          }
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place(at, row)), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
        }
      }
      next_slot();
      return true;
    };
    auto load_queries = [&](const Segment& seg, long long number) {
      const int buffer = (int)(number % kQueries);
      if (number >= kQueries) {
        drain();  // the products that the buffer waits for may need what is under way
        if (!wait(&bar.q_empty[buffer], (unsigned)(number / kQueries - 1) & 1u)) return false;
      }
      const uint32_t at = base + buffer * kQueryBytes;
      constexpr int kEach = TILES * kAttnRows / kTreeLoaders;
      for (int j = 0; j < kEach / kAcross; j++) {
        const int r = lw * kEach + j * kAcross + lane / kPieces, tile = r / kAttnRows, row = r % kAttnRows;
        int node, head;
        const bool there = seg.place(p, r, &node, &head) && inside;
        const unsigned short* from = static_cast<const unsigned short*>(p.a.q);
        if (there) from += query_at(p, seg, node, head) + piece * 8;
        row_copy16(at + tile * kTileBytes + (uint32_t)(piece / 8) * kQueryBlock + (uint32_t)row * 128u + (uint32_t)(((piece & 7) ^ (row & 7)) << 4),
                   (unsigned long long)from, there);
      }
      commit(&bar.q_full[buffer]);
      return true;
    };
    if (work) {
      // Keys run `kBuffers` steps ahead of the values, as the products do.
      Cursor key_at = share.at, value_at = share.at;
      long long key_number = share.first, value_number = share.first, segments = 0, value_segment = 0;
      bool keys_left = true, ok = true, fresh = true;
      Keys place_of[kBuffers + 1];  // keys of the steps whose values are still to come
      int g = segment_of(p, key_at.b, key_at.group, key_at.s.count).g;
      Keys next = locate(key_at, g);
      auto step_keys = [&](int into) {
        if (fresh) {
          renew();
          ok = load_queries(segment_of(p, key_at.b, key_at.group, key_at.s.count), segments++);
          if (!ok) return;
        }
        place_of[into] = next;
        ok = load_keys(next);
        const int b = key_at.b, group = key_at.group;
        keys_left = next_unit(p, key_at, key_number, share.size);
        fresh = key_at.b != b || key_at.group != group;
        if (keys_left) {
          if (fresh) g = segment_of(p, key_at.b, key_at.group, key_at.s.count).g;
          next = locate(key_at, g);
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
        ok = load_values(place_of[0], value_at);
        if (!ok) break;
        const Cursor here = value_at;
        const bool more = next_unit(p, value_at, value_number, share.size);
        if (!more || value_at.b != here.b || value_at.group != here.group) {
          odd |= __shfl_xor_sync(~0u, odd, 16);  // lanes of different rows
          if (kPieces <= 8) odd |= __shfl_xor_sync(~0u, odd, 8);
          if (lane == 0) {
            bar.odd[value_segment % kOddRing][lw] = odd;
            mbar_arrive(&bar.odd_ready[value_segment % kOddRing]);
          }
          value_segment++;
          odd = 0;
        }
#pragma unroll
        for (int i = 0; i + 1 < kBuffers; i++) place_of[i] = place_of[i + 1];
        ahead--;
        if (keys_left) {
          step_keys(kBuffers - 1);
          ahead++;
        }
      }
      drain();
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
      for (long long step = 0; ok; step++) {
        const int buffer = (int)(step % kBuffers), v_slot = slot;
        ok = wait(&bar.slot_full[slot], phase);
        next_slot();
        const bool more = left;
        if (more) scores_wait();
#pragma unroll
        for (int t = 0; t < TILES; t++) {
          ok = ok && wait(&bar.p_ready[t][buffer], (unsigned)(step / kBuffers) & 1u);
          if (!ok) continue;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (leader) {
            const uint64_t v = desc_advance(v_first, (uint32_t)v_slot * kSlotBytes);
#pragma unroll
            for (int kk = 0; kk < kKeys / 16; kk++)
              mma_f16_tmem_a(o_col(t), s_col(t, buffer) + (uint32_t)kk * 8u, desc_advance(v, (uint32_t)kk * 2048u), idesc_o, (!first || kk) ? 1u : 0u);
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
      if (!ok && leader) report(p.c.error_words, kErrorWait);
      __syncwarp();
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
      const bool there = seg.place(p, row, &node, &head);
      const bool active = __any_sync(0xffffffffu, there);
      unsigned long long bits = 0;
      if (active) {
        const Ancestors above = tree_ancestors(p.a.parents + (long long)seg.b * p.a.nodes, p.a.nodes, p.c.error_words);
        bits = tree_of_node(above, there ? node : 0);
        if (!there) bits = 0;
      }
      float m_used = -INFINITY, sum = 0.f;
      int buffer = 0;
      for (bool first = true;; first = false, step++) {
        buffer = (int)(step % kBuffers);
        const uint32_t s_addr = s_col(t, buffer) + lanes;
        ok = wait(&bar.s_full[t][buffer], (unsigned)(step / kBuffers) & 1u);
        if (!ok) break;
        if (active) {
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          // Columns c * kChunk on, hidden ones at -inf. Two tiles leave registers for half a block: the scores are then read twice.
          constexpr int kChunk = TILES == 2 ? 64 : kKeys;
          float s[kChunk];
          const int key0 = now.tile * kKeys;
          auto load = [&](int c) {
#pragma unroll
            for (int i = 0; i < kChunk / 32; i++) tmem_load_32(s_addr + c * kChunk + i * 32, s + i * 32);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            if (a.sign != 1.f) {
#pragma unroll
              for (int e = 0; e < kChunk; e++) s[e] *= a.sign;
            }
            if (key0 + kKeys > here.s.length) {
#pragma unroll
              for (int w = 0; w < kChunk / 32; w++) {
                const unsigned seen = there ? seen_word(key0 + c * kChunk + w * 32, here.s.length, bits) : 0u;
#pragma unroll
                for (int e = 0; e < 32; e++)
                  if (!(seen >> e & 1)) s[w * 32 + e] = -INFINITY;
              }
            }
          };
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
          for (int c = 0; c < kKeys / kChunk; c++) {
            load(c);
#pragma unroll
            for (int e = 0; e < kChunk; e += 8)
#pragma unroll
              for (int i = 0; i < 4; i++) mx[i] = max3(mx[i], s[e + 2 * i], s[e + 2 * i + 1]);
          }
          const float m_block = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;
          float corr = 1.f;
          if (m_block > m_used + Probability<BF16>::kGrow) {
            corr = exp2_approx(m_used - m_block);  // 0 the first time
            m_used = m_block;
            sum *= corr;
          }
          if (!first && __any_sync(0xffffffffu, corr != 1.f)) {
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
          const float shift = m_used == -INFINITY ? 0.f : Probability<BF16>::kLift - m_used;
          float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
          for (int c = 0; c < kKeys / kChunk; c++) {
            if (kChunk < kKeys) load(c);
#pragma unroll
            for (int h = 0; h < kChunk / 64; h++) {
              float packed[32];
#pragma unroll
              for (int e = 0; e < 32; e++) {
                const float x = exp2_approx(fmaf(s[h * 64 + 2 * e], a.scale_log2, shift));
                const float y = exp2_approx(fmaf(s[h * 64 + 2 * e + 1], a.scale_log2, shift));
                const uint32_t pair = pack_pair<BF16>(x, y);
                add_pair<BF16>(pair, part[(2 * e) & 3], part[(2 * e + 1) & 3]);
                packed[e] = __uint_as_float(pair);
              }
              tmem_store_32(s_addr + (c * kChunk / 64 + h) * 32, packed);
            }
          }
          sum += (part[0] + part[1]) + (part[2] + part[3]);
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.p_ready[t][buffer]);
        more = next_unit(p, now, number, share.size);
        if (!more || now.b != here.b || now.group != here.group) break;
      }
      // The results, once the last product is done.
      ok = ok && wait(&bar.s_full[t][buffer], (unsigned)(step / kBuffers + 1) & 1u) &&
           wait(&bar.odd_ready[segments % kOddRing], (unsigned)(segments / kOddRing) & 1u);
      step++;
      if (!ok) break;
      float* part = part_of(p, share, here, segment);
      if (!active) continue;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      unsigned long long odd = 0;
      for (int i = 0; i < kTreeLoaders; i++) odd |= bar.odd[segments % kOddRing][i];
      odd &= bits;
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
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<float4*>(part + row * HD + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
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
      if (part) *reinterpret_cast<float2*>(part + p.slot_rows * HD + 2 * row) = make_float2(m, sum);
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
