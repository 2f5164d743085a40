// Causal attention of packed prompts on the 5th-generation tensor cores: scores, probabilities and results of a tile of 128 query rows
// stay in tensor memory while its keys pass by in blocks (the formulas and the tiles are those of prompt_attention.cu).
//
// Roles of a block of threads, which has one tile; an SM has two, which overlap what either waits for (of 256 dimensions one):
//   copy warp      the queries once, then keys and values, 64 at a time, into a ring of shared-memory slots (tiled tensor-map copies, 128-byte
//                  swizzle)
//   MMA warp       S = Q . K^T and O += P . V with P in tensor memory. The scores have two buffers, so that those of the next block are there
//                  when the softmax warps are done with one
//   softmax warps  four, a query row a thread (its lane of tensor memory), so a row's maximum and sum need no exchange
//
// What bounds it: a block of 128 rows and 64 keys of 128 elements takes 768 cycles of the tensor core's time (256 of scores, 512 of two products with
// the values) and 512 of the exponential unit's (8192 at 16 a cycle), and moves 112 KB through shared memory, 896 cycles at 128 bytes a cycle: the
// scores' product reads the queries (32 KB) and the block's keys, the other two the values, and the copies write both. Measured are 1300 to 1400 cycles,
// the tensor core 61 % busy, the exponential unit 41 %, issue slots 43 %. What fills the rest is not one unit but the order of things: a block's scores,
// maximum, exponentials and product follow each other, and two independent blocks of threads do not hide all of it from each other. Eight softmax
// warps a tile, four for every other block, which hand the rows' maxima to each other, gained nothing (with one number a probability, 4 x 2048 146 -> 155
// us). 8192 and 5461 tokens, 32 heads of 128 over 8 KV heads, masked halves left out: 933 to 1000 us in f16 and 856 to 876 in bf16, 0.8 to 0.9
// PFLOP/s that count, once more by half with the second product, in bursts; 1084 to 1130 from call to call, where the clock settles lower. 4 x 2048 181 to 185 us,
// with 8 heads of 64 47; one prompt of 517 tokens 11.6 us, where launch, first copies, nine blocks of keys one after the other and the way out follow
// each other.
//
// Exponentials all go to the exponential unit: a share of them by polynomials on the FMA units, as the tensor core's rate would want, made
// every case 2 to 15 % slower by the code and the issue slots that it takes. Scores that are read twice in loops, as in umma_tree.cuh, make it 2 to 4 %
// slower here.
//
// Two tiles in a block of threads of twice the size, with blocks of 128 keys that they share and buffers for one block of scores each, were slower up to
// 4096 tokens (with one number a probability, as are the present form's figures in brackets): 517 of 32 heads over 8 14.4 us (10.8), 64 x 20 28 (16),
// 4 x 2048 162 (149), 2 x 4096 258 (254); 2 x 8192 916 (947).
//
// Hidden keys have probability 0, but the tensor core multiplies it by their values, and 0 times infinity or NaN is NaN. So values
// behind the last position of the block of threads are cleared in shared memory, and a warp with a result that is not finite looks at that result's columns:
// which infinities and NaN a row sees says what its results are there, and a row with a result that only a hidden value has spoilt is computed once more, by
// the warp, without these and with probabilities in f32.
#pragma once

#include "umma_rows.cuh"

namespace pjrtx {
namespace umma {

struct PromptKernelArgs {
  PromptArgs p;       // `heads` and `positions` of one tile of 128 rows
  float scale_log2;   // |scale| * log2(e) (1 where scale is zero)
  float sign;         // 1, -1 or 0: what scores are multiplied by first, so that the largest score has the largest exponent
  unsigned long long timeout_ns;
};

constexpr int kPromptKeys = 64, kPromptThreads = 192;
__host__ __device__ constexpr int prompt_slots(int hd) { return hd == 256 ? 5 : hd == 128 ? 4 : 8; }
__host__ __device__ constexpr int prompt_per_sm(int hd) { return hd <= 128 ? 2 : 1; }
__host__ __device__ constexpr uint32_t prompt_tmem(int hd) { return prompt_per_sm(hd) == 2 ? 256 : 512; }
__host__ __device__ constexpr size_t prompt_smem(int hd) {
  const size_t bytes = (size_t)kAttnRows * hd * 2 + (size_t)prompt_slots(hd) * kPromptKeys * hd * 2 + 512 + 1024;
  const size_t least = least_smem(prompt_tmem(hd));
  return bytes < least ? least : bytes;
}
static_assert(prompt_smem(128) <= kSharedSmem && prompt_smem(64) <= kSharedSmem, "two blocks of threads an SM");

__device__ __forceinline__ void tma_load_3d(uint32_t smem_dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_dst),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
               : "memory");
}
// Row `pos` once more, over the keys that it sees; called by a whole warp, `m` and `total` being the row's.
template <bool BF16, int HD>
__device__ __noinline__ void redo_row(const PromptKernelArgs& a, const unsigned short* q, const unsigned short* k, const unsigned short* v,
                                      unsigned short* out, int pos, float m, float total) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const PromptAttention& p = a.p.a;
  const int lane = threadIdx.x % 32;
  float o[HD / 32];
#pragma unroll
  for (int e = 0; e < HD / 32; e++) o[e] = 0.f;
  const float shift = m == -INFINITY ? 0.f : Probability<BF16>::kLift - m;
  for (int key0 = 0; key0 <= pos; key0 += 32) {
    float s = 0.f;
    if (key0 + lane <= pos) {
      const unsigned short* row = k + (key0 + lane) * p.k_stride;
      for (int d = 0; d < p.head_dim; d += 8) {
        float x[8], y[8];
        rows::unpack16<T>(*reinterpret_cast<const uint4*>(row + d), x);
        rows::unpack16<T>(*reinterpret_cast<const uint4*>(q + d), y);
#pragma unroll
        for (int e = 0; e < 8; e++) s = fmaf(x[e], y[e], s);
      }
      s = exp2_approx(fmaf(s * a.sign, a.scale_log2, shift));
    }
    for (int i = 0; i < 32 && key0 + i <= pos; i++) {
      const float w = __shfl_sync(0xffffffffu, s, i);
      const unsigned short* row = v + (key0 + i) * p.v_stride;
#pragma unroll
      for (int e = 0; e < HD / 32; e++)
        if (e * 32 + lane < p.head_dim) o[e] = fmaf(w, (float)reinterpret_cast<const T*>(row)[e * 32 + lane], o[e]);
    }
  }
  const float inverse = rows::inverse_of(total);
#pragma unroll
  for (int e = 0; e < HD / 32; e++)
    if (e * 32 + lane < p.head_dim) reinterpret_cast<T*>(out)[e * 32 + lane] = rows::from_float<T>(o[e] * inverse);
}

// Of the keys up to `pos`, for all lanes of a warp, whose positions are first_pos .. last_pos (some lanes may have none).
template <bool BF16>
__device__ __noinline__ OddColumns prompt_odd_columns(const PromptAttention& p, const unsigned short* k, const unsigned short* v, int c, int first_pos, int last_pos,
                                                      int pos) {
  const int lane = threadIdx.x % 32;
  OddColumns all = {0, 0, 0};
  for (int key = lane; key <= first_pos; key += 32) all.add(odd_columns<BF16>(k + key * p.k_stride, v + key * p.v_stride, c, p.head_dim));
  all.join_lanes();
  for (int key0 = first_pos + 1; key0 <= last_pos; key0 += 32) {
    OddColumns mine = {0, 0, 0};
    if (key0 + lane <= last_pos) mine = odd_columns<BF16>(k + (key0 + lane) * p.k_stride, v + (key0 + lane) * p.v_stride, c, p.head_dim);
    __syncwarp();
    for (int i = 0; i < 32; i++) {
      const OddColumns of_key = {__shfl_sync(0xffffffffu, mine.nan, i), __shfl_sync(0xffffffffu, mine.plus, i), __shfl_sync(0xffffffffu, mine.minus, i)};
      if (key0 + i <= pos) all.add(of_key);
    }
  }
  return all;
}

template <bool BF16, int HD>
__global__ void __launch_bounds__(kPromptThreads, prompt_per_sm(HD))
umma_prompt_kernel(const __grid_constant__ PromptKernelArgs a, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap) {
  constexpr int kKeys = kPromptKeys, kHalves = HD / 64, kSlots = prompt_slots(HD);
  constexpr uint32_t kTileBytes = kAttnRows * HD * 2, kSlotBytes = kKeys * HD * 2;
  constexpr uint32_t kQueryBlock = kAttnRows * 128, kKeyBlock = kKeys * 128;  // bytes of 64 elements of all rows
  constexpr uint32_t kTmemCols = prompt_tmem(HD);
  static_assert(kKeys == 64 && 2 * kKeys + HD <= kTmemCols, "");
  extern __shared__ unsigned char smem_dyn[];
  const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
  unsigned char* base_ptr = smem_dyn + (base - smem_u32(smem_dyn));
  const uint32_t ring = base + kTileBytes;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(base_ptr + kTileBytes + kSlots * kSlotBytes);
  uint64_t* slot_full = q_full + 1;             // [kSlots]
  uint64_t* slot_empty = slot_full + kSlots;    // [kSlots]
  uint64_t* v_clean = slot_empty + kSlots;      // values behind the last position have been cleared
  uint64_t* s_full = v_clean + 1;  // [2] scores of a block are in tensor memory, and the product two blocks before it is done
  uint64_t* p_ready = s_full + 2;  // [2] its probabilities are
  uint64_t* drained = p_ready + 2;  // no product is under way
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  int* flags = reinterpret_cast<int*>(tmem_slot + 1);  // [0] abort

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kMmaWarp = 4, kCopyWarp = 5;
  const PromptAttention& p = a.p.a;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  check_starts(p);
  const PromptTile item = prompt_tile(a.p, prompt_block());
  if (item.tile < 0) return;
  const auto budget = budget_from_now(a.timeout_ns, flags);
  const int g = blockIdx.x / a.p.groups, h0 = blockIdx.x % a.p.groups * a.p.heads, heads = min(a.p.heads, a.p.rep - h0);
  const int first = item.tile * a.p.positions, keys = min(first + a.p.positions, item.tokens);  // the first position, and behind the last
  const int blocks = (keys + kKeys - 1) / kKeys;
  const bool ragged = keys % kKeys != 0;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < kSlots; s++) {
      mbar_init(&slot_full[s], 1);
      mbar_init(&slot_empty[s], 1);
    }
    mbar_init(v_clean, 1);
    mbar_init(drained, 1);
    for (int i = 0; i < 2; i++) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);
    }
    flags[0] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  auto s_col = [&](int buffer) { return tmem_base + (uint32_t)(buffer * kKeys); };
  const uint32_t o_col = tmem_base + 2 * kKeys;

  if (warp >= 4) {
    const bool leader = elect_one();
    if (warp == kCopyWarp) {
      // In the order in which the products use them: K0 K1 V0 K2 V1 ..
      if (leader) {
        mbar_expect_tx(q_full, kHalves * (uint32_t)(a.p.heads * a.p.positions) * 128u);
        for (int c = 0; c < kHalves; c++) tma_load_4d(base + c * kQueryBlock, &qmap, c * 64, h0, g, item.start + first, q_full);
      }
      __syncwarp();
      int slot = 0;
      unsigned phase = 0;
      bool ok = true;
      int keys_of = 0, values_of = 0, issued = 0;  // the next blocks, and copies into slots
      for (; issued < 2 * blocks; issued++) {
        ok = issued < kSlots || __all_sync(0xffffffffu, mbar_wait(&slot_empty[slot], phase ^ 1, budget));
        if (!ok) break;
        const bool is_keys = keys_of < blocks && keys_of < values_of + 2;
        const int block = is_keys ? keys_of++ : values_of++;
        if (leader) {
          const CUtensorMap* map = is_keys ? &kmap : &vmap;
          const uint32_t dst = ring + (uint32_t)slot * kSlotBytes;
          mbar_expect_tx(&slot_full[slot], kSlotBytes);
          for (int c = 0; c < kHalves; c++) tma_load_3d(dst + c * kKeyBlock, map, c * 64, item.start + block * kKeys, g, &slot_full[slot]);
        }
        __syncwarp();
        if (++slot == kSlots) {
          slot = 0;
          phase ^= 1;
        }
      }
      if (ok && ragged) {
        const int last = 2 * blocks - 1;
        if (__all_sync(0xffffffffu, mbar_wait(&slot_full[last % kSlots], (unsigned)(last / kSlots) & 1u, budget))) {
          unsigned char* rows0 = base_ptr + kTileBytes + (last % kSlots) * kSlotBytes;
          const int from = keys % kKeys * 8;  // pieces of 16 bytes
          for (int c = 0; c < kHalves; c++)
            for (int i = from + lane; i < kKeys * 8; i += 32) *reinterpret_cast<uint4*>(rows0 + c * kKeyBlock + i * 16) = make_uint4(0, 0, 0, 0);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(v_clean);
        }
      }
      if (leader) {
        const unsigned long long until = global_timer_ns() + kLandNs;
        wait_landed(q_full, 0, until);
        for (int i = issued - 1; i >= 0 && i >= issued - kSlots; i--) wait_landed(&slot_full[i % kSlots], (unsigned)(i / kSlots) & 1u, until);
      }
      __syncwarp();
    } else if (warp == kMmaWarp) {
      // N = keys with K as a K-major B operand; N = HD with V as an MN-major one (bit 16).
      const uint32_t idesc_s = instr_desc(BF16, kKeys, 0);
      const uint32_t idesc_o = instr_desc(BF16, HD, 0) | 1u << 16;
      const uint64_t q_first = smem_desc(base, 16, 1024), k_first = smem_desc(ring, 16, 1024), v_first = smem_desc(ring, kKeyBlock, 1024);
      int slot = 0;
      unsigned phase = 0;
      auto next_slot = [&]() {
        const int s = slot;
        if (++slot == kSlots) {
          slot = 0;
          phase ^= 1;
        }
        return s;
      };
      auto wait = [&](uint64_t* bar, unsigned parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, budget)) != 0; };
      // Issued by the elected thread.
      auto scores = [&](int buffer, int k_slot) {
        const uint64_t k = desc_advance(k_first, (uint32_t)k_slot * kSlotBytes);
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk++)
          mma_f16(s_col(buffer), desc_advance(q_first, (uint32_t)(kk >> 2) * kQueryBlock + (uint32_t)(kk & 3) * 32u),
                  desc_advance(k, (uint32_t)(kk >> 2) * kKeyBlock + (uint32_t)(kk & 3) * 32u), idesc_s, kk ? 1u : 0u);
      };
      bool ok = wait(q_full, 0);
#pragma unroll
      for (int i = 0; i < 2; i++) {
        if (!ok || i >= blocks) continue;
        const unsigned k_phase = phase;
        const int k_slot = next_slot();
        ok = wait(&slot_full[k_slot], k_phase);
        if (!ok) continue;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (leader) {
          scores(i, k_slot);
          mma_commit(&s_full[i]);
          mma_commit(&slot_empty[k_slot]);
        }
        __syncwarp();
      }
      for (int j = 0; j < blocks && ok; j++) {
        const int buffer = j & 1;
        const unsigned v_phase = phase;
        const int v_slot = next_slot();
        const unsigned k_phase = phase;
        const bool more = j + 2 < blocks;
        const int k_slot = more ? next_slot() : 0;
        ok = wait(&slot_full[v_slot], v_phase) && (j + 1 < blocks || !ragged || wait(v_clean, 0)) && (!more || wait(&slot_full[k_slot], k_phase)) &&
             wait(&p_ready[buffer], (unsigned)(j >> 1) & 1u);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (leader) {
          const uint64_t v = desc_advance(v_first, (uint32_t)v_slot * kSlotBytes);
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; kk++)
            mma_values(o_col, s_col(buffer) + (uint32_t)kk * 16u, desc_advance(v, (uint32_t)kk * 2048u), idesc_o, (j > 0 || kk) ? 1u : 0u);
          if (more) scores(buffer, k_slot);
          mma_commit(&s_full[buffer]);
          mma_commit(&slot_empty[v_slot]);
          if (more) mma_commit(&slot_empty[k_slot]);
        }
        __syncwarp();
      }
      if (leader) {
        if (!ok) report(p.error_words, kErrorWait);
        mma_commit(drained);
        wait_landed(drained, 0, global_timer_ns() + kLandNs);
      }
      __syncwarp();
    }
  } else {
    const uint32_t lanes = (uint32_t)(warp * 32) << 16, o_addr = o_col + lanes;
    const int row = warp * 32 + lane;
    // Rows that are not there have position -1: every key is hidden and nothing is stored.
    const int head = row % a.p.heads, at = row / a.p.heads;
    const int pos = at < a.p.positions && head < heads && first + at < keys ? first + at : -1;
    const int first_pos = first + warp * 32 / a.p.heads;  // of the warp
    float m_used = -INFINITY, sum = 0.f;
    bool ok = true;
    for (int j = 0; j < blocks; j++) {
      const int buffer = j & 1;
      const uint32_t s_addr = s_col(buffer) + lanes;
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[buffer], (unsigned)(j >> 1) & 1u, budget));
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      float s[kKeys / 32][32];
#pragma unroll
      for (int c = 0; c < kKeys / 32; c++) tmem_load_32(s_addr + c * 32, s[c]);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      if (a.sign != 1.f) {
#pragma unroll
        for (int e = 0; e < kKeys; e++) s[e / 32][e % 32] *= a.sign;
      }
      const int key0 = j * kKeys;
      if (key0 + kKeys - 1 > first_pos) {
#pragma unroll
        for (int e = 0; e < kKeys; e++)
          if (key0 + e > pos) s[e / 32][e % 32] = -INFINITY;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      max_of<32>(s[0], mx);
      const float m_block = max_of<32>(s[1], mx) * a.scale_log2;
      if (__any_sync(0xffffffffu, m_block > m_used + Probability<BF16>::kGrow)) {
        const float top = fmaxf(m_used, m_block), corr = top == m_used ? 1.f : exp2_approx(m_used - top);  // 0 the first time
        m_used = top;
        sum *= corr;
        if (j > 0) {
          // The product of the block before may still be adding to the results.
          ok = __all_sync(0xffffffffu, mbar_wait(&s_full[buffer ^ 1], (unsigned)(((j - 1) >> 1) + 1) & 1u, budget));
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
#pragma unroll
      for (int c = 0; c < kKeys / 32; c++) store_probabilities<BF16>(s[c], a.scale_log2, shift, part, s_addr + c * 32);
      const float2 block = pair_split(pair_add(part[0], part[1]));
      sum += block.x + block.y;
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[buffer]);
    }
    ok = ok && __all_sync(0xffffffffu, mbar_wait(&s_full[(blocks - 1) & 1], (unsigned)(((blocks - 1) >> 1) + 1) & 1u, budget));
    if (ok) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const float inverse = rows::inverse_of(sum);
      const int h = g * a.p.rep + h0 + head;
      unsigned short* out = static_cast<unsigned short*>(p.out) + (long long)(item.start + pos) * p.out_stride + h * p.out_head_stride;
      const unsigned short* k = static_cast<const unsigned short*>(p.k) + (long long)item.start * p.k_stride + (long long)g * p.k_head_stride;
      const unsigned short* v = static_cast<const unsigned short*>(p.v) + (long long)item.start * p.v_stride + (long long)g * p.v_head_stride;
      bool spoilt = false;  // by a hidden value
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
        if (__any_sync(0xffffffffu, sums.x + sums.y != 0.f && pos >= 0 && sum == sum)) {
          OddColumns seen = prompt_odd_columns<BF16>(p, k, v, c, first_pos, __reduce_max_sync(0xffffffffu, pos), pos);
          if (sum == 0.f) seen = {seen.any(), 0, 0};
#pragma unroll
          for (int e = 0; e < 32; e++) {
            if (seen.any() >> e & 1) o[e] = seen.of(e);
            else spoilt = spoilt || rows::odd(o[e]);
          }
        }
        if (pos >= 0) {
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            if (c + e < p.head_dim)
              *reinterpret_cast<uint4*>(out + c + e) =
                  make_uint4(pack_pair<BF16>(o[e] * inverse, o[e + 1] * inverse), pack_pair<BF16>(o[e + 2] * inverse, o[e + 3] * inverse),
                             pack_pair<BF16>(o[e + 4] * inverse, o[e + 5] * inverse), pack_pair<BF16>(o[e + 6] * inverse, o[e + 7] * inverse));
        }
      }
      if (p.lse && pos >= 0)
        p.lse[(long long)(item.start + pos) * p.heads + h] =
            sum == 0.f ? -INFINITY : fmaf(m_used - Probability<BF16>::kLift, rows::kLn2, logf(sum));
      // All lanes write a row once more: behind what each has stored of its own.
      __syncwarp();
      unsigned left = __ballot_sync(0xffffffffu, spoilt && pos >= 0);
      for (; left; left &= left - 1) {
        const int r = __ffs(left) - 1, row_pos = __shfl_sync(0xffffffffu, pos, r), row_h = __shfl_sync(0xffffffffu, h, r);
        const long long token = item.start + row_pos;
        redo_row<BF16, HD>(a, static_cast<const unsigned short*>(p.q) + token * p.q_stride + row_h * p.q_head_stride, k, v,
                           static_cast<unsigned short*>(p.out) + token * p.out_stride + row_h * p.out_head_stride, row_pos,
                           __shfl_sync(0xffffffffu, m_used, r), __shfl_sync(0xffffffffu, sum, r));
      }
    } else if (lane == 0) {
      report(p.error_words, kErrorWait);
    }
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
