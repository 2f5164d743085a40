// Attention of one new token per sequence over a paged key-value cache.
//
//   s_t = scale * q . k_t (t < length),  m = max s,  l = sum e^(s_t - m),  out = sum e^(s_t - m) v_t / l,  lse = m + ln l
//
// A sequence without rows gives zeros and an lse of -inf. Rows beyond the length are not read: what a page holds there, or the
// table names for them, does not matter. With a new row in the call, row length - 1 is taken from there and stored.
//
// Bound by memory: at one query position the products take 1 FLOP a byte and query head of a KV head, where the GPU has 250 (bf16).
// So one launch reads every row once with as many bytes in flight as fit, and the softmax keeps a running maximum and sum. Measured
// (bf16, heads of 128, 32 query and 8 KV heads; one call after the other, device time):
//   32 sequences up to 2048 rows, 180 MB: 38.3 us (4.7 TB/s). Rows arrive for 23 us of it, at 7.8 TB/s; before them 4 us of launch,
//   shares and first addresses, behind them 2 to 5 us of joins; blocks take 15 to 30 us for equal shares, why is not known.
//   2 sequences up to 65 536 rows, 64 query heads, 447 MB: 85.5 us (5.2 TB/s). 1 sequence of 517 rows: 7.7 us, all of it these latencies.
//
// Tracking adds to weights[b, g, t] the weights e^(s_t - lse) of the query heads that read KV head g. They need the whole row's
// lse, so the scores (4 bytes a head and key, against 4 * head_dim of key and value) go through the workspace to a second kernel.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../common.h"
#include "arith.cuh"
#include "kernels.h"
#include "paged.cuh"

namespace pjrtx {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// ---- division of the work ------------------------------------------------------------------------------------------
// A unit is a tile of rows (six warps have 8, 16 or 32 each) of one (sequence, KV head, group of query heads), a segment what
// belongs to one of these. Segments have numbers for their tiles and, behind them, for kSegmentCost more: what joining the warps and going on with another segment
// takes. The numbers are cut into equal shares, one for each block that fits the GPU at once; lengths are device data, so each
// block adds them up itself. Where several blocks share a segment, each leaves (max, sum, values) in its slot of the workspace and
// the block that arrives last joins them in block order.
//
// Six warps, two blocks an SM: with twelve warps and one block, whose joins stop all of an SM's loads, batch 32 takes 43.5 us, not
// 38.7 (65 536 rows 82.6, not 87); with four warps and three blocks 65 536 rows take 88.8. kSegmentCost 2 was taken for heads of 128 in
// 16 bits, where a tile is 96 rows (192 for heads of 64, 48 and more for f32): a join and the next start take 3 to 5 us, a tile 1.9; with 0, batch 32 takes 39.2 us and 30 000 rows of one sequence 33.9 (31.6). It costs the shortest
// rows, where a block could have had more segments: 64 sequences of 100 rows 12.2 us, 10.3 with 0.

constexpr int kWarps = 6, kThreads = kWarps * 32;
constexpr int kSegmentCost = 2;

struct AttendSpace {
  float* lse2;         // [batch, heads]: lse / ln 2
  unsigned* counters;  // [batch * kv_heads * head groups]: blocks that have arrived, zero between calls
  float* partials;     // [blocks][2][heads of a group][dims + 2]
  float* scores;       // [batch, kv_heads, capacity, rep] in units of ln 2 (tracking only)
};

struct AttendArgs {
  PagedView c;
  PagedAttend a;
  AttendSpace space;
  int rep, groups;  // query heads of a KV head, groups of them
  int pieces;       // 16-byte pieces of a row
  int tile_rows;    // of a tile: those of a warp times the warps
  unsigned reciprocal;  // floor(2^32 / page_size), at most 2^32 - 1
};

struct Cursor {
  int b, group, tile, tiles, length;  // group = KV head * groups + head group
};

__device__ __forceinline__ int tiles_of(const AttendArgs& p, int length) { return (length + p.tile_rows - 1) / p.tile_rows; }

__device__ __forceinline__ void advance(const AttendArgs& p, Cursor& u) {
  if (++u.tile < u.tiles) return;
  u.tile = 0;
  if (++u.group < p.c.kv_heads * p.groups) return;
  u.group = 0;
  do {
    u.b++;
    u.length = paged_length(p.c, u.b);
    u.tiles = tiles_of(p, u.length);
  } while (u.tiles == 0);
}

// What this block works on: the tiles among numbers [begin, begin + size), the first of them at `first` of these.
struct Share {
  long long begin, quota;
  int size, first;  // first >= size: none
  Cursor at;
};

// The next tile of a share; false at its end.
__device__ __forceinline__ bool next_unit(const AttendArgs& p, Cursor& u, int& at, int size) {
  const int to = at + (u.tile + 1 < u.tiles ? 1 : 1 + kSegmentCost);
  if (to >= size) return false;
  at = to;
  advance(p, u);
  return true;
}

// Called by all threads. `scratch`: shared memory of kWarps long longs and 8 ints.
__device__ __forceinline__ Share share_of_block(const AttendArgs& p, long long* scratch) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int per_thread = (p.c.batch + kThreads - 1) / kThreads;
  const int first = min(p.c.batch, (int)threadIdx.x * per_thread), last = min(p.c.batch, first + per_thread);
  const long long width = (long long)p.c.kv_heads * p.groups;
  auto numbers_of = [&](int tiles) { return tiles ? tiles + kSegmentCost : 0; };
  long long mine = 0;
  for (int b = first; b < last; b++) mine += numbers_of(tiles_of(p, paged_length(p.c, b))) * width;
  long long sum = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long o = __shfl_up_sync(~0u, sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 31) scratch[warp] = sum;
  __syncthreads();
  long long before = sum - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; w++) {
    if (w < warp) before += scratch[w];
    total += scratch[w];
  }
  Share s;
  s.quota = max(1ll, (total + gridDim.x - 1) / gridDim.x);
  s.begin = min(total, blockIdx.x * s.quota);
  s.size = (int)min(total - s.begin, s.quota);
  int* found = reinterpret_cast<int*>(scratch + kWarps);
  if (s.size > 0 && before <= s.begin && s.begin < before + mine) {
    long long rest = s.begin - before;
    Cursor u;
    u.b = first;
    for (;; u.b++) {
      u.length = paged_length(p.c, u.b);
      u.tiles = tiles_of(p, u.length);
      if (rest < numbers_of(u.tiles) * width) break;
      rest -= numbers_of(u.tiles) * width;
    }
    u.group = (int)(rest / (u.tiles + kSegmentCost));
    u.tile = (int)(rest % (u.tiles + kSegmentCost));
    int at = 0;
    if (u.tile >= u.tiles) {  // behind a segment's tiles: the share begins with the next one
      at = u.tiles + kSegmentCost - u.tile;
      if (at < s.size) advance(p, u);
    }
    found[0] = u.b;
    found[1] = u.group;
    found[2] = u.tile;
    found[3] = u.length;
    found[4] = at;
  }
  __syncthreads();
  s.at.b = found[0];
  s.at.group = found[1];
  s.at.tile = found[2];
  s.at.length = found[3];
  s.at.tiles = tiles_of(p, s.at.length);
  s.first = s.size > 0 ? found[4] : 0;
  return s;
}

// ---- rows into shared memory ---------------------------------------------------------------------------------------
// A warp works by itself: it fetches its 8, 16 or 32 rows of each tile with cp.async into stages of its own, so the warps of a block
// meet only at the end of a segment. Row by row, since a row of a page is the longest run that is contiguous in every layout. Rows
// outside the sequence (or without a page) are filled with zeros and masked.

template <typename T, int D, int ROWS>
struct RowStage {
  static constexpr int kPitch = D * (int)sizeof(T) + 16;  // bytes; rows of eight keys fall on different banks
  static constexpr int kBytes = 2 * ROWS * kPitch;
};

__device__ __forceinline__ void copy16(unsigned to, unsigned long long from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy16_or_zero(unsigned to, unsigned long long from, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Where row `lane % ROWS` of this warp's part of a tile lies.
struct RowPlace {
  int page, row;  // page -1: no such row
};

template <int ROWS>
__device__ __forceinline__ RowPlace locate(const AttendArgs& p, const Cursor& u) {
  const int t = u.tile * p.tile_rows + (threadIdx.x / 32) * ROWS + (threadIdx.x & (ROWS - 1));
  RowPlace r = {-1, 0};
  if (t < u.length) {
    int column = (int)__umulhi((unsigned)t, p.reciprocal);  // the quotient or one less
    r.row = t - column * p.c.page_size;
    if (r.row >= p.c.page_size) {
      column++;
      r.row -= p.c.page_size;
    }
    r.page = p.c.table[u.b * p.c.table_stride + column];
    if (r.page < 0 || r.page >= p.c.num_pages) {
      report(p.c.error_words, kErrorPageId);
      r.page = -1;
    }
  }
  return r;
}

__device__ __forceinline__ unsigned long long address_of(const void* p) { return reinterpret_cast<unsigned long long>(p); }

// What a warp knows of a stage besides the rows.
struct StageNote {
  unsigned mask;             // rows that count
  int fresh;                 // the row that came with the call and goes to the pool, -1: none
  unsigned long long store;  // where its key goes
};

// Requests the rows of `u`.
template <typename T, int D, int ROWS>
__device__ __forceinline__ void request(const AttendArgs& p, const Cursor& u, const RowPlace& r, char* stage, StageNote* note) {
  using S = RowStage<T, D, ROWS>;
  constexpr int kPieces = D * (int)sizeof(T) / 16, kAcross = 8;  // eight lanes beside each other on one row
  const int lane = threadIdx.x % 32, g = u.group / p.groups;
  const int t0 = u.tile * p.tile_rows + (threadIdx.x / 32) * ROWS;
  unsigned long long k = 0;  // address of the key; the value's is `apart` further
  const unsigned long long apart_pools = address_of(p.c.v) - address_of(p.c.k);
  unsigned long long apart = apart_pools;
  if (r.page >= 0)
    k = address_of(p.c.k) + (r.page * p.c.page_stride + r.row * p.c.row_stride + g * p.c.head_stride) * (long long)sizeof(T);
  const int fresh = u.length - 1 - t0;  // which of the warp's rows comes with the call
  const bool has_fresh = p.a.k_new && fresh >= 0 && fresh < ROWS;
  if (has_fresh) {
    const long long at = (u.b * p.a.new_batch_stride + g * p.a.new_head_stride) * (long long)sizeof(T);
    const char* k_new = static_cast<const char*>(p.a.k_new) + at;
    const char* v_new = static_cast<const char*>(p.a.v_new) + at;
    if ((lane & (ROWS - 1)) == fresh && k) {
      if (lane < ROWS) note->store = k;
      k = address_of(k_new);
      apart = address_of(v_new) - k;
    }
  }
  constexpr unsigned kAll = ROWS == 32 ? ~0u : (1u << ROWS) - 1;
  const unsigned there = __ballot_sync(~0u, k != 0) & kAll;
  if (lane == 0) {
    note->mask = there;
    note->fresh = has_fresh && (there >> fresh & 1) && u.group % p.groups == 0 ? fresh : -1;
  }
  const unsigned to = (unsigned)__cvta_generic_to_shared(stage) + lane / kAcross * S::kPitch + lane % kAcross * 16;
  const bool whole = there == kAll && p.pieces == kPieces;
#pragma unroll
  for (int j = 0; j < ROWS * kAcross / 32; j++) {
    const int row = lane / kAcross + j * (32 / kAcross);
    unsigned long long kr = __shfl_sync(~0u, k, row), vr = apart;
    if (has_fresh) vr = __shfl_sync(~0u, apart, row);
    const bool valid = kr != 0;
    kr += lane % kAcross * 16;
    vr += kr;
    if (whole) {
#pragma unroll
      for (int i = 0; i < kPieces / kAcross; i++) {
        copy16(to + j * (32 / kAcross) * S::kPitch + i * kAcross * 16, kr + i * kAcross * 16);
        copy16(to + (ROWS + j * (32 / kAcross)) * S::kPitch + i * kAcross * 16, vr + i * kAcross * 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPieces / kAcross; i++) {
        const bool in = valid && lane % kAcross + i * kAcross < p.pieces;
        copy16_or_zero(to + j * (32 / kAcross) * S::kPitch + i * kAcross * 16, in ? kr + i * kAcross * 16 : address_of(p.c.k), in);
        copy16_or_zero(to + (ROWS + j * (32 / kAcross)) * S::kPitch + i * kAcross * 16, in ? vr + i * kAcross * 16 : address_of(p.c.v), in);
      }
    }
  }
}

// Stores the row that came with the call from its stage into the pool.
template <typename T, int D, int ROWS>
__device__ __forceinline__ void store_fresh(const AttendArgs& p, const StageNote& note, const char* stage) {
  if (note.fresh < 0) return;
  const char* from = stage + note.fresh * RowStage<T, D, ROWS>::kPitch;
  char* to = reinterpret_cast<char*>(note.store);
  for (int i = threadIdx.x % 32; i < p.pieces; i += 32) {
    reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(from)[i];
    reinterpret_cast<uint4*>(to + (address_of(p.c.v) - address_of(p.c.k)))[i] = reinterpret_cast<const uint4*>(from + ROWS * RowStage<T, D, ROWS>::kPitch)[i];
  }
}

// ---- the arithmetic of one warp ------------------------------------------------------------------------------------

template <typename T> struct Mma16;
template <> struct Mma16<__nv_bfloat16> {
  static __device__ __forceinline__ unsigned pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
  }
  static constexpr float kLift = 0.f, kWhole = -INFINITY;  // kWhole: exponent of the least positive probability that `split` takes
  // (a, b) >= 0 as the sum of two pairs, the first rounded towards zero; the second is 0 only where a or b is.
  static __device__ __forceinline__ uint2 split(float a, float b) {
    const float ra = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u), rb = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
    constexpr float kLeast = 1.1754944e-38f;  // 2^-126
    return make_uint2(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632),
                      pack(fmaxf(ra, fminf(a, kLeast)), fmaxf(rb, fminf(b, kLeast))));
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Mma16<__half> {
  static __device__ __forceinline__ unsigned pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
  }
  static constexpr float kLift = 15.f;
  static constexpr float kWhole = -8.f;  // 2^-23 of the largest
  // For 0 and from 2^kWhole on: the first number leaves at least 2^-11 of the probability to the second, which is then off by 2^-25.
  static __device__ __forceinline__ uint2 split(float a, float b) {
    constexpr float kPart = 0.99951171875f;  // 1 - 2^-11
    unsigned w;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b * kPart), "f"(a * kPart));
    const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return make_uint2(w, pack(a - back.x, b - back.y));
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ void mma_tf32(float (&d)[4], const float (&a)[4], float b0, float b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])), "r"(__float_as_uint(a[3])),
                 "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}

__device__ __forceinline__ void load_matrices(unsigned (&r)[4], unsigned at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(unsigned (&r)[4], unsigned at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ unsigned transpose(unsigned a) {
  unsigned d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// 16-bit types: rows and dimensions are the long sides of the products, heads the eight columns of m16n8k16, so that up to eight
// query heads cost no more than one: scores^T [16 rows x heads] = K q^T, values^T [dims x heads] += V^T p^T. A probability goes in
// as two 16-bit numbers, itself cut off and the rest: as one, it would be as far off as the result's own rounding. Neither is zero or
// negative where the probability is above zero, so that an infinite value stays infinite; both are zero where it is zero. f16 takes
// 2^15 times the probabilities, and tiles with one below 2^-23 of the largest go in as tf32: f16 ends at 2^-39, and to lose what is
// below, or to raise it to that, changes a result whose likelier rows have small values. Tiles without one cost 1 % at most for the
// question; with one in nearly every tile 32 sequences up to 2048 rows take 40.5 us, not 38.4, two up to 65 536 87.2, not 85.1.
// Tensor memory wants 64 rows at least on its M side and the scores through it to the softmax and back; with 1/60 of
// its rate used (four heads) there is nothing to win by that. Lane i holds heads (i % 4) * 2 and + 1 of every eight.
template <typename T, int D, int NB, int ROWS>
struct MmaWarp {
  static constexpr int kHeads = 8 * NB, kRows = ROWS, R = ROWS / 16;
  static constexpr int kSharedBytes = 0;
  unsigned q[D / 16][NB][2];
  float o[D / 16][NB][4];
  float m[NB][2], l[NB][2];

  // Requests the queries of a segment; nothing else of the one before is touched.
  __device__ __forceinline__ void load(const AttendArgs& p, const Cursor& u) {
    const int lane = threadIdx.x % 32, g = u.group / p.groups, h0 = (u.group % p.groups) * kHeads;
#pragma unroll
    for (int n = 0; n < NB; n++) {
      const int h = h0 + n * 8 + lane / 4;
      const T* from = static_cast<const T*>(p.a.q) + u.b * p.a.q_batch_stride + (long long)(g * p.rep + h) * p.a.q_head_stride;
#pragma unroll
      for (int i = 0; i < D / 16; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const int d = i * 16 + j * 8 + (lane % 4) * 2;
          q[i][n][j] = h < p.rep && d < p.c.head_dim ? *reinterpret_cast<const unsigned*>(from + d) : 0u;
        }
    }
  }
  __device__ __forceinline__ void start(const AttendArgs&, const Cursor&, char*) {
#pragma unroll
    for (int n = 0; n < NB; n++) {
#pragma unroll
      for (int i = 0; i < D / 16; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) o[i][n][j] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }
  }

  __device__ __forceinline__ void step(const AttendArgs& p, const Cursor& u, const char* stage, unsigned mask, float scale2) {
    constexpr int kPitch = RowStage<T, D, ROWS>::kPitch;
    const int lane = threadIdx.x % 32;
    const unsigned k_at = (unsigned)__cvta_generic_to_shared(stage), v_at = k_at + ROWS * kPitch;
    float s[R][NB][4];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[r][n][j] = 0.f;
    const unsigned k_lane = k_at + ((lane / 8 % 2) * 8 + lane % 8) * kPitch + (lane / 16) * 16;
#pragma unroll
    for (int i = 0; i < D / 16; i++)
#pragma unroll
      for (int r = 0; r < R; r++) {
        unsigned a[4];
        load_matrices(a, k_lane + r * 16 * kPitch + i * 32);
#pragma unroll
        for (int n = 0; n < NB; n++) Mma16<T>::mma(s[r][n], a, q[i][n][0], q[i][n][1]);
      }
    bool grows = false;
    float top[NB][2];
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        top[n][j] = -INFINITY;
#pragma unroll
        for (int r = 0; r < R; r++) {
          s[r][n][j] = mask >> (r * 16 + lane / 4) & 1 ? s[r][n][j] * scale2 : -INFINITY;
          s[r][n][2 + j] = mask >> (r * 16 + lane / 4 + 8) & 1 ? s[r][n][2 + j] * scale2 : -INFINITY;
          top[n][j] = max_nan(top[n][j], max_nan(s[r][n][j], s[r][n][2 + j]));
        }
        grows |= !(top[n][j] <= m[n][j]);
      }
    if (p.c.weights) {
#pragma unroll
      for (int r = 0; r < R; r++) store_scores(p, u, s[r], r);
    }
    if (__any_sync(~0u, grows)) {
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          float t = top[n][j];
#pragma unroll
          for (int d = 4; d < 32; d *= 2) t = max_nan(t, __shfl_xor_sync(~0u, t, d));
          t = max_nan(m[n][j], t);
          const float f = m[n][j] == -INFINITY ? 0.f : exp2_fast(m[n][j] - t);
          m[n][j] = t;
          l[n][j] *= f;
#pragma unroll
          for (int i = 0; i < D / 16; i++) {
            o[i][n][j] *= f;
            o[i][n][2 + j] *= f;
          }
        }
    }
    bool wide = false;  // asked of the exponents, so that the answer is there when the exponentials are
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          s[r][n][j] -= m[n][j % 2] == -INFINITY ? 0.f : m[n][j % 2] - Mma16<T>::kLift;
          wide |= s[r][n][j] < Mma16<T>::kWhole && s[r][n][j] > -INFINITY;
        }
    if constexpr (Mma16<T>::kLift > 0.f) wide = __any_sync(~0u, wide);
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          s[r][n][j] = exp2_fast(s[r][n][j]);
          s[r][n][2 + j] = exp2_fast(s[r][n][2 + j]);
          l[n][j] += s[r][n][j] + s[r][n][2 + j];
        }
    const unsigned v_lane = v_at + ((lane / 16) * 8 + lane % 8) * kPitch + (lane / 8 % 2) * 16;
    if constexpr (Mma16<T>::kLift > 0.f) {
      if (wide) return add_wide(s, v_lane);
    }
    unsigned big[R][NB][2], small[R][NB][2];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const uint2 parts = Mma16<T>::split(s[r][n][2 * k], s[r][n][2 * k + 1]);
          big[r][n][k] = transpose(parts.x);
          small[r][n][k] = transpose(parts.y);
        }
#pragma unroll
    for (int i = 0; i < D / 16; i++)
#pragma unroll
      for (int r = 0; r < R; r++) {
        unsigned a[4];
        load_matrices_transposed(a, v_lane + r * 16 * kPitch + i * 32);
#pragma unroll
        for (int n = 0; n < NB; n++) {
          Mma16<T>::mma(o[i][n], a, big[r][n][0], big[r][n][1]);
          Mma16<T>::mma(o[i][n], a, small[r][n][0], small[r][n][1]);
        }
      }
  }

  // The values of a tile under probabilities that f16 does not hold: as tf32, which has the range of f32 and in which f16 values are
  // exact, a probability as two numbers of 11 bits. Eight rows a product: even ones in slots 0 to 3, odd ones in 4 to 7, as they lie
  // in the halves of the registers that the transposed load fills.
  __device__ __forceinline__ void add_wide(const float (&s)[R][NB][4], unsigned v_lane) {
    constexpr int kPitch = RowStage<T, D, ROWS>::kPitch;
    const int lane = threadIdx.x % 32, from = lane % 4 * 8 + lane / 8;  // the lane that has this head's row 2 (lane % 4); row + 1: 4 further
    const bool odd = lane / 4 & 1;                                      // head
#pragma unroll
    for (int r = 0; r < R; r++) {
      float big[NB][4], small[NB][4];  // rows 2 (lane % 4) and + 1, then the same of the upper eight
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float x = __shfl_sync(~0u, s[r][n][k / 2 * 2], from + k % 2 * 4), y = __shfl_sync(~0u, s[r][n][k / 2 * 2 + 1], from + k % 2 * 4);
          const float w = odd ? y : x;
          big[n][k] = __uint_as_float(__float_as_uint(w) & 0xffffe000u);
          small[n][k] = fmaxf(w - big[n][k], fminf(w, 1.1754944e-38f));  // as in Mma16<__nv_bfloat16>::split
        }
#pragma unroll
      for (int i = 0; i < D / 16; i++) {
        unsigned a[4];
        load_matrices_transposed(a, v_lane + r * 16 * kPitch + i * 32);
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&a[k])), hi = __half22float2(*reinterpret_cast<const __half2*>(&a[k + 1]));
          const float v[4] = {lo.x, hi.x, lo.y, hi.y};
#pragma unroll
          for (int n = 0; n < NB; n++) {
            mma_tf32(o[i][n], v, big[n][k], big[n][k + 1]);
            mma_tf32(o[i][n], v, small[n][k], small[n][k + 1]);
          }
        }
      }
    }
  }

  // Of 16 rows, the r-th of the warp's.
  __device__ __forceinline__ void store_scores(const AttendArgs& p, const Cursor& u, const float (&s)[NB][4], int r) const {
    const int lane = threadIdx.x % 32, g = u.group / p.groups, h0 = (u.group % p.groups) * kHeads;
    const int t = u.tile * p.tile_rows + (threadIdx.x / 32) * ROWS + r * 16 + lane / 4;
    const bool lo = t < u.length, hi = t + 8 < u.length;  // a row without a page has -inf
    float* to = p.space.scores + (((long long)u.b * p.c.kv_heads + g) * p.c.page_size * p.c.max_pages + t) * p.rep + h0;
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int h = n * 8 + (lane % 4) * 2 + j;
        if (h0 + h >= p.rep) continue;
        if (lo) to[h] = s[n][j];
        if (hi) to[8 * p.rep + h] = s[n][2 + j];
      }
  }

  // Leaves this warp's references (the maxima, but for the lift) and sums in stat[head][2].
  __device__ __forceinline__ void statistics(float* stat) {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
#pragma unroll
        for (int d = 4; d < 32; d *= 2) l[n][j] += __shfl_xor_sync(~0u, l[n][j], d);
        if (lane < 4) {
          stat[2 * (n * 8 + lane * 2 + j)] = m[n][j] - Mma16<T>::kLift;
          stat[2 * (n * 8 + lane * 2 + j) + 1] = l[n][j];
        }
      }
  }
  // This warp's sums to values[head * pitch + dim].
  __device__ __forceinline__ void values(float* to, int pitch) const {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
          for (int r = 0; r < 2; r++) to[(n * 8 + (lane % 4) * 2 + j) * pitch + i * 16 + r * 8 + lane / 4] = o[i][n][2 * r + j];
  }
};

// f32: CUDA cores, two products an instruction. Scores: eight lanes beside each other have a row, pieces of 16 bytes in turn, so that
// a piece of a query serves four rows; the sums are exchanged so that a lane ends with the scores of one head. Values: lane i has
// D / 32 neighbouring dimensions of all heads. With eight heads a KV head this is bound by what a warp waits for between its own
// instructions (17 sequences up to 3877 rows of 8 KV heads of 128, 360 MB: 89 us, issue slots 39 % used), with fewer by memory.
template <int D, int H, int ROWS>
struct FmaWarp {
  static constexpr int kHeads = H, kRows = ROWS, V = D / 32;
  static constexpr int R = ROWS / 4, kOwn = R * H / 8;  // rows of eight lanes; scores a lane ends with
  static_assert(kOwn > 0);
  static constexpr int kSharedBytes = H * D * 4 + kWarps * kRows * H * 4;  // queries; probabilities of every warp
  Pair o[H][V / 2];
  float m, l;  // of this lane's head
  const float* queries;
  float* probabilities;

  static __device__ __forceinline__ int head_of(int lane) { return lane % 8 * H / 8; }
  static __device__ __forceinline__ int row_of(int lane, int i) { return lane / 8 + 4 * (lane % 8 * kOwn % R + i); }
  // Of 2 N sums of the lane and as many of the one `D2` further, each keeps one half and gets the other's share of it.
  template <int N, int D2>
  static __device__ __forceinline__ void exchange(float (&s)[R * H]) {
    const bool upper = threadIdx.x & D2;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float keep = upper ? s[N + i] : s[i], give = upper ? s[i] : s[N + i];
      s[i] = keep + __shfl_xor_sync(~0u, give, D2);
    }
  }
  // Over the lanes that have the same head.
  template <typename F>
  static __device__ __forceinline__ float over_head(float x, F&& join) {
    if (H <= 4) x = join(x, __shfl_xor_sync(~0u, x, 1));
    if (H <= 2) x = join(x, __shfl_xor_sync(~0u, x, 2));
    x = join(x, __shfl_xor_sync(~0u, x, 8));
    return join(x, __shfl_xor_sync(~0u, x, 16));
  }

  __device__ __forceinline__ void load(const AttendArgs&, const Cursor&) {}
  __device__ __forceinline__ void start(const AttendArgs& p, const Cursor& u, char* shared) {
    const int g = u.group / p.groups, h0 = (u.group % p.groups) * H;
    float* to = reinterpret_cast<float*>(shared);
    queries = to;
    probabilities = to + H * D + (threadIdx.x / 32) * kRows * H;
    __syncthreads();
    for (int i = threadIdx.x; i < H * D; i += kThreads) {
      const int h = h0 + i / D, d = i % D;
      to[i] = h < p.rep && d < p.c.head_dim
                  ? static_cast<const float*>(p.a.q)[u.b * p.a.q_batch_stride + (long long)(g * p.rep + h) * p.a.q_head_stride + d] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < H; h++)
#pragma unroll
      for (int i = 0; i < V / 2; i++) o[h][i] = pair_of(0.f, 0.f);
    m = -INFINITY;
    l = 0.f;
  }

  __device__ __forceinline__ void step(const AttendArgs& p, const Cursor& u, const char* stage, unsigned mask, float scale2) {
    constexpr int kPitch = RowStage<float, D, kRows>::kPitch;
    const int lane = threadIdx.x % 32;
    float s[R * H];  // [head][row]
    constexpr int kAtOnce = H == 8 ? 2 : R;  // rows, as registers go
#pragma unroll
    for (int j0 = 0; j0 < R; j0 += kAtOnce) {
      Pair sums[kAtOnce * H];
#pragma unroll
      for (int i = 0; i < kAtOnce * H; i++) sums[i] = pair_of(0.f, 0.f);
      const char* k = stage + (lane / 8 + 4 * j0) * kPitch + lane % 8 * 16;
      const float* q = queries + lane % 8 * 4;
#pragma unroll 2
      for (int i = 0; i < D / 32; i++) {
        ulonglong2 x[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; j++) x[j] = *reinterpret_cast<const ulonglong2*>(k + 4 * j * kPitch + i * 128);
#pragma unroll
        for (int h = 0; h < H; h++) {
          const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(q + h * D + i * 32);
#pragma unroll
          for (int j = 0; j < kAtOnce; j++) sums[h * kAtOnce + j] = pair_fma(x[j].x, y.x, pair_fma(x[j].y, y.y, sums[h * kAtOnce + j]));
        }
      }
#pragma unroll
      for (int h = 0; h < H; h++)
#pragma unroll
        for (int j = 0; j < kAtOnce; j++) {
          const float2 two = pair_split(sums[h * kAtOnce + j]);
          s[h * R + j0 + j] = two.x + two.y;
        }
    }
    exchange<R * H / 2, 4>(s);
    exchange<R * H / 4, 2>(s);
    exchange<R * H / 8, 1>(s);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kOwn; i++) {
      s[i] = mask >> row_of(lane, i) & 1 ? s[i] * scale2 : -INFINITY;
      top = max_nan(top, s[i]);
    }
    if (p.c.weights) {
      const int g = u.group / p.groups, h = (u.group % p.groups) * H + head_of(lane);
      const int t0 = u.tile * p.tile_rows + (threadIdx.x / 32) * kRows;
      float* to = p.space.scores + (((long long)u.b * p.c.kv_heads + g) * p.c.page_size * p.c.max_pages + t0) * p.rep + h;
#pragma unroll
      for (int i = 0; i < kOwn; i++)
        if (h < p.rep && t0 + row_of(lane, i) < u.length) to[row_of(lane, i) * p.rep] = s[i];
    }
    if (__any_sync(~0u, !(top <= m))) {
      top = max_nan(m, over_head(top, [](float a, float b) { return max_nan(a, b); }));
      const float f = m == -INFINITY ? 0.f : exp2_fast(m - top);
      m = top;
      l *= f;
#pragma unroll
      for (int h = 0; h < H; h++) {
        const float of_head = __shfl_sync(~0u, f, h * 8 / H);
#pragma unroll
        for (int i = 0; i < V / 2; i++) o[h][i] = pair_mul(o[h][i], pair_of(of_head, of_head));
      }
    }
#pragma unroll
    for (int i = 0; i < kOwn; i++) {
      const float w = exp2_fast(s[i] - (m == -INFINITY ? 0.f : m));
      probabilities[row_of(lane, i) * H + head_of(lane)] = w;
      l += w;
    }
    __syncwarp();
    const char* v = stage + kRows * kPitch + lane * V * 4;
#pragma unroll 4
    for (int t = 0; t < kRows; t++) {
      Pair x[V / 2];
      if constexpr (V == 2) {
        x[0] = *reinterpret_cast<const Pair*>(v + t * kPitch);
      } else {
#pragma unroll
        for (int i = 0; i < V / 2; i += 2) {
          const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(v + t * kPitch + i * 8);
          x[i] = two.x;
          x[i + 1] = two.y;
        }
      }
      float w[H];
      if constexpr (H == 2) *reinterpret_cast<float2*>(w) = *reinterpret_cast<const float2*>(probabilities + t * H);
#pragma unroll
      for (int h = 0; h + 4 <= H; h += 4) *reinterpret_cast<float4*>(w + h) = *reinterpret_cast<const float4*>(probabilities + t * H + h);
#pragma unroll
      for (int h = 0; h < H; h++)
#pragma unroll
        for (int i = 0; i < V / 2; i++) o[h][i] = pair_fma(pair_of(w[h], w[h]), x[i], o[h][i]);
    }
    __syncwarp();
  }

  __device__ __forceinline__ void statistics(float* stat) {
    const int lane = threadIdx.x % 32;
    l = over_head(l, [](float a, float b) { return a + b; });
    if (lane < 8 && lane * H % 8 == 0) {
      stat[2 * head_of(lane)] = m;
      stat[2 * head_of(lane) + 1] = l;
    }
  }
  __device__ __forceinline__ void values(float* to, int pitch) const {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int h = 0; h < H; h++)
#pragma unroll
      for (int i = 0; i < V / 2; i++) *reinterpret_cast<float2*>(to + h * pitch + lane * V + 2 * i) = pair_split(o[h][i]);
  }
};

// ---- the kernel ----------------------------------------------------------------------------------------------------

template <typename W>
struct JoinSpace {  // at the end of a segment
  static constexpr int H = W::kHeads;
  float2 stat[kWarps][H];  // (max, sum)
  long long scratch[kWarps + 4];
  StageNote note[kWarps][8];
  int last;
};

template <typename T> __device__ __forceinline__ void store4(T* to, float4 x);
template <> __device__ __forceinline__ void store4(float* to, float4 x) { *reinterpret_cast<float4*>(to) = x; }
template <> __device__ __forceinline__ void store4(__half* to, float4 x) {
  *reinterpret_cast<uint2*>(to) = make_uint2(Mma16<__half>::pack(x.x, x.y), Mma16<__half>::pack(x.z, x.w));
}
template <> __device__ __forceinline__ void store4(__nv_bfloat16* to, float4 x) {
  *reinterpret_cast<uint2*>(to) = make_uint2(Mma16<__nv_bfloat16>::pack(x.x, x.y), Mma16<__nv_bfloat16>::pack(x.z, x.w));
}

__device__ __forceinline__ void store_lse(const AttendArgs& p, int b, int h, float top, float total) {
  const long long at = (long long)b * p.a.heads + h;
  const float lse2 = total == 0.f ? -INFINITY : top + log2f(total);
  p.space.lse2[at] = lse2;
  if (p.a.lse) p.a.lse[at] = lse2 * kLn2;
}

// Four dimensions of the result from sums under the maximum `top`.
template <typename T>
__device__ __forceinline__ void finish(const AttendArgs& p, int b, int h, int d, T* out, float4 x, float top, float total) {
  if (d == 0) store_lse(p, b, h, top, total);
  if (d >= p.c.head_dim) return;
  const float inverse = total == 0.f ? 0.f : 1.f / total;
  x.x *= inverse; x.y *= inverse; x.z *= inverse; x.w *= inverse;
  store4(out + d, x);
}

// Joins the `count` parts of a segment. One block's parts are kSlot * 2 floats apart, but for the first, which is a slot later.
// The block reads them all (4 KB a part with eight heads of 128) from L2, so every thread has as many loads in flight as it has
// registers for; where there are fewer results than threads, several threads share one and take every so many-th part.
template <typename T, typename W, int D>
__device__ __forceinline__ void merge(const AttendArgs& p, int b, int h0, int heads, const float* parts, int count, T* out, char* space) {
  constexpr int H = W::kHeads, kSlot = H * (D + 2), kAtOnce = 10;
  auto part = [&](int i) { return parts + (i == 0 ? kSlot : (long long)i * 2 * kSlot); };
  const int items = heads * (D / 4);
  int sharers = 1;
  while (sharers * 2 * items <= kThreads) sharers *= 2;
  for (int j0 = 0; j0 < items; j0 += kThreads) {
    const int j = sharers > 1 ? (int)threadIdx.x % items : j0 + (int)threadIdx.x, first = sharers > 1 ? (int)threadIdx.x / items : 0;
    const bool works = j < items && first < sharers;
    const int h = works ? j / (D / 4) : 0, d = j % (D / 4) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, total = 0.f;
    if (works)
      for (int i0 = first; i0 < count; i0 += sharers * kAtOnce) {
        float4 y[kAtOnce];
        float2 stat[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; k++) {
          const int i = i0 + k * sharers;
          stat[k] = make_float2(-INFINITY, 0.f);
          if (i < count) {
            stat[k] = __ldcg(reinterpret_cast<const float2*>(part(i) + H * D + 2 * h));
            y[k] = __ldcg(reinterpret_cast<const float4*>(part(i) + j * 4));
          }
        }
        float to = top;
#pragma unroll
        for (int k = 0; k < kAtOnce; k++) to = max_nan(to, stat[k].x);
        const float keep = top == -INFINITY ? 0.f : exp2_fast(top - to);
        x.x *= keep; x.y *= keep; x.z *= keep; x.w *= keep;
        total *= keep;
        top = to;
#pragma unroll
        for (int k = 0; k < kAtOnce; k++)
          if (stat[k].x != -INFINITY) {
            const float f = exp2_fast(stat[k].x - top);
            total = fmaf(f, stat[k].y, total);
            x.x = fmaf(f, y[k].x, x.x);
            x.y = fmaf(f, y[k].y, x.y);
            x.z = fmaf(f, y[k].z, x.z);
            x.w = fmaf(f, y[k].w, x.w);
          }
      }
    if (sharers > 1) {
      float4* sums = reinterpret_cast<float4*>(space);
      float2* stats = reinterpret_cast<float2*>(sums + kThreads);
      sums[threadIdx.x] = x;
      stats[threadIdx.x] = make_float2(top, total);
      __syncthreads();
      if (first > 0 || !works) continue;
      for (int k = 1; k < sharers; k++) {
        const float4 y = sums[k * items + j];
        const float2 o = stats[k * items + j];
        const float to = max_nan(top, o.x), f = top == -INFINITY ? 0.f : exp2_fast(top - to), e = o.x == -INFINITY ? 0.f : exp2_fast(o.x - to);
        total = total * f + o.y * e;
        x.x = x.x * f + y.x * e; x.y = x.y * f + y.y * e; x.z = x.z * f + y.z * e; x.w = x.w * f + y.w * e;
        top = to;
      }
    }
    if (works) finish(p, b, h0 + h, d, out + h * p.a.out_head_stride, x, top, total);
  }
}

template <typename T, typename W, int D, int STAGES, int PER_SM>
__global__ void __launch_bounds__(kThreads, PER_SM) paged_attend_kernel(const __grid_constant__ AttendArgs p) {
  using Stage = RowStage<T, D, W::kRows>;
  using Join = JoinSpace<W>;
  constexpr int H = W::kHeads, kPitch = D + 4;
  static_assert(H * kPitch * 4 <= Stage::kBytes, "a warp's sums take the place of a stage");
  extern __shared__ __align__(16) char smem[];
  char* shared = smem + kWarps * STAGES * Stage::kBytes;
  Join& join = *reinterpret_cast<Join*>(shared + W::kSharedBytes);
  PJRTX_PDL_PROLOGUE();
  const int warp = threadIdx.x / 32;
  char* stages = smem + warp * STAGES * Stage::kBytes;
  for (int b = blockIdx.x; b < p.c.batch; b += gridDim.x) {  // idle sequences
    if (threadIdx.x == 0) paged_check_length(p.c, b);
    if (paged_length(p.c, b) > 0) continue;
    T* out = static_cast<T*>(p.a.out) + b * p.a.out_batch_stride;
    for (int i = threadIdx.x; i < p.a.heads * p.c.head_dim; i += kThreads)
      out[i / p.c.head_dim * p.a.out_head_stride + i % p.c.head_dim] = from_float<T>(0.f);
    for (int h = threadIdx.x; h < p.a.heads; h += kThreads) store_lse(p, b, h, 0.f, 0.f);
  }
  const Share share = share_of_block(p, join.scratch);
  if (share.first >= share.size) return;
  const float scale2 = p.a.scale * kLog2e;

  Cursor ahead = share.at, now = share.at;  // the next tile to request, the one at work
  int ahead_at = share.first, at = share.first;
  bool more_ahead = true;
  {
    RowPlace place[STAGES];
    Cursor tile[STAGES];
    int requested = 0;
#pragma unroll
    for (int s = 0; s < STAGES; s++)
      if (more_ahead) {
        place[s] = locate<W::kRows>(p, ahead);
        tile[s] = ahead;
        requested = s + 1;
        more_ahead = next_unit(p, ahead, ahead_at, share.size);
      }
#pragma unroll
    for (int s = 0; s < STAGES; s++) {
      if (s < requested) request<T, D, W::kRows>(p, tile[s], place[s], stages + s * Stage::kBytes, &join.note[warp][s]);
      copies_commit();
    }
  }
  RowPlace next = {-1, 0};
  if (more_ahead) next = locate<W::kRows>(p, ahead);

  W work;
  work.load(p, now);
  work.start(p, now, shared);
  auto refill = [&](int stage) {
    if (more_ahead) {
      request<T, D, W::kRows>(p, ahead, next, stages + stage * Stage::kBytes, &join.note[warp][stage]);
      more_ahead = next_unit(p, ahead, ahead_at, share.size);
      if (more_ahead) next = locate<W::kRows>(p, ahead);
    }
    copies_commit();
  };
  for (int stage = 0;; stage = stage + 1 == STAGES ? 0 : stage + 1) {
    copies_wait<STAGES - 1>();
    __syncwarp();
    store_fresh<T, D, W::kRows>(p, join.note[warp][stage], stages + stage * Stage::kBytes);
    work.step(p, now, stages + stage * Stage::kBytes, join.note[warp][stage].mask, scale2);
    __syncwarp();
    const Cursor done = now;
    const long long segment = share.begin + at - done.tile;  // number of its first tile
    const bool more = next_unit(p, now, at, share.size);
    if (more && done.tile + 1 < done.tiles) {
      refill(stage);
      continue;
    }

    // This block's part of the segment is complete. The warps' sums take the place of the stages just read.
    if (more) work.load(p, now);
    work.statistics(&join.stat[warp][0].x);
    work.values(reinterpret_cast<float*>(stages + stage * Stage::kBytes), kPitch);
    __syncthreads();
    const int g = done.group / p.groups, h0 = (done.group % p.groups) * H;
    const int heads = min(H, p.rep - h0);
    const long long first = segment / share.quota, last = (segment + done.tiles - 1) / share.quota;
    const int others = (int)(last - first);
    // Slot 1 of a block holds the segment that begins in it, slot 0 the one that began before it.
    constexpr int kSlot = H * (D + 2);
    float* mine = p.space.partials + ((long long)blockIdx.x * 2 + (blockIdx.x == first ? 1 : 0)) * kSlot;
    T* out = static_cast<T*>(p.a.out) + done.b * p.a.out_batch_stride + (long long)(g * p.rep + h0) * p.a.out_head_stride;
    const float* sums = reinterpret_cast<const float*>(smem + stage * Stage::kBytes);
    for (int j = threadIdx.x; j < heads * (D / 4); j += kThreads) {
      const int h = j / (D / 4), d = j % (D / 4) * 4;
      float top = -INFINITY, total = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; w++) top = max_nan(top, join.stat[w][h].x);
#pragma unroll
      for (int w = 0; w < kWarps; w++) {
        const float2 stat = join.stat[w][h];
        const float f = stat.x == -INFINITY ? 0.f : exp2_fast(stat.x - top);
        const float4 y = *reinterpret_cast<const float4*>(sums + w * (STAGES * Stage::kBytes / 4) + h * kPitch + d);
        total = fmaf(f, stat.y, total);
        x.x = fmaf(f, y.x, x.x);
        x.y = fmaf(f, y.y, x.y);
        x.z = fmaf(f, y.z, x.z);
        x.w = fmaf(f, y.w, x.w);
      }
      if (others == 0) {
        finish(p, done.b, g * p.rep + h0 + h, d, out + h * p.a.out_head_stride, x, top, total);
      } else {
        *reinterpret_cast<float4*>(mine + j * 4) = x;
        if (d == 0) *reinterpret_cast<float2*>(mine + H * D + 2 * h) = make_float2(top, total);
      }
    }
    if (others) {
      __syncthreads();
      if (threadIdx.x == 0) {  // its fences stand for the whole block: the barriers order the others' accesses before and behind them
        __threadfence();
        join.last = atomicInc(p.space.counters + (long long)done.b * p.c.kv_heads * p.groups + done.group, (unsigned)others) == (unsigned)others;
        __threadfence();
      }
      __syncthreads();
      if (join.last) {
        merge<T, W, D>(p, done.b, g * p.rep + h0, heads, p.space.partials + first * 2 * kSlot, others + 1, out,
                       smem + stage * Stage::kBytes);  // the first warp's sums have been read
      }
    }
    if (!more) break;
    __syncthreads();  // the stages are filled again, and so is `join`
    refill(stage);
    work.start(p, now, shared);
  }
}

constexpr int kTrackThreads = 256;

// weights[t] += sum over heads of e^(s_t - lse). A thread a row. What it needs is requested at once, also where the row turns out
// not to be there: the kernel is a few microseconds behind the attention, and most of them are one trip to memory. 16 sequences up
// to 4096 rows: 6 us of the 45 of both kernels (13 MB of scores and weights, mostly from L2).
template <int REP>  // query heads of a KV head; 0: any number
__global__ void __launch_bounds__(kTrackThreads) paged_track_kernel(PagedView c, AttendSpace space, int heads, int appended) {
  PJRTX_PDL_PROLOGUE();
  const int g = blockIdx.y, b = blockIdx.z, rep = heads / c.kv_heads, capacity = c.page_size * c.max_pages;
  const long long base = ((long long)b * c.kv_heads + g) * capacity;
  const float* lse2 = space.lse2 + (long long)b * heads + g * rep;
  for (int t = blockIdx.x * kTrackThreads + threadIdx.x; t < capacity; t += gridDim.x * kTrackThreads) {
    const int n = paged_length(c, b);
    const float* s = space.scores + (base + t) * rep;
    float w = 0.f;
    if constexpr (REP > 0) {
      const float was = c.weights[base + t];
      float x[REP], l[REP];
#pragma unroll
      for (int r = 0; r < REP; r++) {
        x[r] = s[r];
        l[r] = lse2[r];
      }
#pragma unroll
      for (int r = 0; r < REP; r++) w += l[r] == -INFINITY ? 0.f : exp2_fast(x[r] - l[r]);
      if (!(appended && t == n - 1)) w += was;
    } else {
      for (int r = 0; r < rep; r++) w += lse2[r] == -INFINITY ? 0.f : exp2_fast(s[r] - lse2[r]);
      if (!(appended && t == n - 1)) w += c.weights[base + t];
    }
    if (t >= n) break;
    c.weights[base + t] = w;
    if (appended && t == n - 1) c.positions[base + t] = c.tokens[b] - 1;
  }
}

// Which kernel a shape runs on.
struct AttendPlan {
  int dims = 0;    // dimensions a row is padded to
  int heads = 0;   // query heads of a group
  int rows = 0;    // of a warp's part of a tile
  int stages = 0, per_sm = 0;
  size_t smem = 0;
};

template <typename T, typename W, int D, int STAGES>
constexpr size_t attend_smem() {
  return (size_t)kWarps * STAGES * RowStage<T, D, W::kRows>::kBytes + W::kSharedBytes + sizeof(JoinSpace<W>);
}

// Dimensions are padded to 64, 128 or 256, and each width gets the stages and blocks an SM that its shared memory and registers allow:
//   16 bits, 64: 32 rows a warp and step, since 16 (4 KB) wait longer for each other than they take: 46.6 us, not 42.1, where 128 MB
//   are read. For 128 the same costs a block's second stage: 39.5 us, not 38.7.
//   16 bits, over 8 query heads a KV head: 16 columns at once, which read the rows once but leave registers for one block (three
//   stages; four: 24.9, not 24.0; two blocks spill: 33.9). 16 heads, 32 sequences up to 8000 rows: 53.6 us, as two groups of eight
//   56.5; 12 heads, 8 sequences: 16.2, not 17.1; with little to read the two groups are the faster (2 sequences: 17.9, not 21.8).
//   f32, 128 and more: two stages of 8 rows, not one of 16 (rows in flight while others are at work): 8 sequences up to 2048 rows 26.4
//   us, not 27.1, 4 of 155 with eight heads a KV head 11.6, not 13.9. 64: two stages of 16, not four of 8: 69.0 us, not 80.5, at 53
//   sequences up to 2487. Two blocks an SM, not one with twice the stages: 26.4 us, not 32.8.
//   f32, up to 4 query heads a KV head: arithmetic for four: 26.4 us, 31.9 with that for eight. Up to 2 and heads of 65 to 128: for two,
//   one stage of 16 rows: 50 sequences up to 399 rows 30.8 us, 33.8 with that for four (heads of 64: 38.8 and 39.0, so not there).
template <typename F>
auto with_kernel(int dtype, int head_dim, int rep, F&& f) {
#define PJRTX_ATTEND(T, W, D, S, N) return f(paged_attend_kernel<T, W, D, S, N>, AttendPlan{D, W::kHeads, W::kRows, S, N, attend_smem<T, W, D, S>()})
#define PJRTX_ATTEND_MMA(T, NB)                                                 \
  if (head_dim <= 64) { using W = MmaWarp<T, 64, NB, 32>; PJRTX_ATTEND(T, W, 64, 2, 2); }  \
  if (head_dim <= 128) { using W = MmaWarp<T, 128, NB, 16>; PJRTX_ATTEND(T, W, 128, NB == 1 ? 2 : 3, NB == 1 ? 2 : 1); } \
  { using W = MmaWarp<T, 256, 1, 16>; PJRTX_ATTEND(T, W, 256, 2, 1); }
#define PJRTX_ATTEND_FMA(H)                                                     \
  if (head_dim <= 64) { using W = FmaWarp<64, H, 16>; PJRTX_ATTEND(float, W, 64, 2, 2); }  \
  if (head_dim <= 128) { using W = FmaWarp<128, H, 8>; PJRTX_ATTEND(float, W, 128, 2, 2); } \
  { using W = FmaWarp<256, H, 8>; PJRTX_ATTEND(float, W, 256, 2, 1); }
  if (dtype == kF32) {
    if (rep <= 2 && head_dim > 64 && head_dim <= 128) { using W = FmaWarp<128, 2, 16>; PJRTX_ATTEND(float, W, 128, 1, 2); }
    if (rep <= 4) { PJRTX_ATTEND_FMA(4) }
    PJRTX_ATTEND_FMA(8)
  }
  if (dtype == kF16) {
    if (rep <= 8) { PJRTX_ATTEND_MMA(__half, 1) }
    PJRTX_ATTEND_MMA(__half, 2)
  }
  if (rep <= 8) { PJRTX_ATTEND_MMA(__nv_bfloat16, 1) }
  PJRTX_ATTEND_MMA(__nv_bfloat16, 2)
#undef PJRTX_ATTEND_FMA
#undef PJRTX_ATTEND_MMA
#undef PJRTX_ATTEND
}

uint64_t round256(uint64_t n) { return (n + 255) / 256 * 256; }

struct AttendLayout {
  uint64_t counters, partials, scores, bytes;
};

// Places go by the largest batch, so that the counters stay where they are.
AttendLayout attend_layout(const PagedView& c, int heads, const AttendPlan& plan, bool track, int sm_count) {
  const int rep = heads / c.kv_heads, groups = (rep + plan.heads - 1) / plan.heads;
  AttendLayout l;
  l.counters = round256((uint64_t)c.batch_max * heads * 4);
  l.partials = l.counters + round256((uint64_t)c.batch_max * c.kv_heads * groups * 4);
  l.scores = l.partials + round256((uint64_t)sm_count * plan.per_sm * 2 * plan.heads * (plan.dims + 2) * 4);
  l.bytes = l.scores + (track ? (uint64_t)c.batch_max * heads * c.capacity() * 4 : 0);
  return l;
}

}  // namespace

WorkspaceSize paged_attend_workspace(const PagedView& c, int heads, bool track, int sm_count) {
  return with_kernel(c.dtype, c.head_dim, heads / c.kv_heads, [&](auto, const AttendPlan& plan) {
    const AttendLayout l = attend_layout(c, heads, plan, track, sm_count);
    return WorkspaceSize{l.bytes, l.partials};
  });
}

int paged_attend_launch(const PagedView& c, const PagedAttend& a, int sm_count, bool pdl, cudaStream_t stream) {
  AttendArgs p;
  p.c = c;
  p.a = a;
  p.rep = a.heads / c.kv_heads;
  p.pieces = c.head_dim * (int)dtype_size(c.dtype) / 16;
  p.reciprocal = (unsigned)std::min<uint64_t>((1ull << 32) / c.page_size, 0xffffffffu);
  const bool ok = with_kernel(c.dtype, c.head_dim, p.rep, [&](auto kernel, const AttendPlan& plan) {
    const AttendLayout l = attend_layout(c, a.heads, plan, false, sm_count);
    char* space = static_cast<char*>(a.workspace);
    p.groups = (p.rep + plan.heads - 1) / plan.heads;
    p.tile_rows = kWarps * plan.rows;
    p.space.lse2 = reinterpret_cast<float*>(space);
    p.space.counters = reinterpret_cast<unsigned*>(space + l.counters);
    p.space.partials = reinterpret_cast<float*>(space + l.partials);
    p.space.scores = reinterpret_cast<float*>(space + l.scores);
    if (!raise_smem_limit((const void*)kernel, (int)plan.smem)) return false;
    const long long numbers = (long long)c.batch * c.kv_heads * p.groups * ((c.capacity() + p.tile_rows - 1) / p.tile_rows + kSegmentCost);
    const long long blocks = std::min<long long>(numbers, (long long)sm_count * plan.per_sm);
    return launch_kernel(kernel, dim3((unsigned)blocks), dim3(kThreads), plan.smem, stream, pdl, p) == cudaSuccess;
  });
  if (!ok) return 0;
  if (!c.weights) return 1;
  const long long pairs = (long long)c.batch * c.kv_heads;
  const long long blocks = std::max<long long>(1, std::min((c.capacity() + kTrackThreads - 1) / kTrackThreads, 8ll * sm_count / pairs + 1));
  auto kernel = p.rep == 1 ? paged_track_kernel<1> : p.rep == 2 ? paged_track_kernel<2> : p.rep == 4 ? paged_track_kernel<4>
                : p.rep == 8 ? paged_track_kernel<8> : paged_track_kernel<0>;
  return launch_kernel(kernel, dim3((unsigned)blocks, (unsigned)c.kv_heads, (unsigned)c.batch), dim3(kTrackThreads), 0, stream, true, c, p.space,
                       a.heads, (int)(a.k_new != nullptr)) == cudaSuccess ? 2 : 0;
}

}  // namespace pjrtx
