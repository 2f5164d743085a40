// Causal attention of whole prompts, packed one behind the other, with grouped query heads. A tile of query rows is some positions of
// one sequence times the query heads of a KV head: row x is head x % heads of position x / heads, so the rows of a tile share its keys.
//
// The starts of the sequences are on the device: the grid has a block for every tile that there can be, sequence b's from
// starts[b] / positions + b on (a sequence of n tokens has at most that many before the next one's), and blocks without a tile leave. The
// tiles of a sequence run from its end, where they have most to do, to its beginning, a tile for all KV heads before the next tile.
//
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = e^(scale q_i . k_j - m_i), j <= i of the same sequence,  m_i following max_j scale q_i . k_j
//
// Of n tokens that is 2 n (n + 1) heads head_dim operations on 2 n (heads + kv_heads) head_dim elements: bound by arithmetic from some hundred
// tokens on, by latency below. 16-bit types go to the tensor cores (umma_prompt.cuh), f32 to the CUDA cores (row_attention.cuh).
#include <algorithm>
#include <type_traits>

#include "../common.h"
#include "kernels.h"
#include "paged.cuh"
#include "row_attention.cuh"

namespace pjrtx {

namespace {

struct PromptArgs {
  PromptAttention a;
  int rep, heads, groups;  // query heads of a KV head; those of a tile; tiles that share a position
  int positions;           // of a tile
};

struct PromptTile {
  int start, tokens, tile;  // tile < 0: none
};

// Tile `x` of the launch, for all lanes of a warp. Sequences that are not in order are skipped.
__device__ __forceinline__ PromptTile prompt_tile(const PromptArgs& p, long long x) {
  const int lane = threadIdx.x % 32, positions = p.positions, *starts = p.a.starts;
  int b = 0, n = p.a.sequences;
  while (n > 1) {  // the last sequence whose first tile is not behind x
    const int step = (n + 31) / 32, at = b + lane * step;
    const bool before = lane * step < n && starts[at] / positions + (long long)at <= x;
    const int seen = max(1, __popc(__ballot_sync(~0u, before)));
    b += (seen - 1) * step;
    n = min(step, n - (seen - 1) * step);
  }
  const int start = starts[b], end = starts[b + 1];
  PromptTile t = {start, end - start, -1};
  if (start < 0 || end < start || end > p.a.tokens) return t;
  const long long at = x - (start / positions + (long long)b), tiles = (t.tokens + positions - 1) / positions;
  if (at >= 0 && at < tiles) t.tile = (int)(tiles - 1 - at);
  return t;
}

// The grid: heads by tiles, the tiles folded where one axis does not hold them.
constexpr long long kGridAxis = 65535;
__device__ __forceinline__ long long prompt_block() { return blockIdx.z * kGridAxis + blockIdx.y; }
inline dim3 prompt_grid(const PromptArgs& p) {
  const long long tiles = p.a.tokens / p.positions + p.a.sequences;
  return dim3((unsigned)(p.a.kv_heads * p.groups), (unsigned)std::min(tiles, kGridAxis), (unsigned)((tiles + kGridAxis - 1) / kGridAxis));
}

__device__ __forceinline__ void check_starts(const PromptAttention& a) {
  if (blockIdx.x) return;
  const long long step = (long long)gridDim.y * gridDim.z * blockDim.x;
  for (long long b = (blockIdx.z * (long long)gridDim.y + blockIdx.y) * blockDim.x + threadIdx.x; b < a.sequences; b += step)
    if (a.starts[b] < 0 || a.starts[b + 1] < a.starts[b] || a.starts[b + 1] > a.tokens) report(a.error_words, kErrorLength);
}

}  // namespace
}  // namespace pjrtx

#include "umma_prompt.cuh"

namespace pjrtx {
namespace {

// In f32.
constexpr int kRowsOfThread = 4;

template <int D>
__global__ void __launch_bounds__(rows::kThreads) prompt_rows_kernel(const __grid_constant__ PromptArgs p) {
  PJRTX_PDL_PROLOGUE();
  using namespace rows;
  constexpr int R = kRowsOfThread;
  using Space = Shared<D, R>;
  extern __shared__ __align__(16) char smem[];
  Space& s = *reinterpret_cast<Space*>(smem);
  const PromptAttention& a = p.a;
  check_starts(a);
  const PromptTile t = prompt_tile(p, prompt_block());
  if (t.tile < 0) return;
  const int g = blockIdx.x / p.groups, h0 = blockIdx.x % p.groups * p.heads, heads = min(p.heads, p.rep - h0);
  const int first = t.tile * p.positions, positions = min(p.positions, t.tokens - first);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  auto place = [&](int r, int* position, int* head) {
    *position = first + r / p.heads;
    *head = r % p.heads;
    return r / p.heads < positions && *head < heads;
  };
  const int keys = first + positions;
  const float* any = static_cast<const float*>(a.q);
  const float* k = static_cast<const float*>(a.k) + (long long)t.start * a.k_stride + (long long)g * a.k_head_stride;
  const float* v = static_cast<const float*>(a.v) + (long long)t.start * a.v_stride + (long long)g * a.v_head_stride;
  auto request = [&](int stage) {
    constexpr int kOfWarp = Space::kKeys / 8;
    const int key = stage * Space::kKeys + warp * kOfWarp + lane;
    const bool there = lane < kOfWarp && key < keys;
    request_rows<D, Space::kKeys>(s.k[stage & 1], there ? k + key * a.k_stride : nullptr, a.head_dim, any);
    request_rows<D, Space::kKeys>(s.v[stage & 1], there ? v + key * a.v_stride : nullptr, a.head_dim, any);
  };
  {
    constexpr int kOfWarp = Space::kRows / 8;
    int position, head;
    const float* q = nullptr;
    if (lane < kOfWarp && place(warp * kOfWarp + lane, &position, &head))
      q = any + (long long)(t.start + position) * a.q_stride + (long long)(g * p.rep + h0 + head) * a.q_head_stride;
    request_rows<D, Space::kRows>(s.q, q, a.head_dim, any);
  }
  request(0);
  Sight sight[R];
  Sums<D, R> sum;
  sum.clear();
#pragma unroll
  for (int i = 0; i < R; i++) {
    int position, head;
    sight[i] = {place(ty * R + i, &position, &head) ? position + 1 : 0, 0ull};
  }
  int reach = 0;
#pragma unroll
  for (int i = 0; i < R; i++) reach = max(reach, sight[i].limit);
  reach = __reduce_max_sync(~0u, reach);
  const int blocks = (keys + Space::kKeys - 1) / Space::kKeys;
  for (int j = 0; j < blocks; j++)
    block_of_keys<true, D, R>(s, sum, sight, j, j * Space::kKeys, keys, reach, keys, a.scale * kLog2e, [&] {
      if (j + 1 < blocks) request(j + 1);
    });
#pragma unroll
  for (int i = 0; i < R; i++) {
    int position, head;
    if (!place(ty * R + i, &position, &head)) continue;
    const long long row = t.start + position;
    const int h = g * p.rep + h0 + head;
    const float inverse = inverse_of(sum.l[i]);
    float* out = static_cast<float*>(a.out) + row * a.out_stride + h * a.out_head_stride;
#pragma unroll
    for (int c = 0; c < D / 64; c++) {
      const float2 x = pair_split(sum.o[i][c][0]), y = pair_split(sum.o[i][c][1]);
      if (c * 64 + tx * 4 < a.head_dim) store4(out + c * 64 + tx * 4, make_float4(x.x * inverse, x.y * inverse, y.x * inverse, y.y * inverse));
    }
    if (a.lse && tx == 0) a.lse[row * a.heads + h] = lse_of(sum.m[i], sum.l[i]);
  }
}

template <int D>
int launch_rows(PromptArgs p, bool pdl, cudaStream_t stream) {
  using Space = rows::Shared<D, kRowsOfThread>;
  if (!raise_smem_limit((const void*)prompt_rows_kernel<D>, (int)sizeof(Space))) return 0;
  p.heads = std::min(p.rep, Space::kRows);
  p.groups = (p.rep + p.heads - 1) / p.heads;
  p.positions = Space::kRows / p.heads;
  return launch_kernel(prompt_rows_kernel<D>, prompt_grid(p), dim3(rows::kThreads), sizeof(Space), stream, pdl, p) == cudaSuccess;
}

template <bool BF16, int HD>
int launch_umma(const umma::PromptKernelArgs& a, bool pdl, cudaStream_t stream) {
  const PromptAttention& p = a.p.a;
  const long long q_extents[4] = {p.head_dim, a.p.rep, p.kv_heads, p.tokens}, k_extents[3] = {p.head_dim, p.tokens, p.kv_heads};
  const long long q_strides[3] = {p.q_head_stride, a.p.rep * p.q_head_stride, p.q_stride};
  const long long k_strides[2] = {p.k_stride, p.k_head_stride}, v_strides[2] = {p.v_stride, p.v_head_stride};
  const int q_box[4] = {64, a.p.heads, 1, a.p.positions}, k_box[3] = {64, umma::kPromptKeys, 1};
  CUtensorMap qmap, kmap, vmap;
  if (!umma::encode_map(&qmap, p.q, !BF16, 4, q_extents, q_strides, q_box) || !umma::encode_map(&kmap, p.k, !BF16, 3, k_extents, k_strides, k_box) ||
      !umma::encode_map(&vmap, p.v, !BF16, 3, k_extents, v_strides, k_box))
    return 0;
  constexpr size_t smem = umma::prompt_smem(HD);
  auto kernel = umma::umma_prompt_kernel<BF16, HD>;
  if (!raise_smem_limit((const void*)kernel, (int)smem)) return 0;
  return launch_kernel(kernel, prompt_grid(a.p), dim3(umma::kPromptThreads), smem, stream, pdl, a, qmap, kmap, vmap) == cudaSuccess;
}

template <bool BF16>
int launch_umma_of(PromptArgs p, bool pdl, cudaStream_t stream) {
  umma::PromptKernelArgs a;
  p.heads = std::min(p.rep, umma::kAttnRows);
  p.groups = (p.rep + p.heads - 1) / p.heads;
  p.positions = umma::kAttnRows / p.heads;
  a.p = p;
  const float scale = p.a.scale;
  a.scale_log2 = scale == 0.f ? 1.f : (scale < 0.f ? -scale : scale) * rows::kLog2e;
  a.sign = scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f;
  a.timeout_ns = wait_timeout_ns();
  return p.a.head_dim <= 64    ? launch_umma<BF16, 64>(a, pdl, stream)
         : p.a.head_dim <= 128 ? launch_umma<BF16, 128>(a, pdl, stream)
                               : launch_umma<BF16, 256>(a, pdl, stream);
}

}  // namespace

int prompt_attention_launch(const PromptAttention& a, bool pdl, cudaStream_t stream) {
  PromptArgs p;
  p.a = a;
  p.rep = a.heads / a.kv_heads;
  if (a.dtype == kF16) return launch_umma_of<false>(p, pdl, stream);
  if (a.dtype == kBF16) return launch_umma_of<true>(p, pdl, stream);
  return a.head_dim <= 64 ? launch_rows<64>(p, pdl, stream) : a.head_dim <= 128 ? launch_rows<128>(p, pdl, stream) : launch_rows<256>(p, pdl, stream);
}

}  // namespace pjrtx
