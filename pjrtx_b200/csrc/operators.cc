#include "operators.h"

#include <cmath>

#include "kernels/kernels.h"

namespace pjrtx {

namespace {

constexpr int64_t kMaxHeadDim = 256;
constexpr int64_t kMaxCapacity = 1 << 30;  // rows of one sequence
constexpr int64_t kMaxTracked = 1ll << 40;  // scores of a tracked cache's workspace: 4 TB; sizes beyond 2^60 would not fit 64 bits
constexpr int64_t kMaxPacked = 1 << 24, kMaxSequences = 1 << 20;  // of packed prompts
constexpr int64_t kMaxVocab = 1 << 22;     // the chunk maxima of a row stay in shared memory

bool refuse(const char* fmt, long long a = 0, long long b = 0, long long c = 0) {
  set_last_error(fmt, a, b, c);
  return false;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Whether a stride keeps 16-byte pieces aligned; where the axis has one element it is not used.
bool stride_ok(int64_t stride, int64_t extent, int dtype) { return extent <= 1 || (stride > 0 && stride * (int64_t)dtype_size(dtype) % 16 == 0); }

bool entered(const CurrentDevice& scope, const Device* dev) { return scope.ok || refuse("cudaSetDevice(%lld) failed", dev->ordinal); }

bool launched(int kernels, const char* what) {
  if (kernels > 0) return true;
  set_last_error("%s: launch failed: %s", what, cudaGetErrorString(cudaGetLastError()));
  return false;
}

// Completes a view with the cache's geometry and checks it.
bool complete(const PagedCache& cache, PagedView* v, bool sequences = true) {
  const PagedCacheConfig& c = cache.config;
  v->batch_max = (int)c.batch;
  v->kv_heads = (int)c.kv_heads;
  v->head_dim = (int)c.head_dim;
  v->page_size = (int)c.page_size;
  v->max_pages = (int)c.max_pages;
  v->dtype = c.dtype;
  v->error_words = cache.device->operator_words_dev;
  if (v->batch < 0 || v->batch > c.batch) return refuse("paged cache: a batch of %lld, the cache was made for up to %lld", v->batch, c.batch);
  // Arrays of no sequences may have no address.
  if (!v->k || !v->v || (sequences && v->batch > 0 && (!v->table || !v->lengths))) return refuse("paged cache: null pages, page table or lengths");
  if (v->num_pages < 1 || v->num_pages > INT32_MAX) return refuse("paged cache: %lld pages", v->num_pages);
  if (!aligned16(v->k) || !aligned16(v->v) || !stride_ok(v->page_stride, v->num_pages, c.dtype) ||
      !stride_ok(v->row_stride, c.page_size, c.dtype) || !stride_ok(v->head_stride, c.kv_heads, c.dtype))
    return refuse("paged cache: pages need 16-byte aligned rows (page, row and head strides %lld, %lld, %lld elements)", v->page_stride,
                  v->row_stride, v->head_stride);
  if (sequences && v->batch > 1 && v->table_stride < c.max_pages)
    return refuse("paged cache: a page table of %lld columns, the cache has %lld pages a sequence", v->table_stride, c.max_pages);
  if ((v->weights != nullptr) != (v->positions != nullptr)) return refuse("paged cache: weights and positions go together");
  if (v->weights && !c.track) return refuse("paged cache: weights need a cache that was made to track them");
  return true;
}

}  // namespace

PagedCache* paged_cache_create(int ordinal, const PagedCacheConfig& c) {
  auto bad = [](bool) -> PagedCache* { return nullptr; };
  if (!dtype_is_float(c.dtype)) return bad(refuse("paged cache: element type %lld; f32, f16 and bf16 are supported", c.dtype));
  if (c.batch < 1 || c.batch > 65535 || c.kv_heads < 1 || c.kv_heads > 65535 || c.heads < c.kv_heads || c.heads > 65535 || c.heads % c.kv_heads)
    return bad(refuse("paged cache: batch %lld, %lld query heads, %lld KV heads (up to 65535 each, query heads a multiple of KV heads)", c.batch,
                      c.heads, c.kv_heads));
  if (c.head_dim < 1 || c.head_dim > kMaxHeadDim || c.head_dim * (int64_t)dtype_size(c.dtype) % 16)
    return bad(refuse("paged cache: head dimension %lld (up to %lld, a multiple of 16 bytes)", c.head_dim, kMaxHeadDim));
  if (c.page_size < 1 || c.max_pages < 1 || c.page_size > kMaxCapacity || c.max_pages > kMaxCapacity || c.page_size * c.max_pages > kMaxCapacity)
    return bad(refuse("paged cache: %lld pages of %lld rows a sequence (up to %lld rows)", c.max_pages, c.page_size, kMaxCapacity));
  if (c.track && c.batch * c.heads * (c.page_size * c.max_pages) > kMaxTracked)
    return bad(refuse("paged cache: %lld sequences, %lld query heads and %lld rows are too many for a workspace of scores", c.batch, c.heads,
                      c.page_size * c.max_pages));
  if (c.tree_nodes < 0 || c.tree_nodes > kTreeNodesMax)
    return bad(refuse("paged cache: trees of %lld nodes (up to %lld)", c.tree_nodes, kTreeNodesMax));
  Device* dev = get_device_aside(ordinal);
  if (!dev) return nullptr;
  PagedCache made;
  made.device = dev;
  made.config = c;
  PagedView v;
  v.batch = v.batch_max = (int)c.batch;
  v.kv_heads = (int)c.kv_heads;
  v.head_dim = (int)c.head_dim;
  v.page_size = (int)c.page_size;
  v.max_pages = (int)c.max_pages;
  v.dtype = c.dtype;
  const WorkspaceSize attend = paged_attend_workspace(v, (int)c.heads, c.track, dev->sm_count);
  const WorkspaceSize evict = c.track ? paged_evict_workspace(v) : WorkspaceSize{0, 0};
  const uint64_t evict_at = (attend.bytes + 255) / 256 * 256;
  const uint64_t tree_at = (evict_at + evict.bytes + 255) / 256 * 256;
  const uint64_t tree = c.tree_nodes ? paged_tree_workspace(v, (int)c.heads, (int)c.tree_nodes, dev->sm_count) : 0;
  made.bytes = tree ? tree_at + tree : evict_at + evict.bytes;
  CurrentDevice scope(dev->ordinal);
  if (!entered(scope, dev)) return nullptr;
  made.attend_space = device_malloc(dev, made.bytes);
  if (!made.attend_space) return nullptr;
  made.evict_space = c.track ? static_cast<char*>(made.attend_space) + evict_at : nullptr;
  made.tree_space = tree ? static_cast<char*>(made.attend_space) + tree_at : nullptr;
  // Other streams may use the workspaces once this returns.
  const bool ok = check_cuda(cudaMemsetAsync(made.attend_space, 0, attend.zeroed, dev->stream), "cudaMemsetAsync") &&
                  (!c.track || check_cuda(cudaMemsetAsync(made.evict_space, 0, evict.zeroed, dev->stream), "cudaMemsetAsync")) &&
                  check_cuda(cudaStreamSynchronize(dev->stream), "cudaStreamSynchronize");
  if (!ok) {
    device_free(dev, made.attend_space, made.bytes);
    return nullptr;
  }
  return new PagedCache(made);
}

void paged_cache_destroy(PagedCache* cache) {
  if (!cache) return;
  CurrentDevice scope(cache->device->ordinal);
  cudaDeviceSynchronize();  // calls on any stream may still use the workspaces
  device_free(cache->device, cache->attend_space, cache->bytes);
  delete cache;
}

int paged_cache_append(const PagedCache& cache, PagedView view, const PagedAppend& a, cudaStream_t stream) {
  if (!complete(cache, &view)) return 0;
  const PagedCacheConfig& c = cache.config;
  if (view.weights && !view.tokens) return refuse("append: a tracked cache needs the sequences' token counts");
  if (a.rows < 0 || a.rows > INT32_MAX) return refuse("append: %lld new rows", a.rows);
  if (view.batch == 0 || a.rows == 0) return 1;
  if (!a.k_new || !a.v_new || !aligned16(a.k_new) || !aligned16(a.v_new) || !stride_ok(a.batch_stride, view.batch, c.dtype) ||
      !stride_ok(a.row_stride, a.rows, c.dtype) || !stride_ok(a.head_stride, c.kv_heads, c.dtype))
    return refuse("append: new rows need 16-byte aligned pointers and strides (%lld, %lld, %lld elements)", a.batch_stride, a.row_stride, a.head_stride);
  CurrentDevice scope(cache.device->ordinal);
  if (!entered(scope, cache.device)) return 0;
  return launched(paged_append_launch(view, a, cache.device->sm_count, true, stream), "append");
}

int paged_cache_attend(const PagedCache& cache, PagedView view, PagedAttend a, cudaStream_t stream) {
  if (!complete(cache, &view)) return 0;
  const PagedCacheConfig& c = cache.config;
  a.heads = (int)c.heads;
  a.workspace = cache.attend_space;
  if (view.batch == 0) return 1;
  if ((a.k_new != nullptr) != (a.v_new != nullptr)) return refuse("attend: a new key and a new value go together");
  if (view.weights && a.k_new && !view.tokens) return refuse("attend: a tracked cache needs the sequences' token counts with a new row");
  if (!std::isfinite(a.scale)) return refuse("attend: the scale is not finite");
  if (!a.q || !a.out || !aligned16(a.q) || !aligned16(a.out) || !stride_ok(a.q_batch_stride, view.batch, c.dtype) ||
      !stride_ok(a.q_head_stride, c.heads, c.dtype) || !stride_ok(a.out_batch_stride, view.batch, c.dtype) ||
      !stride_ok(a.out_head_stride, c.heads, c.dtype))
    return refuse("attend: queries and results need 16-byte aligned pointers and strides");
  if (a.k_new && (!aligned16(a.k_new) || !aligned16(a.v_new) || !stride_ok(a.new_batch_stride, view.batch, c.dtype) ||
                  !stride_ok(a.new_head_stride, c.kv_heads, c.dtype)))
    return refuse("attend: the new row needs 16-byte aligned pointers and strides (%lld, %lld elements)", a.new_batch_stride, a.new_head_stride);
  CurrentDevice scope(cache.device->ordinal);
  if (!entered(scope, cache.device)) return 0;
  return launched(paged_attend_launch(view, a, cache.device->sm_count, true, stream), "attend");
}

int paged_cache_evict(const PagedCache& cache, PagedView view, PagedEvict e, cudaStream_t stream) {
  if (!complete(cache, &view)) return 0;
  e.workspace = cache.evict_space;
  if (e.keep < 1 || e.recent < 0 || e.sinks < 0 || (int64_t)e.recent + e.sinks > e.keep)
    return refuse("evict: %lld rows to keep, %lld recent and %lld first tokens (at least 1, and room for the protected ones)", e.keep, e.recent, e.sinks);
  if (view.batch == 0) return 1;
  if (!view.weights || !view.tokens) return refuse("evict: weights, positions and the sequences' token counts are needed");
  if (!e.lengths_out || !e.weights_out || !e.positions_out) return refuse("evict: null lengths, weights or positions to write");
  CurrentDevice scope(cache.device->ordinal);
  if (!entered(scope, cache.device)) return 0;
  return launched(paged_evict_launch(view, e, cache.device->sm_count, true, stream), "evict");
}

int paged_cache_attend_tree(const PagedCache& cache, PagedView view, PagedTree a, cudaStream_t stream) {
  if (!complete(cache, &view)) return 0;
  const PagedCacheConfig& c = cache.config;
  a.heads = (int)c.heads;
  a.workspace = cache.tree_space;
  if (a.nodes < 0 || a.nodes > c.tree_nodes) return refuse("attend to a tree: %lld nodes, the cache was made for up to %lld", a.nodes, c.tree_nodes);
  if (view.batch == 0 || a.nodes == 0) return 1;
  if (!std::isfinite(a.scale)) return refuse("attend to a tree: the scale is not finite");
  if (!a.parents) return refuse("attend to a tree: null parents");
  if (!a.q || !a.out || !aligned16(a.q) || !aligned16(a.out) || !stride_ok(a.q_batch_stride, view.batch, c.dtype) ||
      !stride_ok(a.q_node_stride, a.nodes, c.dtype) || !stride_ok(a.q_head_stride, c.heads, c.dtype) ||
      !stride_ok(a.out_batch_stride, view.batch, c.dtype) || !stride_ok(a.out_node_stride, a.nodes, c.dtype) ||
      !stride_ok(a.out_head_stride, c.heads, c.dtype))
    return refuse("attend to a tree: queries and results need 16-byte aligned pointers and strides");
  if (!a.k_new || !a.v_new || !aligned16(a.k_new) || !aligned16(a.v_new) || !stride_ok(a.new_batch_stride, view.batch, c.dtype) ||
      !stride_ok(a.new_node_stride, a.nodes, c.dtype) || !stride_ok(a.new_head_stride, c.kv_heads, c.dtype))
    return refuse("attend to a tree: its keys and values need 16-byte aligned pointers and strides (%lld, %lld, %lld elements)", a.new_batch_stride,
                  a.new_node_stride, a.new_head_stride);
  if (a.out == a.q || a.out == a.k_new || a.out == a.v_new) return refuse("attend to a tree: the results can not take the place of an input");
  CurrentDevice scope(cache.device->ordinal);
  if (!entered(scope, cache.device)) return 0;
  return launched(paged_tree_launch(view, a, cache.device->sm_count, true, stream), "attend to a tree");
}

int paged_cache_store(const PagedCache& cache, PagedView view, const PagedStore& a, cudaStream_t stream) {
  view.batch = 0;
  if (!complete(cache, &view, false)) return 0;
  const PagedCacheConfig& c = cache.config;
  if (a.rows < 0 || a.rows > INT32_MAX) return refuse("store: %lld rows", a.rows);
  if (view.num_pages * c.page_size > INT32_MAX) return refuse("store: %lld pages of %lld rows, slots have 32 bits", view.num_pages, c.page_size);
  if (a.rows == 0) return 1;
  if (!a.slots) return refuse("store: null slots");
  if (!a.k_new || !a.v_new || !aligned16(a.k_new) || !aligned16(a.v_new) || !stride_ok(a.row_stride, a.rows, c.dtype) ||
      !stride_ok(a.head_stride, c.kv_heads, c.dtype))
    return refuse("store: rows need 16-byte aligned pointers and strides (%lld, %lld elements)", a.row_stride, a.head_stride);
  CurrentDevice scope(cache.device->ordinal);
  if (!entered(scope, cache.device)) return 0;
  return launched(paged_store_launch(view, a, cache.device->sm_count, true, stream), "store");
}

int paged_cache_assign(const PagedCache& cache, PagedAssign a, int64_t batch, int64_t num_pages, cudaStream_t stream) {
  const PagedCacheConfig& c = cache.config;
  if (batch < 0 || batch > c.batch) return refuse("assign pages: a batch of %lld, the cache was made for up to %lld", batch, c.batch);
  if (num_pages < 1 || num_pages > INT32_MAX || num_pages * c.page_size > INT32_MAX)
    return refuse("assign pages: %lld pages of %lld rows (up to 2^31 - 1 rows)", num_pages, c.page_size);
  if (a.tokens < 0 || a.tokens > INT32_MAX) return refuse("assign pages: %lld tokens", a.tokens);
  if (!a.free_pages || !a.free_count || !a.free_pages_out || !a.free_count_out) return refuse("assign pages: null stack of free pages");
  if (batch > 0 && (!a.lengths || !a.held || !a.table || !a.held_out || !a.table_out)) return refuse("assign pages: null lengths, page counts or page table");
  if (batch > 1 && (a.table_stride < c.max_pages || a.table_out_stride < c.max_pages))
    return refuse("assign pages: a page table of %lld and %lld columns, the cache has %lld pages a sequence", a.table_stride, a.table_out_stride, c.max_pages);
  if (a.table == a.table_out && a.table && batch > 1 && a.table_stride != a.table_out_stride)
    return refuse("assign pages: in place, but the table's rows are %lld and %lld apart", a.table_stride, a.table_out_stride);
  if (a.tokens > 0 && a.slots && !a.starts) return refuse("assign pages: slots need the starts of the sequences");
  if (a.tokens > 0 && !a.slots) return refuse("assign pages: null slots");
  a.batch = (int)batch;
  a.num_pages = (int)num_pages;
  a.page_size = (int)c.page_size;
  a.max_pages = (int)c.max_pages;
  a.error_words = cache.device->operator_words_dev;
  CurrentDevice scope(cache.device->ordinal);
  if (!entered(scope, cache.device)) return 0;
  return launched(paged_assign_launch(a, true, stream), "assign pages");
}

int paged_cache_path_slots(const PagedCache& cache, PagedPath a, int64_t batch, int64_t nodes, cudaStream_t stream) {
  const PagedCacheConfig& c = cache.config;
  if (batch < 0 || batch > c.batch) return refuse("path slots: a batch of %lld, the cache was made for up to %lld", batch, c.batch);
  if (nodes < 0 || nodes > kTreeNodesMax) return refuse("path slots: %lld nodes (up to %lld)", nodes, kTreeNodesMax);
  if (batch == 0) return 1;
  if (!a.table || !a.lengths || !a.leaves || !a.lengths_out || (nodes > 0 && (!a.parents || !a.slots)))
    return refuse("path slots: null page table, lengths, parents, leaves or slots");
  if (batch > 1 && a.table_stride < c.max_pages)
    return refuse("path slots: a page table of %lld columns, the cache has %lld pages a sequence", a.table_stride, c.max_pages);
  a.batch = (int)batch;
  a.nodes = (int)nodes;
  a.page_size = (int)c.page_size;
  a.max_pages = (int)c.max_pages;
  a.error_words = cache.device->operator_words_dev;
  CurrentDevice scope(cache.device->ordinal);
  if (!entered(scope, cache.device)) return 0;
  return launched(paged_path_launch(a, true, stream), "path slots");
}

int prompt_attention(int ordinal, PromptAttention a, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t sequences, cudaStream_t stream) {
  if (!dtype_is_float(a.dtype)) return refuse("prompt attention: element type %lld; f32, f16 and bf16 are supported", a.dtype);
  if (kv_heads < 1 || kv_heads > 65535 || heads < kv_heads || heads > 65535 || heads % kv_heads)
    return refuse("prompt attention: %lld query heads, %lld KV heads (up to 65535 each, query heads a multiple of KV heads)", heads, kv_heads);
  if (head_dim < 1 || head_dim > kMaxHeadDim || head_dim * (int64_t)dtype_size(a.dtype) % 16)
    return refuse("prompt attention: head dimension %lld (up to %lld, a multiple of 16 bytes)", head_dim, kMaxHeadDim);
  if (a.tokens < 0 || a.tokens > kMaxPacked || sequences < 0 || sequences > kMaxSequences)
    return refuse("prompt attention: %lld tokens of %lld sequences (up to 2^24 and 2^20)", a.tokens, sequences);
  if (!std::isfinite(a.scale)) return refuse("prompt attention: the scale is not finite");
  if (a.tokens == 0 || sequences == 0) return 1;
  if (!a.starts) return refuse("prompt attention: null starts");
  if (!a.q || !a.k || !a.v || !a.out || !aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.out) ||
      !stride_ok(a.q_stride, a.tokens, a.dtype) || !stride_ok(a.q_head_stride, heads, a.dtype) || !stride_ok(a.k_stride, a.tokens, a.dtype) ||
      !stride_ok(a.k_head_stride, kv_heads, a.dtype) || !stride_ok(a.v_stride, a.tokens, a.dtype) || !stride_ok(a.v_head_stride, kv_heads, a.dtype) ||
      !stride_ok(a.out_stride, a.tokens, a.dtype) || !stride_ok(a.out_head_stride, heads, a.dtype))
    return refuse("prompt attention: queries, keys, values and results need 16-byte aligned pointers and strides");
  if (a.out == a.q || a.out == a.k || a.out == a.v) return refuse("prompt attention: the results can not take the place of an input");
  a.heads = (int)heads;
  a.kv_heads = (int)kv_heads;
  a.head_dim = (int)head_dim;
  a.sequences = (int)sequences;
  Device* dev = get_device_aside(ordinal);
  if (!dev) return 0;
  a.error_words = dev->operator_words_dev;
  CurrentDevice scope(dev->ordinal);
  if (!entered(scope, dev)) return 0;
  return launched(prompt_attention_launch(a, true, stream), "prompt attention");
}

namespace {

bool check_logits(const char* what, int dtype, const void* logits, long long rows, long long vocab, long long row_stride, const int* tokens, float scale) {
  if (!dtype_is_float(dtype)) {
    set_last_error("%s: element type %d; f32, f16 and bf16 are supported", what, dtype);
    return false;
  }
  if (rows < 0 || rows > (1 << 27) || vocab < 1 || vocab > kMaxVocab || (rows > 1 && row_stride < vocab)) {
    set_last_error("%s: %lld rows of %lld logits, %lld apart (up to 2^27 rows of %lld)", what, rows, vocab, row_stride, (long long)kMaxVocab);
    return false;
  }
  if (!(scale > 0.f) || !std::isfinite(scale)) {
    set_last_error("%s: the scale must be positive and finite", what);
    return false;
  }
  if (rows && (!logits || !tokens || (uintptr_t)logits % dtype_size(dtype))) {
    set_last_error("%s: null or misaligned logits, or no tokens", what);
    return false;
  }
  return true;
}

}  // namespace

int token_log_probs(int ordinal, TokenScore s, cudaStream_t stream) {
  const char* what = "token log probabilities";
  if (!check_logits(what, s.dtype, s.logits, s.rows, s.vocab, s.row_stride, s.tokens, s.scale)) return 0;
  if (s.top < 0 || s.top > kScoreTopMax || s.top > s.vocab)
    return refuse("token log probabilities: %lld alternatives (up to %lld, and no more than the vocabulary's %lld)", s.top, kScoreTopMax, s.vocab);
  if (s.top && !s.top_ids && !s.top_log_probs) return refuse("token log probabilities: alternatives are asked for and have no place");
  if (s.rows == 0) return 1;
  if (!s.log_probs) return refuse("token log probabilities: null result");
  Device* dev = get_device_aside(ordinal);
  if (!dev) return 0;
  s.error_words = dev->operator_words_dev;
  CurrentDevice scope(dev->ordinal);
  if (!entered(scope, dev)) return 0;
  return launched(token_score_launch(s, dev->sm_count, true, stream), what);
}

int token_log_probs_backward(int ordinal, TokenScoreGrad s, cudaStream_t stream) {
  const char* what = "gradient of token log probabilities";
  if (!check_logits(what, s.dtype, s.logits, s.rows, s.vocab, s.row_stride, s.tokens, s.scale)) return 0;
  if (!s.grad_log_probs && !s.grad_entropy) return refuse("gradient of token log probabilities: no incoming gradient");
  if (s.rows * (s.vocab / 1024 + 2) > INT32_MAX) return refuse("gradient of token log probabilities: %lld x %lld logits in one call", s.rows, s.vocab);
  if (s.rows == 0) return 1;
  if (!s.lse || (s.grad_entropy && !s.entropy)) return refuse("gradient of token log probabilities: null log-sum-exp or entropy");
  if (!s.grad_logits || (uintptr_t)s.grad_logits % dtype_size(s.dtype) || (s.rows > 1 && s.grad_row_stride < s.vocab))
    return refuse("gradient of token log probabilities: null, misaligned or overlapping result rows");
  if (s.grad_logits == s.logits && s.rows > 1 && s.grad_row_stride != s.row_stride)
    return refuse("gradient of token log probabilities: in place, but the rows are %lld and %lld apart", s.row_stride, s.grad_row_stride);
  Device* dev = get_device_aside(ordinal);
  if (!dev) return 0;
  s.error_words = dev->operator_words_dev;
  CurrentDevice scope(dev->ordinal);
  if (!entered(scope, dev)) return 0;
  return launched(token_score_grad_launch(s, dev->sm_count, true, stream), what);
}

int operators_status(int ordinal, cudaStream_t stream) {
  Device* dev = get_device_aside(ordinal);
  if (!dev) return 0;
  CurrentDevice scope(dev->ordinal);
  if (!entered(scope, dev)) return 0;
  return check_cuda(cudaStreamSynchronize(stream), "cudaStreamSynchronize") && check_operator_words(dev);
}

}  // namespace pjrtx
