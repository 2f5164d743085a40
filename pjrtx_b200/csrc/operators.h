// Operators that a host calls directly with device pointers and a stream of its own (no plan, no executable): argument checks,
// workspaces, launches. The kernels are in kernels/paged_cache.cu, paged_attention.cu, tree_attention.cu,
// page_tables.cu, prompt_attention.cu and token_score.cu.
#pragma once

#include "device.h"
#include "kernels/operators.h"

namespace pjrtx {

struct PagedCacheConfig {
  int dtype = kInvalid;
  bool track = false;
  int64_t batch = 0, heads = 0, kv_heads = 0, head_dim = 0, page_size = 0, max_pages = 0;
  int64_t tree_nodes = 0;
};

// Geometry and workspaces of one kind of cache; a program keeps one for all layers of a shape. Calls on one handle share its
// workspaces, so they must not overlap on the GPU.
struct PagedCache {
  Device* device = nullptr;
  PagedCacheConfig config;
  void* attend_space = nullptr;  // one allocation
  void* evict_space = nullptr;   // in it, with tracking
  void* tree_space = nullptr;    // in it, with tree_nodes
  uint64_t bytes = 0;
};

// Arguments are checked before the device is touched.
PagedCache* paged_cache_create(int ordinal, const PagedCacheConfig& config);  // nullptr + last_error
void paged_cache_destroy(PagedCache* cache);

// The callers fill in what their arguments say; the cache adds its geometry. 1, or 0 with last_error set.
int paged_cache_append(const PagedCache& cache, PagedView view, const PagedAppend& args, cudaStream_t stream);
int paged_cache_attend(const PagedCache& cache, PagedView view, PagedAttend args, cudaStream_t stream);
int paged_cache_evict(const PagedCache& cache, PagedView view, PagedEvict args, cudaStream_t stream);
int paged_cache_attend_tree(const PagedCache& cache, PagedView view, PagedTree args, cudaStream_t stream);
int paged_cache_store(const PagedCache& cache, PagedView view, const PagedStore& args, cudaStream_t stream);
// The sizes come as 64-bit numbers: what a kernel holds in fewer bits is checked first.
int paged_cache_assign(const PagedCache& cache, PagedAssign args, int64_t batch, int64_t num_pages, cudaStream_t stream);
int paged_cache_path_slots(const PagedCache& cache, PagedPath args, int64_t batch, int64_t nodes, cudaStream_t stream);
int prompt_attention(int ordinal, PromptAttention args, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t sequences, cudaStream_t stream);
int token_log_probs(int ordinal, TokenScore args, cudaStream_t stream);
int token_log_probs_backward(int ordinal, TokenScoreGrad args, cudaStream_t stream);
// Waits for the stream; 0 with last_error set where an operator on the device has met what only the device sees.
int operators_status(int ordinal, cudaStream_t stream);

}  // namespace pjrtx
