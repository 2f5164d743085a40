// Launch wrappers of the operators that a host calls directly, on its own stream: a paged key-value cache (append, attend,
// evict) and the scoring of logits (log probabilities, entropy, likeliest tokens, gradient). As in kernels.h, a wrapper
// enqueues on the given stream and returns the number of kernels it launched (0 = a launch failed). Arguments were checked.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace pjrtx {

// Codes for arguments which only the device can see. Kernels set error_words[code - kErrorPageId], host-mapped memory of the device.
constexpr int kErrorPageId = 40;   // a page table entry of a sequence's own rows names no page of the pool
constexpr int kErrorLength = 41;   // a length is negative or beyond the page table, or a count does not fit its length
constexpr int kErrorToken = 42;    // a token id is not below the vocabulary size
constexpr int kErrorWords = 3;

// Row t of sequence b: page table[b * table_stride + t / page_size], row t % page_size of it; element d of KV head g of that row
// is at page * page_stride + row * row_stride + g * head_stride + d in both pools. Strides count elements.
struct PagedView {
  void* k = nullptr;
  void* v = nullptr;
  long long num_pages = 0, page_stride = 0, row_stride = 0, head_stride = 0;
  const int* table = nullptr;
  long long table_stride = 0;
  const int* lengths = nullptr;  // visible rows of each sequence, those that the call appends among them
  // Tracking (null: none): tokens[b] seen by sequence b so far; weights / positions [batch, kv_heads, capacity].
  const int* tokens = nullptr;
  float* weights = nullptr;
  int* positions = nullptr;
  int batch = 0, batch_max = 0;  // of this call, and of any call on the same workspaces
  int kv_heads = 0, head_dim = 0, page_size = 0, max_pages = 0;
  int dtype = 0;
  int* error_words = nullptr;
  long long capacity() const { return (long long)page_size * max_pages; }
};

struct PagedAppend {
  const void* k_new = nullptr;  // [batch, rows, kv_heads, head_dim] through the strides
  const void* v_new = nullptr;
  long long batch_stride = 0, row_stride = 0, head_stride = 0;
  long long rows = 0;
  const int* counts = nullptr;  // new rows of each sequence (null: `rows` of every one)
};
int paged_append_launch(const PagedView& c, const PagedAppend& a, int sm_count, bool pdl, cudaStream_t stream);

struct PagedAttend {
  const void* q = nullptr;  // [batch, heads, head_dim] through the strides; query head h reads KV head h / (heads / kv_heads)
  long long q_batch_stride = 0, q_head_stride = 0;
  void* out = nullptr;
  long long out_batch_stride = 0, out_head_stride = 0;
  float* lse = nullptr;         // [batch, heads], may be null
  const void* k_new = nullptr;  // [batch, kv_heads, head_dim]: becomes row lengths[b] - 1 (null: that row is in the pool)
  const void* v_new = nullptr;
  long long new_batch_stride = 0, new_head_stride = 0;
  int heads = 0;
  float scale = 1.f;
  void* workspace = nullptr;
};
// Device memory that a call needs for `c`; the first `zeroed` bytes hold counters, which start out at zero and are left so.
struct WorkspaceSize {
  uint64_t bytes, zeroed;
};
WorkspaceSize paged_attend_workspace(const PagedView& c, int heads, bool track, int sm_count);
int paged_attend_launch(const PagedView& c, const PagedAttend& a, int sm_count, bool pdl, cudaStream_t stream);

struct PagedEvict {
  int keep = 0, recent = 0, sinks = 0;
  int* lengths_out = nullptr;      // may be the view's own, as may the next two
  float* weights_out = nullptr;
  int* positions_out = nullptr;
  void* workspace = nullptr;
};
WorkspaceSize paged_evict_workspace(const PagedView& c);
int paged_evict_launch(const PagedView& c, const PagedEvict& e, int sm_count, bool pdl, cudaStream_t stream);

struct TokenScore {
  int dtype = 0;
  const void* logits = nullptr;  // [rows, vocab], rows row_stride elements apart
  long long rows = 0, vocab = 0, row_stride = 0;
  const int* tokens = nullptr;
  float scale = 1.f;
  float* log_probs = nullptr;
  float* entropy = nullptr;  // this one and the rest may be null
  float* lse = nullptr;
  int* top_ids = nullptr;
  float* top_log_probs = nullptr;
  int top = 0;
  int* error_words = nullptr;
};
constexpr int kScoreTopMax = 64;
int token_score_launch(const TokenScore& s, int sm_count, bool pdl, cudaStream_t stream);

struct TokenScoreGrad {
  int dtype = 0;
  const void* logits = nullptr;
  void* grad_logits = nullptr;  // may be the logits themselves
  long long rows = 0, vocab = 0, row_stride = 0, grad_row_stride = 0;
  const int* tokens = nullptr;
  const float* lse = nullptr;
  const float* entropy = nullptr;
  const float* grad_log_probs = nullptr;  // null: zeros
  const float* grad_entropy = nullptr;    // null: zeros, `entropy` is then not read
  float scale = 1.f;
  int* error_words = nullptr;
};
int token_score_grad_launch(const TokenScoreGrad& s, int sm_count, bool pdl, cudaStream_t stream);

}  // namespace pjrtx
