// The operators' entry points on a machine of two devices that exists only here: the CUDA runtime is a few functions that keep a current
// device, the kernels' launches note where they were made. Prints what is wrong; nothing when all is right.
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "operators.h"

using namespace pjrtx;

static int g_current = 0, g_launched_on = -1, g_refused = -1;
static char g_error[512];

namespace pjrtx {
void set_last_error(const char* fmt, ...) {
  va_list args;
  va_start(args, fmt);
  vsnprintf(g_error, sizeof g_error, fmt, args);
  va_end(args);
}
const char* last_error() { return g_error; }
static int note() {
  g_launched_on = g_current;
  return 1;
}
WorkspaceSize paged_attend_workspace(const PagedView&, int, bool, int) { return {1024, 256}; }
WorkspaceSize paged_evict_workspace(const PagedView&) { return {1024, 256}; }
int paged_append_launch(const PagedView&, const PagedAppend&, int, bool, cudaStream_t) { return note(); }
int paged_attend_launch(const PagedView&, const PagedAttend&, int, bool, cudaStream_t) { return note(); }
int paged_evict_launch(const PagedView&, const PagedEvict&, int, bool, cudaStream_t) { return note(); }
int token_score_launch(const TokenScore&, int, bool, cudaStream_t) { return note(); }
int token_score_grad_launch(const TokenScoreGrad&, int, bool, cudaStream_t) { return note(); }
}  // namespace pjrtx

extern "C" {
cudaError_t cudaGetDeviceCount(int* n) { return *n = 2, cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { return *d = g_current, cudaSuccess; }
cudaError_t cudaSetDevice(int d) {
  if (d < 0 || d > 1 || d == g_refused) return cudaErrorInvalidDevice;
  g_current = d;
  return cudaSuccess;
}
cudaError_t cudaGetDeviceProperties_v2(cudaDeviceProp* p, int) {
  memset(p, 0, sizeof *p);
  p->major = 10;
  p->multiProcessorCount = 148;
  return cudaSuccess;
}
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned) { return *s = (cudaStream_t)8, cudaSuccess; }
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { return *e = (cudaEvent_t)8, cudaSuccess; }
cudaError_t cudaDeviceGetDefaultMemPool(cudaMemPool_t* p, int) { return *p = (cudaMemPool_t)8, cudaSuccess; }
cudaError_t cudaMemPoolSetAttribute(cudaMemPool_t, cudaMemPoolAttr, void*) { return cudaSuccess; }
cudaError_t cudaMallocHost(void** p, size_t n) { return *p = calloc(1, n), cudaSuccess; }
cudaError_t cudaHostAlloc(void** p, size_t n, unsigned) { return *p = calloc(1, n), cudaSuccess; }
cudaError_t cudaHostGetDevicePointer(void** d, void* h, unsigned) { return *d = h, cudaSuccess; }
cudaError_t cudaMallocAsync(void** p, size_t n, cudaStream_t) { return *p = calloc(1, n), cudaSuccess; }
cudaError_t cudaFreeAsync(void* p, cudaStream_t) { return free(p), cudaSuccess; }
cudaError_t cudaMemsetAsync(void*, int, size_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaDeviceSynchronize() { return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "refused"; }
}

static void expect(bool ok, const char* what) {
  if (!ok) printf("%s: current %d, launched on %d, last error: %s\n", what, g_current, g_launched_on, g_error);
}

int main(int argc, char** argv) {
  alignas(16) static char memory[4096];
  static int ints[64];
  float* floats = reinterpret_cast<float*>(memory);
  // The first use of device 1, with device 0 current, by the entry point that the argument names.
  const char* first = argc > 1 ? argv[1] : "";
  TokenScore score;
  score.dtype = kF32; score.logits = memory; score.rows = 1; score.vocab = 8; score.row_stride = 8; score.tokens = ints; score.log_probs = floats;
  TokenScoreGrad grad;
  grad.dtype = kF32; grad.logits = memory; grad.grad_logits = memory; grad.rows = 1; grad.vocab = 8; grad.row_stride = grad.grad_row_stride = 8;
  grad.tokens = ints; grad.lse = floats; grad.grad_log_probs = floats;
  PagedCacheConfig config;
  config.dtype = kF32; config.track = true; config.batch = config.heads = config.kv_heads = 1; config.head_dim = 4; config.page_size = 16; config.max_pages = 2;
  PagedView view;
  view.k = view.v = memory; view.num_pages = 2; view.page_stride = 64; view.row_stride = view.head_stride = 4; view.table = ints; view.table_stride = 2;
  view.lengths = view.tokens = ints; view.batch = 1; view.weights = floats; view.positions = ints;
  PagedAppend append;
  append.k_new = append.v_new = memory; append.rows = 1;
  PagedAttend attend;
  attend.q = attend.out = memory;
  PagedEvict evict;
  evict.keep = 4; evict.lengths_out = ints; evict.weights_out = floats; evict.positions_out = ints;

  PagedCache* cache = nullptr;
  if (!strcmp(first, "score")) token_log_probs(1, score, nullptr);
  if (!strcmp(first, "grad")) token_log_probs_backward(1, grad, nullptr);
  if (!strcmp(first, "status")) operators_status(1, nullptr);
  if (!strcmp(first, "stream")) get_device_aside(1);
  if (!strcmp(first, "cache")) cache = paged_cache_create(1, config);
  expect(g_current == 0, "first use");
  if (!cache) cache = paged_cache_create(1, config);
  expect(cache && g_current == 0, "cache");

  auto each = [&](bool want, const char* what) {
    auto one = [&](int got, bool launches) {
      expect((got != 0) == want && g_current == 0 && (!want || !launches || g_launched_on == 1) && (want || g_launched_on == -1), what);
      g_launched_on = -1;
    };
    one(paged_cache_append(*cache, view, append, nullptr), true);
    one(paged_cache_attend(*cache, view, attend, nullptr), true);
    one(paged_cache_evict(*cache, view, evict, nullptr), true);
    one(token_log_probs(1, score, nullptr), true);
    one(token_log_probs_backward(1, grad, nullptr), true);
    one(operators_status(1, nullptr), false);
  };
  g_launched_on = -1;
  each(true, "call");
  g_refused = 1;  // the device can not be made current any more
  each(false, "refused device");
  expect(!paged_cache_create(1, config) && g_current == 0, "cache on a refused device");
  g_refused = -1;
  expect(!token_log_probs(2, score, nullptr) && g_current == 0, "no such device");
  paged_cache_destroy(cache);
  expect(g_current == 0, "destroy");
  return 0;
}
