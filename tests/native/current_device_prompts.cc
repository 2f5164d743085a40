// The entry points of prompts, trees, page tables and slots on the two devices of current_device.cc.
#define main decoding_main
#include "current_device.cc"
#undef main

namespace pjrtx {
uint64_t paged_tree_workspace(const PagedView&, int, int, int) { return 1024; }
int paged_tree_launch(const PagedView&, const PagedTree&, int, bool, cudaStream_t) { return note(); }
int paged_store_launch(const PagedView&, const PagedStore&, int, bool, cudaStream_t) { return note(); }
int paged_assign_launch(const PagedAssign&, bool, cudaStream_t) { return note(); }
int paged_path_launch(const PagedPath&, bool, cudaStream_t) { return note(); }
int prompt_attention_launch(const PromptAttention&, bool, cudaStream_t) { return note(); }
}  // namespace pjrtx

int main(int argc, char** argv) {
  alignas(16) static char memory[4096], results[4096];
  static int ints[64];
  PromptAttention prompt;
  prompt.dtype = kF32; prompt.q = prompt.k = prompt.v = memory; prompt.out = results; prompt.tokens = 1; prompt.starts = ints;
  PagedCacheConfig config;
  config.dtype = kF32; config.batch = config.heads = config.kv_heads = 1; config.head_dim = 4; config.page_size = 16; config.max_pages = 2;
  config.tree_nodes = 4;
  PagedView view;
  view.k = view.v = memory; view.num_pages = 2; view.page_stride = 64; view.row_stride = view.head_stride = 4; view.table = ints; view.table_stride = 2;
  view.lengths = ints; view.batch = 1;
  PagedTree tree;
  tree.q = tree.k_new = tree.v_new = memory; tree.out = results; tree.parents = ints; tree.nodes = 1;
  PagedStore store;
  store.k_new = store.v_new = memory; store.rows = 1; store.slots = ints;
  PagedAssign assign;
  assign.lengths = assign.held = assign.table = assign.free_pages = assign.free_count = ints;
  assign.held_out = assign.table_out = assign.free_pages_out = assign.free_count_out = ints;
  assign.table_stride = assign.table_out_stride = 2;
  PagedPath path;
  path.table = path.lengths = path.parents = path.leaves = path.slots = path.lengths_out = ints; path.table_stride = 2;

  // The first use of device 1, with device 0 current, by prompts or by the cache.
  if (argc > 1 && !strcmp(argv[1], "prompt")) prompt_attention(1, prompt, 1, 1, 4, 1, nullptr);
  expect(g_current == 0, "first use");
  PagedCache* cache = paged_cache_create(1, config);
  expect(cache && g_current == 0, "cache");
  auto each = [&](bool want, const char* what) {
    auto one = [&](int got) {
      expect((got != 0) == want && g_current == 0 && g_launched_on == (want ? 1 : -1), what);
      g_launched_on = -1;
    };
    one(prompt_attention(1, prompt, 1, 1, 4, 1, nullptr));
    one(paged_cache_attend_tree(*cache, view, tree, nullptr));
    one(paged_cache_store(*cache, view, store, nullptr));
    one(paged_cache_assign(*cache, assign, 1, 4, nullptr));
    one(paged_cache_path_slots(*cache, path, 1, 1, nullptr));
  };
  g_launched_on = -1;
  each(true, "call");
  g_refused = 1;  // the device can not be made current any more
  each(false, "refused device");
  expect(!paged_cache_create(1, config) && g_current == 0, "cache on a refused device");
  g_refused = -1;
  expect(!prompt_attention(2, prompt, 1, 1, 4, 1, nullptr) && g_current == 0, "no such device");
  paged_cache_destroy(cache);
  expect(g_current == 0, "destroy");
  return 0;
}
