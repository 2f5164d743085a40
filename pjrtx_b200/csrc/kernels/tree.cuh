// Trees of drafted tokens: a node's ancestors as bits.
#pragma once

#include "paged.cuh"

namespace pjrtx {

// Ancestors of nodes `lane` and `lane + 32`, themselves among them.
struct Ancestors {
  unsigned long long low, high;
};

__device__ __forceinline__ unsigned long long tree_of_node(const Ancestors& a, int node) {
  const unsigned long long low = __shfl_sync(~0u, a.low, node & 31), high = __shfl_sync(~0u, a.high, node & 31);
  return node < 32 ? low : high;
}

// By doubling: after i rounds a node knows its 2^i nearest ancestors and where to go on. Called by a whole warp; a parent that is not a
// node before its child is reported and counts as none, so every way ends. Only the parents of the first `nodes` are read: what lies behind
// a sequence's nodes may hold anything.
__device__ __forceinline__ Ancestors tree_ancestors(const int* parents, int nodes, int* error_words) {
  const int lane = threadIdx.x % 32;
  int up[2];
  unsigned long long set[2];
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int node = lane + u * 32;
    up[u] = node < nodes ? parents[node] : -1;
    if (up[u] < -1 || up[u] >= node) {
      report(error_words, kErrorParent);
      up[u] = -1;
    }
    set[u] = 1ull << node;
  }
  for (int reach = 1; reach < nodes; reach *= 2) {
    unsigned long long add[2];
    int next[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int at = max(up[u], 0);
      const unsigned long long low = __shfl_sync(~0u, set[0], at & 31), high = __shfl_sync(~0u, set[1], at & 31);
      const int low_up = __shfl_sync(~0u, up[0], at & 31), high_up = __shfl_sync(~0u, up[1], at & 31);
      add[u] = up[u] < 0 ? 0 : at < 32 ? low : high;
      next[u] = up[u] < 0 ? -1 : at < 32 ? low_up : high_up;
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      set[u] |= add[u];
      up[u] = next[u];
    }
  }
  return {set[0], set[1]};
}

}  // namespace pjrtx
