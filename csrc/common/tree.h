// Bounds rules of the drafted-token trees, shared by the sm_100a kernels and
// the host library (whose exports the CPU tests call).
#pragma once
#include <stdint.h>

#if defined(__CUDACC__)
#define TREE_HD __host__ __device__ __forceinline__
#else
#define TREE_HD inline
#endif

namespace tree {

constexpr int MAX_NODES = 64;  // one 64-bit ancestor mask per node
constexpr int PAGE = 16;       // tokens per KV page

// Keys of a lane: its cached prefix [0, base) and n_tree drafted nodes at
// rows base .. base + n_tree - 1, or -1 when they do not lie within t_lim
// keys and the table's `width` pages.
TREE_HD int lane_keys(int base, int n_tree, int t_lim, int width) {
  if (base < 0 || n_tree < 0 || n_tree > MAX_NODES) return -1;
  const int64_t t = (int64_t)base + n_tree;
  if (t > t_lim || t > (int64_t)width * PAGE) return -1;
  return (int)t;
}

TREE_HD bool page_ok(int page, int n_pages) { return page >= 0 && page < n_pages; }

// Whether key j of a lane is visible to a query with the given mask.
TREE_HD bool visible(int j, int base, int n_tree, uint64_t mask) {
  if (j < base) return j >= 0;
  return j - base < n_tree && ((mask >> (j - base)) & 1);
}

// Whether entry i of an accepted path (0 = p_0 < p_1 < ...) can be moved: inside
// the n-node tree and the table's `width` pages.
TREE_HD bool path_ok(const int* path, int i, int n, int base, int width) {
  const int p = path[i];
  if (base < 0 || p >= n || (i == 0 ? p != 0 : p <= path[i - 1])) return false;
  return (int64_t)base + p < (int64_t)width * PAGE;
}

// Parent of node i, or -1 where `parent` does not name an earlier node.
TREE_HD int parent_of(const int* parent, int i) {
  const int p = parent[i];
  return p >= 0 && p < i ? p : -1;
}

}  // namespace tree
