// Trees of drafted tokens, as the drafted-token kernels read them.
//
// The nodes of all trees are packed rows; tree s is rows cu[s] .. cu[s + 1), at
// most kTreeNodes of them, and parents[row] is the index of a node's parent
// within its own tree.  A node comes after its parent: a parent that is not an
// earlier node of the tree makes the node a root.  With 64 nodes the lanes of a
// wavefront are the nodes, and a node's ancestors are the bits of one word.
#pragma once

#include "common.hpp"

namespace sophia {

constexpr int kTreeNodes = 64;

struct Trees {
  const int32_t *cu;        // [n_trees + 1]
  const int32_t *parents;   // [rows]
  int64_t rows;
  int max_nodes;            // nodes of a tree past this many are not looked at
};

// First row and node count of tree s, within the rows whatever cu holds.
__device__ __forceinline__ int tree_nodes(const Trees &t, int s, int64_t &base) {
  const int64_t first = t.cu[s], end = t.cu[s + 1];
  base = iclamp64(first, 0, t.rows);
  return static_cast<int>(iclamp64(imin64(end, t.rows) - base, 0, t.max_nodes));
}

__device__ __forceinline__ int tree_parent(const Trees &t, int64_t base, int n, int node) {
  const int p = node < n ? t.parents[base + node] : -1;
  return p >= 0 && p < node ? p : -1;
}

// Every node's path (itself and its ancestors) as bits, in the lane of the node:
// doublings, after r of them `mask` holds the 2^r nodes next to the node on its path
// and `up` the one above those.  `jump(r, up)` sees each round's `up`, of as many
// rounds as the deepest path needs.
template <typename F>
__device__ __forceinline__ uint64_t tree_paths(int parent, int n, int lane, F jump) {
  uint64_t mask = lane < n ? 1ull << lane : 0;
  int up = parent;
#pragma unroll
  for (int r = 0; r < 6; ++r) {
    if (!__any(up >= 0)) break;
    jump(r, up);
    const int from = up < 0 ? lane : up;
    const uint32_t lo = __shfl(static_cast<uint32_t>(mask), from, 64);
    const uint32_t hi = __shfl(static_cast<uint32_t>(mask >> 32), from, 64);
    const int above = __shfl(up, from, 64);
    if (up >= 0) mask |= static_cast<uint64_t>(hi) << 32 | lo;
    up = up >= 0 ? above : -1;
  }
  return mask;
}

__device__ __forceinline__ f4 mfma_f32(float a, float b, const f4 &c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < INFINITY; }

// Sum, and maximum, over the 16 lanes of a row, in each of them.
__device__ __forceinline__ float row_sum16(float v) {
  v += dpp_rotate<0x128>(v);
  v += dpp_rotate<0x124>(v);
  v += dpp_rotate<0x122>(v);
  return v + dpp_rotate<0x121>(v);
}

__device__ __forceinline__ float row_max16(float v) {
  v = fmaxf(v, dpp_rotate<0x128>(v));
  v = fmaxf(v, dpp_rotate<0x124>(v));
  v = fmaxf(v, dpp_rotate<0x122>(v));
  return fmaxf(v, dpp_rotate<0x121>(v));
}

// Sum over this lane and those before it, without the LDS crossbar: shifts within
// the rows of 16 lanes, then each row's last sum on to the rows behind it.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int v) {
  v = dpp_add<0x111, 0xf>(v);   // row_shr:1, 2, 4, 8
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);   // row_bcast:15 into rows 1 and 3
  return dpp_add<0x143, 0xc>(v);   // row_bcast:31 into rows 2 and 3
}

}  // namespace sophia
