// draft_tree.hpp — trees of drafted tokens: the newest tokens of a sequence, at most 64 of them, each with the place
// of its parent among them.  A wave holds a tree with node j in lane j.
#pragma once

#include "serve.hpp"

namespace bsgk {

constexpr int kTreeNodes = 64;

// The parent of node `lane` of a sequence whose tokens begin at `from`; -1 where there is none, where the node does not
// exist, and where it is no earlier node.  parents == null: a chain.
__device__ __forceinline__ int load_parent(const int32_t* parents, int64_t from, int count, int lane) {
  const int v = lane < count ? (parents ? parents[from + lane] : lane - 1) : -1;
  return v >= 0 && v < lane ? v : -1;
}

__device__ __forceinline__ int from_lane(int v, int lane) { return __builtin_amdgcn_ds_bpermute(lane << 2, v); }
__device__ __forceinline__ uint64_t from_lane(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)from_lane((int)(v >> 32), lane) << 32 | (uint32_t)from_lane((int)v, lane);
}

// Node `lane` and its ancestors, as bits: a node takes over what its ancestor 1, 2, 4 ... steps up has, and that one's
// ancestor as many steps further up, so that a chain of 64 takes six rounds.
__device__ __forceinline__ uint64_t lineage_of(int parent, int lane) {
  uint64_t mask = 1ull << lane;
  for (int up = parent; __any(up >= 0);) {
    const int at = up < 0 ? lane : up;
    mask |= from_lane(mask, at);
    const int next = from_lane(up, at);
    up = up < 0 ? -1 : next;
  }
  return mask;
}

// How many ancestors node `lane` has.
__device__ __forceinline__ int depth_of(int parent, int lane) {
  int depth = parent >= 0 ? 1 : 0;
  for (int up = parent; __any(up >= 0);) {
    const int at = up < 0 ? lane : up;
    const int more = from_lane(depth, at), next = from_lane(up, at);
    if (up >= 0) depth += more, up = next;
  }
  return depth;
}

}  // namespace bsgk
