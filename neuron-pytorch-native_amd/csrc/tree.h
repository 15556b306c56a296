// Trees of drafted tokens: device helpers shared by the kernels that verify them.
//
// parent [B][T], T <= 64: node t of a request hangs on node parent[t] where that lies in [0, t), else on the
// committed tokens alone. A node sees the committed tokens, its ancestors and itself. A wave holds a
// request's tree, lane t its node t.
#pragma once

#include "npn_common.h"

namespace npn {

constexpr int kMaxNodes = 64;

// The lane's node's parent, -1: none (lanes past T are nodes without one).
__device__ __forceinline__ int tree_parent(const int32_t* parent, int T, int lane) {
  const int p = lane < T ? parent[lane] : -1;
  return p >= 0 && p < lane ? p : -1;
}

// Node `lane` and its ancestors as bits, by pointer doubling: after k steps a lane knows 2^k nodes up and
// the next one.
__device__ __forceinline__ uint64_t tree_ancestors(int parent, int T, int lane) {
  uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
  int up = parent;
  for (int n = 1; n < T; n <<= 1) {
    const int from = up < 0 ? lane : up;
    const uint32_t l = (uint32_t)__shfl((int)lo, from, kWave), h = (uint32_t)__shfl((int)hi, from, kWave);
    const int next = __shfl(up, from, kWave);
    lo |= l;
    hi |= h;
    up = up < 0 ? up : next;
  }
  return ((uint64_t)hi << 32) | lo;
}

// Lane `from`'s bits (wave-uniform `from`).
__device__ __forceinline__ uint64_t tree_bits(uint64_t bits, int from) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, from);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), from);
  return ((uint64_t)hi << 32) | lo;
}

// Entries of a path that count: from the first on, nodes of [0, T) in ascending order. `node` is the lane's
// entry (-1 past T).
__device__ __forceinline__ int path_length(int node, int T, int lane, bool ok = true) {
  const int before = __shfl_up(node, 1, kWave);
  const bool good = ok && lane < T && node < T && node > (lane > 0 ? before : -1);
  const uint64_t bad = ~__builtin_amdgcn_ballot_w64(good);
  return bad ? __builtin_ctzll(bad) : kMaxNodes;
}

}  // namespace npn
