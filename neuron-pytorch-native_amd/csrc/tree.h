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

__device__ __forceinline__ uint64_t shfl64(uint64_t x, int from) {
  const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)x, from, kWave);
  return ((uint64_t)(uint32_t)__shfl((int)(x >> 32), from, kWave) << 32) | lo;
}

// Node `lane` and its ancestors as bits, by pointer doubling: after k steps a lane knows 2^k nodes up and
// the next one. `sum`, the lane's number, becomes the sum over those nodes'.
__device__ __forceinline__ uint64_t tree_ancestors(int parent, int T, int lane, double& sum) {
  uint64_t bits = 1ull << lane;
  int up = parent;
  for (int n = 1; n < T; n <<= 1) {
    const int from = up < 0 ? lane : up;
    const uint64_t other = shfl64(bits, from), more = shfl64((uint64_t)__double_as_longlong(sum), from);
    const int next = __shfl(up, from, kWave);
    bits |= other;
    sum += up < 0 ? 0.0 : __longlong_as_double((long long)more);
    up = up < 0 ? up : next;
  }
  return bits;
}
__device__ __forceinline__ uint64_t tree_ancestors(int parent, int T, int lane) {
  double none = 0.0;
  return tree_ancestors(parent, T, lane, none);
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
