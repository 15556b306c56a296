// The walk through a tree of drafted tokens: from node 0 to the first child whose token the target has
// chosen at the node, until there is none (lossless for target tokens that are each node's own sample).
// New op; the reference has no speculative path on the device (contrib/qwen3.6-27b/static_decode.py:1313
// is its argmax).
//
// One wave a request, lane t its node t: a step is one ballot over "my parent is this node and my token
// is its target's", so the walk takes as many steps as it accepts drafts and no memory in between. Bound
// by a launch and one chain of loads: 1.9 us for one request of 16 nodes, 2.9 for 256 of 64.
#include "tree.h"

namespace {

struct AcceptTreeArgs {
  const int64_t* target;  // [B][T]
  const int64_t* draft;
  const int32_t* parent;
  const int32_t* q_len;   // [B]
  int32_t* accepted;      // [B]
  int32_t* path;          // [B][T]
  int64_t* out_ids;
  int B, T;
};

__global__ __launch_bounds__(64) void accept_tree_kernel(AcceptTreeArgs a) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const size_t at = (size_t)b * a.T + lane;
  const bool in = lane < a.T;
  const int parent = npn::tree_parent(a.parent + (size_t)b * a.T, a.T, lane);
  const uint64_t target = in ? (uint64_t)a.target[at] : 0, draft = in ? (uint64_t)a.draft[at] : 0;
  const int n = min(max(a.q_len[b], 0), a.T);
  int node = 0, count = 0, my_node = -1;
  uint64_t my_id = ~0ull;
  while (n > 0) {  // node grows at every turn but the last
    const uint64_t token = npn::tree_bits(target, node);
    if (lane == count) {
      my_node = node;
      my_id = token;
    }
    ++count;
    const uint64_t next =
        __builtin_amdgcn_ballot_w64(parent == node && lane < n && draft == token && (int64_t)token >= 0);
    if (next == 0) break;
    node = __builtin_ctzll(next);
  }
  if (in) {
    a.path[at] = my_node;
    a.out_ids[at] = (int64_t)my_id;
  }
  if (lane == 0) a.accepted[b] = count - 1;
}

}  // namespace

extern "C" int npn_accept_tree(const int64_t* target_ids, const int64_t* draft_ids, const int32_t* parent,
                               const int32_t* q_len, int32_t* accepted, int32_t* path, int64_t* out_ids,
                               int B, int T, void* stream) {
  NPN_REQUIRE(target_ids && draft_ids && parent && q_len && accepted && path && out_ids, NPN_ERR_NULL);
  NPN_REQUIRE(B >= 1 && B <= 65535 && T >= 1 && T <= npn::kMaxNodes, NPN_ERR_SHAPE);
  const AcceptTreeArgs a{target_ids, draft_ids, parent, q_len, accepted, path, out_ids, B, T};
  hipLaunchKernelGGL(accept_tree_kernel, dim3(B), dim3(64), 0, static_cast<hipStream_t>(stream), a);
  return npn_launch_status();
}
