"""The gated-DeltaNet layer over a tree of drafted tokens on gfx950 (new ops, next to
deltanet::verify_batched; the token step is deltanet::full_batched's,
contrib/qwen3.6-27b/kernels/deltanet_full_batched_ops.py:22-41).

A tree: parent [B, T] int32, T <= 64; node t hangs on node parent[b, t] where that lies in [0, t), else on
the committed tokens alone; node 0 is the last committed token.

  deltanet::verify_tree(state [B*Hv*128, 128] f32, parent, mixed_qkv [B*T*QKV] bf16,
                        conv_state [B*QKV, 3] bf16, conv_weight, conv_bias, a_out, b_out [B*T*Hv] f32,
                        z [B*T*Hv, 128] bf16, A_log, dt_bias, norm_weight)
      -> (out [B*T*Hv, 128] bf16, records [B*T*((Hk+Hv)*128 + Hv)] f32)
      Every node's token step from the state and conv window behind its parent. No state per node:
      records (k, u and decay of each node) are what a commit needs.
  deltanet::commit_tree_(states, conv_states, mixed_qkvs, records, path [B, T] int32, v_heads) -> ()
      Lists of every layer's tensors; states and conv_states are moved along the path (the accepted nodes
      in order, -1 behind; spec::accept_tree's) in place, all layers in one launch.

include/npn_spec_verify.h has the details and limits.
"""
import torch

from deltanet_full_batched_ops import K_DIM, V_DIM, heads_from_shapes
from npn_native import check_all, check_lists, launch, register

MAX_NODES = 64
I32, F32, BF16 = torch.int32, torch.float32, torch.bfloat16


def tree_shape(t, name):
    """(B, T) of a [B, T] argument of a tree."""
    if t.dim() != 2:
        raise RuntimeError(f"{name} must be [B, T], got {tuple(t.shape)}")
    B, T = t.shape
    if not 1 <= T <= MAX_NODES:
        raise RuntimeError(f"a tree has 1 to {MAX_NODES} nodes, {name} has T={T}")
    if not 1 <= B <= 65535:
        raise RuntimeError(f"unsupported batch of {B} trees")
    return B, T


def _records(B, T, hk, hv):
    return B * T * ((hk + hv) * K_DIM + hv)


def _verify_tree_fake(state, parent, mixed_qkv, conv_state, conv_weight, conv_bias, a_out, b_out, z, A_log,
                      dt_bias, norm_weight):
    hk, hv = heads_from_shapes(conv_weight.shape[0], A_log.shape[0])
    B, T = parent.shape
    return (state.new_empty((B * T * hv, V_DIM), dtype=BF16), state.new_empty((_records(B, T, hk, hv),)))


@register("deltanet::verify_tree",
          "(Tensor state, Tensor parent, Tensor mixed_qkv, Tensor conv_state, Tensor conv_weight, "
          "Tensor conv_bias, Tensor a_out, Tensor b_out, Tensor z, Tensor A_log, Tensor dt_bias, "
          "Tensor norm_weight) -> (Tensor, Tensor)", _verify_tree_fake)
def verify_tree(state, parent, mixed_qkv, conv_state, conv_weight, conv_bias, a_out, b_out, z, A_log,
                dt_bias, norm_weight):
    B, T = tree_shape(parent, "parent")
    qkv, hv = conv_weight.shape[0], A_log.numel()
    hk, hv = heads_from_shapes(qkv, hv)
    dev, n = state.device, B * T * hv
    check_all(dev, (state, "state", F32, (B * hv * K_DIM, V_DIM)), (parent, "parent", I32, (B, T)),
              (mixed_qkv, "mixed_qkv", BF16, B * T * qkv), (conv_state, "conv_state", BF16, (B * qkv, 3)),
              (conv_weight, "conv_weight", F32, (qkv, 4)), (conv_bias, "conv_bias", F32, qkv),
              (a_out, "a_out", F32, n), (b_out, "b_out", F32, n), (z, "z", BF16, n * V_DIM),
              (A_log, "A_log", F32, hv), (dt_bias, "dt_bias", F32, hv),
              (norm_weight, "norm_weight", F32, V_DIM))
    out = torch.empty((n, V_DIM), dtype=BF16, device=dev)
    records = torch.empty(_records(B, T, hk, hv), dtype=F32, device=dev)
    launch(dev, "npn_deltanet_verify_tree", state, parent, mixed_qkv, conv_state, conv_weight, conv_bias,
           a_out, b_out, z, A_log, dt_bias, norm_weight, out, records, B, T, hk, hv)
    return out, records


def _commit_tree_fake(states, conv_states, mixed_qkvs, records, path, v_heads):
    return None


@register("deltanet::commit_tree_",
          "(Tensor(a!)[] states, Tensor(b!)[] conv_states, Tensor[] mixed_qkvs, Tensor[] records, "
          "Tensor path, int v_heads) -> ()", _commit_tree_fake)
def commit_tree_(states, conv_states, mixed_qkvs, records, path, v_heads):
    layers = len(states)
    if not layers == len(conv_states) == len(mixed_qkvs) == len(records):
        raise RuntimeError("commit_tree_: one conv_state, mixed_qkv and records for each state")
    B, T = tree_shape(path, "path")
    dev = path.device
    check_all(dev, (path, "path", I32, (B, T)))
    if layers == 0:
        return
    qkv = conv_states[0].shape[0] // B
    hk, hv = heads_from_shapes(qkv, v_heads)
    lists = check_lists(dev, (states, "states", F32, (B * hv * K_DIM, V_DIM)),
                        (conv_states, "conv_states", BF16, (B * qkv, 3)), (mixed_qkvs, "mixed_qkvs", BF16, B * T * qkv),
                        (records, "records", F32, _records(B, T, hk, hv)))
    launch(dev, "npn_deltanet_commit_tree", *lists, layers, path, B, T, hk, hv)
