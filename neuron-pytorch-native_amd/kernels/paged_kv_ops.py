"""Paged 8-bit KV cache ops on gfx950 (new ops; the reference's decode graph keeps a dense cache,
contrib/qwen3.6-27b/static_decode.py:880-931).

The cache of one attention layer: N blocks of bs = 16, 32, 64 or 128 rows,
  cache_k [N, Hkv, bs, 256], cache_v [N, Hkv, 256, bs] (dims as rows) int8 holding e4m3fn bytes,
  k_scale, v_scale [N, Hkv] f32, powers of two: value = e4m3 * scale.
One block table serves all layers. Lengths stay on the device, so a step plans its own pages:

  paged::update_blocks_(kv_len [B] int32, new_len [B] int32, block_table [B, P] int32,
                        num_blocks [B] int32, free_blocks [N] int32, free_count [1] int32,
                        block_size, T) -> (slots [B, T] int64, granted [B] int32)
      Gives back the blocks past ceil((kv_len + new_len) / bs) and grants the missing ones, in
      request order while they last; block_table, num_blocks and the stack of free blocks are
      updated in place. slots of the new rows (-1: none), granted = new_len or 0 where refused.
  gqa::kv_append_paged(key, value [B, T, Hkv, 256] bf16, k_norm [256] f32, cos_table,
                       sin_table [positions, 64] f32, kv_len [B] int32, slots [B, T] int64,
                       cache_k, cache_v, k_scale, v_scale) -> ()
      gqa::kv_append into the pages: e4m3 rows, a block's scale growing as its rows need.
  gqa::tail_verify_paged(query, gate [B, T, Hq, 256] bf16, q_norm [256] f32, cos_table,
                         sin_table, cache_k, cache_v, k_scale, v_scale, block_table [B, P] int32,
                         kv_len [B] int32, q_len [B] int32) -> out [B, T, Hq, 256] bf16
      gqa::tail_verify over the pages: row (b, t, h) attends positions [0, kv_len[b] + t]; rows
      t >= q_len[b] are 0 (pass granted). T = 1 decodes, a long T is a prompt's chunk.

include/npn_spec_verify.h has the details and limits.
"""
import torch

from npn_native import check_all, launch, query as size_query, register

HEAD_DIM = 256
ROPE_DIM = 64
BLOCK_SIZES = (16, 32, 64, 128)
I32, I64, I8, F32, BF16 = torch.int32, torch.int64, torch.int8, torch.float32, torch.bfloat16


def _cache_sizes(cache_k):
    """(N, Hkv, block size) of a cache's keys."""
    if cache_k.dim() != 4:
        raise RuntimeError(f"cache_k must be [N, Hkv, bs, {HEAD_DIM}], got {tuple(cache_k.shape)}")
    n, hkv, bs, _ = cache_k.shape
    if bs not in BLOCK_SIZES:
        raise RuntimeError(f"block size must be one of {BLOCK_SIZES}, got {bs}")
    return n, hkv, bs


def _dims(t, name, n):
    if t.dim() != n:
        raise RuntimeError(f"{name} must have {n} dimensions, got {tuple(t.shape)}")
    return t.shape


def _update_blocks_fake(kv_len, new_len, block_table, num_blocks, free_blocks, free_count,
                        block_size, T):
    B = block_table.shape[0]
    return kv_len.new_empty((B, T), dtype=I64), kv_len.new_empty((B,))


@register("paged::update_blocks_",
          "(Tensor kv_len, Tensor new_len, Tensor(a!) block_table, Tensor(b!) num_blocks, "
          "Tensor(c!) free_blocks, Tensor(d!) free_count, int block_size, int T) "
          "-> (Tensor, Tensor)", _update_blocks_fake)
def update_blocks_(kv_len, new_len, block_table, num_blocks, free_blocks, free_count, block_size, T):
    if block_size not in BLOCK_SIZES:
        raise RuntimeError(f"block size must be one of {BLOCK_SIZES}, got {block_size}")
    if T < 1:
        raise RuntimeError(f"T must be at least 1, got {T}")
    B, P = _dims(block_table, "block_table", 2)
    n = free_blocks.numel()
    if max(B * T, B * P) > 2 ** 30 or n >= 2 ** 31:
        raise RuntimeError(f"unsupported update_blocks_ sizes B={B} T={T} P={P} N={n}")
    dev = kv_len.device
    check_all(dev, (kv_len, "kv_len", I32, B), (new_len, "new_len", I32, B),
              (block_table, "block_table", I32, (B, P)), (num_blocks, "num_blocks", I32, B),
              (free_blocks, "free_blocks", I32, n), (free_count, "free_count", I32, 1))
    slots = torch.empty((B, T), dtype=I64, device=dev)
    granted = torch.empty(B, dtype=I32, device=dev)
    launch(dev, "npn_paged_update_blocks", kv_len, new_len, block_table, num_blocks, free_blocks,
           free_count, slots, granted, B, P, n, block_size, T)
    return slots, granted


def _kv_append_fake(key, value, k_norm, cos_table, sin_table, kv_len, slots, cache_k, cache_v,
                    k_scale, v_scale):
    return None


@register("gqa::kv_append_paged",
          "(Tensor key, Tensor value, Tensor k_norm, Tensor cos_table, Tensor sin_table, "
          "Tensor kv_len, Tensor slots, Tensor(a!) cache_k, Tensor(b!) cache_v, "
          "Tensor(c!) k_scale, Tensor(d!) v_scale) -> ()", _kv_append_fake)
def kv_append_paged(key, value, k_norm, cos_table, sin_table, kv_len, slots, cache_k, cache_v,
                    k_scale, v_scale):
    n, hkv, bs = _cache_sizes(cache_k)
    B, T = _dims(slots, "slots", 2)
    positions = cos_table.shape[0]
    dev, row, table = key.device, (B, T, hkv, HEAD_DIM), (positions, ROPE_DIM)
    check_all(dev, (key, "key", BF16, row), (value, "value", BF16, row),
              (k_norm, "k_norm", F32, HEAD_DIM), (cos_table, "cos_table", F32, table),
              (sin_table, "sin_table", F32, table), (kv_len, "kv_len", I32, B),
              (slots, "slots", I64, (B, T)), (cache_k, "cache_k", I8, (n, hkv, bs, HEAD_DIM)),
              (cache_v, "cache_v", I8, (n, hkv, HEAD_DIM, bs)), (k_scale, "k_scale", F32, (n, hkv)),
              (v_scale, "v_scale", F32, (n, hkv)))
    launch(dev, "npn_gqa_kv_append_paged", key, value, k_norm, cos_table, sin_table, positions,
           kv_len, slots, cache_k, cache_v, k_scale, v_scale, B, T, hkv, n, bs)


def _tail_verify_fake(query, gate, q_norm, cos_table, sin_table, cache_k, cache_v, k_scale, v_scale,
                      block_table, kv_len, q_len):
    return torch.empty_like(query)


@register("gqa::tail_verify_paged",
          "(Tensor query, Tensor gate, Tensor q_norm, Tensor cos_table, Tensor sin_table, "
          "Tensor cache_k, Tensor cache_v, Tensor k_scale, Tensor v_scale, Tensor block_table, "
          "Tensor kv_len, Tensor q_len) -> Tensor", _tail_verify_fake)
def tail_verify_paged(query, gate, q_norm, cos_table, sin_table, cache_k, cache_v, k_scale, v_scale,
                      block_table, kv_len, q_len):
    n, hkv, bs = _cache_sizes(cache_k)
    B, T, hq, _ = _dims(query, "query", 4)
    P, positions = _dims(block_table, "block_table", 2)[1], cos_table.shape[0]
    dev, row, table = query.device, (B, T, hq, HEAD_DIM), (positions, ROPE_DIM)
    check_all(dev, (query, "query", BF16, row), (gate, "gate", BF16, row),
              (q_norm, "q_norm", F32, HEAD_DIM), (cos_table, "cos_table", F32, table),
              (sin_table, "sin_table", F32, table), (cache_k, "cache_k", I8, (n, hkv, bs, HEAD_DIM)),
              (cache_v, "cache_v", I8, (n, hkv, HEAD_DIM, bs)), (k_scale, "k_scale", F32, (n, hkv)),
              (v_scale, "v_scale", F32, (n, hkv)), (block_table, "block_table", I32, (B, P)),
              (kv_len, "kv_len", I32, B), (q_len, "q_len", I32, B))
    n_ws = size_query("npn_gqa_tail_verify_paged_workspace_size", B, T, hq, hkv, P, bs)
    if n_ws == 0:
        raise RuntimeError(f"unsupported tail_verify_paged sizes B={B} T={T} Hq={hq} Hkv={hkv} "
                           f"P={P} bs={bs}")
    ws = torch.empty(n_ws, dtype=torch.uint8, device=dev)
    out = torch.empty_like(query)
    launch(dev, "npn_gqa_tail_verify_paged", query, gate, q_norm, cos_table, sin_table, positions,
           cache_k, cache_v, k_scale, v_scale, block_table, kv_len, q_len, out, B, T, hq, hkv, n, P,
           bs, ws, n_ws)
    return out
