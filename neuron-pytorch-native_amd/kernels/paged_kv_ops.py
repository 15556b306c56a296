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

from npn_native import call, query as size_query, require, stream_of

HEAD_DIM = 256
ROPE_DIM = 64
BLOCK_SIZES = (16, 32, 64, 128)


def _require_cache(cache_k, cache_v, k_scale, v_scale):
    """Checks the four cache tensors; returns (N, Hkv, block size)."""
    if cache_k.dim() != 4:
        raise RuntimeError(f"cache_k must be [N, Hkv, bs, {HEAD_DIM}], got {tuple(cache_k.shape)}")
    n, hkv, bs, _ = cache_k.shape
    if bs not in BLOCK_SIZES:
        raise RuntimeError(f"block size must be one of {BLOCK_SIZES}, got {bs}")
    require(cache_k, "cache_k", torch.int8, shape=(n, hkv, bs, HEAD_DIM))
    require(cache_v, "cache_v", torch.int8, shape=(n, hkv, HEAD_DIM, bs))
    require(k_scale, "k_scale", torch.float32, shape=(n, hkv))
    require(v_scale, "v_scale", torch.float32, shape=(n, hkv))
    return n, hkv, bs


@torch.library.custom_op("paged::update_blocks_", device_types="cuda",
                         mutates_args=("block_table", "num_blocks", "free_blocks", "free_count"))
def update_blocks_(
    kv_len: torch.Tensor,       # [B] int32
    new_len: torch.Tensor,      # [B] int32
    block_table: torch.Tensor,  # [B, P] int32 (in place)
    num_blocks: torch.Tensor,   # [B] int32 (in place)
    free_blocks: torch.Tensor,  # [N] int32 (in place)
    free_count: torch.Tensor,   # [1] int32 (in place)
    block_size: int,
    T: int,
) -> tuple[torch.Tensor, torch.Tensor]:
    if block_size not in BLOCK_SIZES:
        raise RuntimeError(f"block size must be one of {BLOCK_SIZES}, got {block_size}")
    if T < 1:
        raise RuntimeError(f"T must be at least 1, got {T}")
    B, P = block_table.shape
    n = free_blocks.numel()
    require(kv_len, "kv_len", torch.int32, numel=B)
    require(new_len, "new_len", torch.int32, numel=B)
    require(block_table, "block_table", torch.int32)
    require(num_blocks, "num_blocks", torch.int32, numel=B)
    require(free_blocks, "free_blocks", torch.int32)
    require(free_count, "free_count", torch.int32, numel=1)
    slots = torch.empty((B, T), dtype=torch.int64, device=kv_len.device)
    granted = torch.empty(B, dtype=torch.int32, device=kv_len.device)
    with torch.cuda.device(kv_len.device):
        call("npn_paged_update_blocks", kv_len, new_len, block_table, num_blocks, free_blocks,
             free_count, slots, granted, B, P, n, block_size, T, stream_of(kv_len))
    return slots, granted


@update_blocks_.register_fake
def _(kv_len, new_len, block_table, num_blocks, free_blocks, free_count, block_size, T):
    B = block_table.shape[0]
    return (kv_len.new_empty((B, T), dtype=torch.int64), kv_len.new_empty((B,)))


@torch.library.custom_op("gqa::kv_append_paged", device_types="cuda",
                         mutates_args=("cache_k", "cache_v", "k_scale", "v_scale"))
def kv_append_paged(
    key: torch.Tensor,        # [B, T, Hkv, 256] bf16 (k projection, pre-norm)
    value: torch.Tensor,      # [B, T, Hkv, 256] bf16
    k_norm: torch.Tensor,     # [256] f32
    cos_table: torch.Tensor,  # [positions, 64] f32
    sin_table: torch.Tensor,  # [positions, 64] f32
    kv_len: torch.Tensor,     # [B] int32
    slots: torch.Tensor,      # [B, T] int64
    cache_k: torch.Tensor,    # [N, Hkv, bs, 256] int8 (in place)
    cache_v: torch.Tensor,    # [N, Hkv, 256, bs] int8 (in place)
    k_scale: torch.Tensor,    # [N, Hkv] f32 (in place)
    v_scale: torch.Tensor,    # [N, Hkv] f32 (in place)
) -> None:
    n, hkv, bs = _require_cache(cache_k, cache_v, k_scale, v_scale)
    B, T = slots.shape
    positions = cos_table.shape[0]
    require(key, "key", torch.bfloat16, shape=(B, T, hkv, HEAD_DIM))
    require(value, "value", torch.bfloat16, shape=(B, T, hkv, HEAD_DIM))
    require(k_norm, "k_norm", torch.float32, numel=HEAD_DIM)
    require(cos_table, "cos_table", torch.float32, shape=(positions, ROPE_DIM))
    require(sin_table, "sin_table", torch.float32, shape=(positions, ROPE_DIM))
    require(kv_len, "kv_len", torch.int32, numel=B)
    require(slots, "slots", torch.int64)
    with torch.cuda.device(key.device):
        call("npn_gqa_kv_append_paged", key, value, k_norm, cos_table, sin_table, positions,
             kv_len, slots, cache_k, cache_v, k_scale, v_scale, B, T, hkv, n, bs, stream_of(key))


@kv_append_paged.register_fake
def _(key, value, k_norm, cos_table, sin_table, kv_len, slots, cache_k, cache_v, k_scale, v_scale):
    return None


@torch.library.custom_op("gqa::tail_verify_paged", mutates_args=(), device_types="cuda")
def tail_verify_paged(
    query: torch.Tensor,        # [B, T, Hq, 256] bf16
    gate: torch.Tensor,         # [B, T, Hq, 256] bf16
    q_norm: torch.Tensor,       # [256] f32
    cos_table: torch.Tensor,    # [positions, 64] f32
    sin_table: torch.Tensor,    # [positions, 64] f32
    cache_k: torch.Tensor,      # [N, Hkv, bs, 256] int8
    cache_v: torch.Tensor,      # [N, Hkv, 256, bs] int8
    k_scale: torch.Tensor,      # [N, Hkv] f32
    v_scale: torch.Tensor,      # [N, Hkv] f32
    block_table: torch.Tensor,  # [B, P] int32
    kv_len: torch.Tensor,       # [B] int32
    q_len: torch.Tensor,        # [B] int32
) -> torch.Tensor:
    n, hkv, bs = _require_cache(cache_k, cache_v, k_scale, v_scale)
    B, T, hq, dh = query.shape
    if dh != HEAD_DIM:
        raise RuntimeError(f"head dim must be {HEAD_DIM}")
    P, positions = block_table.shape[-1], cos_table.shape[0]
    require(query, "query", torch.bfloat16)
    require(gate, "gate", torch.bfloat16, shape=query.shape)
    require(q_norm, "q_norm", torch.float32, numel=HEAD_DIM)
    require(cos_table, "cos_table", torch.float32, shape=(positions, ROPE_DIM))
    require(sin_table, "sin_table", torch.float32, shape=(positions, ROPE_DIM))
    require(block_table, "block_table", torch.int32, shape=(B, P))
    require(kv_len, "kv_len", torch.int32, numel=B)
    require(q_len, "q_len", torch.int32, numel=B)
    n_ws = size_query("npn_gqa_tail_verify_paged_workspace_size", B, T, hq, hkv, P, bs)
    if n_ws == 0:
        raise RuntimeError(f"unsupported tail_verify_paged sizes B={B} T={T} Hq={hq} Hkv={hkv} "
                           f"P={P} bs={bs}")
    ws = torch.empty(n_ws, dtype=torch.uint8, device=query.device)
    out = torch.empty_like(query)
    with torch.cuda.device(query.device):
        call("npn_gqa_tail_verify_paged", query, gate, q_norm, cos_table, sin_table, positions,
             cache_k, cache_v, k_scale, v_scale, block_table, kv_len, q_len, out, B, T, hq, hkv, n,
             P, bs, ws, n_ws, stream_of(query))
    return out


@tail_verify_paged.register_fake
def _(query, gate, q_norm, cos_table, sin_table, cache_k, cache_v, k_scale, v_scale, block_table,
      kv_len, q_len):
    return torch.empty_like(query)
