"""Sampling of plain decode's tokens on gfx950 (new op; the reference's on-device path is an argmax,
contrib/qwen3.6-27b/static_decode.py:1313).

  spec::sample(logits [R, V] f32 or bf16, temperature [R] f32, top_k [R] int32, top_p [R] f32,
               min_p [R] f32, u [R] f32) -> ids [R] int64
      One token per row with the row's own settings: tokens ranked by logit (ties: lower index
      first) and weighed by exp((l - max) / temperature), cut to the first top_k, then to the
      top_p share of those, then to weights >= min_p, and sampled by inversion with the given
      uniform u. temperature <= 0 takes the first rank; top_k <= 0, top_p >= 1 and min_p <= 0 are
      off. -1 where a row has no token above -infinity.

include/npn_spec_verify.h has the details. Sums are exact integers: the same inputs give the same
ids in every run and whatever else shares the batch.
"""
import torch

from npn_native import call, require, stream_of


@torch.library.custom_op("spec::sample", mutates_args=(), device_types="cuda")
def sample(
    logits: torch.Tensor,       # [R, V] f32 or bf16
    temperature: torch.Tensor,  # [R] f32
    top_k: torch.Tensor,        # [R] int32
    top_p: torch.Tensor,        # [R] f32
    min_p: torch.Tensor,        # [R] f32
    u: torch.Tensor,            # [R] f32
) -> torch.Tensor:
    R, V = logits.shape
    bf16 = logits.dtype == torch.bfloat16
    require(logits, "logits", torch.bfloat16 if bf16 else torch.float32)
    require(temperature, "temperature", torch.float32, numel=R)
    require(top_k, "top_k", torch.int32, numel=R)
    require(top_p, "top_p", torch.float32, numel=R)
    require(min_p, "min_p", torch.float32, numel=R)
    require(u, "u", torch.float32, numel=R)
    ids = torch.empty(R, dtype=torch.int64, device=logits.device)
    with torch.cuda.device(logits.device):
        call("npn_sample", logits, int(bf16), temperature, top_k, top_p, min_p, u, ids, R, V,
             stream_of(logits))
    return ids


@sample.register_fake
def _(logits, temperature, top_k, top_p, min_p, u):
    return logits.new_empty((logits.shape[0],), dtype=torch.int64)
