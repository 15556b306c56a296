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

from npn_native import check_all, launch, query as size_query, register

I32, F32 = torch.int32, torch.float32


def _sample_fake(logits, temperature, top_k, top_p, min_p, u):
    return logits.new_empty((logits.shape[0],), dtype=torch.int64)


@register("spec::sample",
          "(Tensor logits, Tensor temperature, Tensor top_k, Tensor top_p, Tensor min_p, Tensor u) "
          "-> Tensor", _sample_fake)
def sample(logits, temperature, top_k, top_p, min_p, u):
    if logits.dim() != 2:
        raise RuntimeError(f"logits must be [R, V], got {tuple(logits.shape)}")
    R, V = logits.shape
    bf16 = logits.dtype == torch.bfloat16
    dev = logits.device
    check_all(dev, (logits, "logits", torch.bfloat16 if bf16 else F32, (R, V)),
              (temperature, "temperature", F32, R), (top_k, "top_k", I32, R),
              (top_p, "top_p", F32, R), (min_p, "min_p", F32, R), (u, "u", F32, R))
    ids = torch.empty(R, dtype=torch.int64, device=dev)
    n_ws = size_query("npn_sample_workspace_size", R, V)
    if n_ws == 0:
        raise RuntimeError(f"unsupported sample sizes R={R} V={V}")
    ws = torch.empty(n_ws, dtype=torch.uint8, device=dev)
    launch(dev, "npn_sample", logits, int(bf16), temperature, top_k, top_p, min_p, u, ids, R, V, ws,
           n_ws)
    return ids
