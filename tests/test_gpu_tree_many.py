"""gqa::tree_verify_paged against the oracle where trees are many, as in a serving batch: each launch that is chosen by
how many rows, heads and requests there are. Tolerances as in test_gpu_tree.py."""
import numpy as np
import pytest
import torch

from oracle import tree as ot
from _util import BF16_U, assert_rel_close
from test_gpu_tree import _args, _attend_inputs, _check

pytestmark = pytest.mark.gpu


def _lengths(B, T, longest, seed):
    """Committed rows and nodes of each request: none, few and, of the first, many; some sit out, some have fewer than T
    nodes."""
    rng = np.random.default_rng(seed)
    kv, n = rng.integers(0, longest + 1, B), np.where(rng.random(B) < 0.5, T, rng.integers(0, T + 1, B))
    kv[rng.random(B) < 0.2] = 0
    kv[0], n[1] = 6 * longest, 0
    return kv, n


@pytest.mark.parametrize("B,T,H,grp,bs,longest", [
    (70, 2, 4, 6, 16, 90),      # 280 pairs of 16 rows: a workgroup each and more; four rows of q' a wave
    (44, 5, 4, 6, 32, 150),     # 176 of 32
    (32, 8, 4, 6, 16, 200),     # 128 of 48
    (45, 8, 4, 6, 128, 90),     # 180 of 48
    (24, 10, 4, 6, 16, 100),    # two groups of 32 each, 192 pairs
    (12, 16, 2, 6, 64, 200),    # groups of 128, a quarter of them idle, 24 pairs
    (24, 16, 4, 6, 16, 120),    # 96 pairs of 128: a second round of workgroups may pay
    (16, 32, 4, 6, 32, 150),    # two groups of 128 each, appends of 32 rows
    (12, 30, 4, 6, 64, 300),
    (9, 64, 4, 6, 64, 200),     # three groups each, appends of 64 rows
    (8, 64, 4, 6, 128, 300),
    (30, 13, 4, 8, 128, 60),    # 104 rows, 120 pairs
])
def test_many_trees(ops, B, T, H, grp, bs, longest):
    kv, n = _lengths(B, T, longest, seed=B + T)
    _check(ops, _attend_inputs(B, T, H, grp, bs, kv, n, 4, seed=B * T))


@pytest.mark.parametrize("B,T,bs", [(96, 16, 64), (65, 22, 128), (96, 8, 64)])
def test_many_trees_over_long_contexts(ops, B, T, bs):
    """As many pairs of groups of 128 as are cut for a second round of workgroups where their keys are many enough
    (and of 48 rows, cut but for one round): some requests against the oracle, some against calls of their own, which
    are cut otherwise: both within the tolerance of the formula, so within twice that of each other. The requests share
    the pages of their first 12800 rows."""
    long = 12800
    kv, n = _lengths(B, T, 70, seed=B)
    n[n == 0] = 1
    d = _attend_inputs(B, T, 1, 6, bs, kv, n, 4, seed=B)
    more = _attend_inputs(1, 1, 1, 6, bs, [long - 1], [1], 1, seed=B + 1, spare=0)
    N = len(d["cache"][0])
    d["cache"] = [np.concatenate(x) for x in zip(d["cache"], more["cache"])]
    d["table"] = np.concatenate([np.repeat(more["table"] + N, B, 0), d["table"]], 1).astype(np.int32)
    d["kv"] = (d["kv"] + long).astype(np.int32)
    cos, sin = (np.concatenate([np.zeros((long, 64), np.float32), x]) for x in (d["cos"], d["sin"]))
    d["cos"], d["sin"] = cos, sin  # (the rows of the nodes' positions are all that count)
    args = _args(d)
    got = ops.gqa.tree_verify_paged(*args)
    torch.cuda.synchronize()
    cache = [a.cpu().numpy() for a in args[8:12]]
    cache[0], cache[1] = cache[0].view(np.uint8), cache[1].view(np.uint8)
    f = lambda k, b: d[k][b:b + 1].double().numpy()  # noqa: E731
    qn = d["q_norm"].double().numpy()
    for b in (0, 1, B // 2, B - 1):
        ref = ot.tree_verify(f("query", b), f("gate", b), qn, d["cos"], d["sin"], cache, d["table"][b:b + 1], d["kv"][b:b + 1],
                             d["n"][b:b + 1], d["parent"][b:b + 1])
        assert_rel_close(got[b:b + 1].float().cpu().numpy(), ref, tol=2e-3, out_unit=BF16_U, name=f"request {b}")
    fresh = _args(d)
    for b in range(2, B, B // 8):
        own = [a[b:b + 1].contiguous() if i in (0, 1, 2, 3, 12, 13, 14, 15, 16) else a for i, a in enumerate(fresh)]
        one = ops.gqa.tree_verify_paged(*own)
        assert_rel_close(got[b:b + 1].float().cpu().numpy(), one.float().cpu().double().numpy(), tol=4e-3, out_unit=2 * BF16_U)
