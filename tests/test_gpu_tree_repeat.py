"""The tree-verification ops give the same bits in every call, whatever their outputs' and workspaces' memory held."""
import numpy as np
import pytest
import torch

from test_gpu_tree import _args, _attend_inputs, _dn, _verify, cuda, some_paths, trees

pytestmark = pytest.mark.gpu


def _poison(byte):
    """Freed memory for the next call's outputs and workspaces, every byte set."""
    for size in (1 << 9, 1 << 12, 1 << 16, 1 << 20, 1 << 21, 1 << 23, 1 << 25, 1 << 27):
        held = [torch.full((size,), byte, dtype=torch.uint8, device="cuda") for _ in range(6)]
        del held


def _repeats(call, make):
    """call(make()) with memory that held zeros, ones and NaN: the same outputs and, of what it writes, the same."""
    first = None
    for byte in (0x00, 0xFF, 0x7F, 0x01):
        args = make()
        torch.cuda.synchronize()
        _poison(byte)
        out = call(args)
        torch.cuda.synchronize()
        out = [t.clone() for t in out]
        if first is None:
            first = out
        # bits: NaN is as good as another number
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(out, first)), byte


@pytest.mark.parametrize("B,T,H,grp,bs,kv,n", [
    (1, 1, 1, 1, 16, [0], [1]), (2, 2, 4, 6, 16, [63, 3000], [2, 2]), (2, 5, 2, 6, 32, [5000, 0], [5, 4]),
    (4, 8, 4, 6, 64, [37, 600, 9000, 5], [8, 0, 8, 3]), (1, 16, 4, 6, 64, [16000], [16]), (3, 10, 2, 6, 16, [900, 0, 61], [10, 9, 0]),
    (2, 64, 4, 6, 64, [4000, 130], [64, 20]), (9, 20, 4, 6, 16, [0, 5, 100, 300, 700, 1100, 64, 128, 33], [20, 19, 1, 20, 17, 20, 0, 20, 2]),
])
def test_attention(ops, B, T, H, grp, bs, kv, n):
    d = _attend_inputs(B, T, H, grp, bs, kv, n, 4, seed=T)
    _repeats(lambda a: [ops.gqa.tree_verify_paged(*a), *a[8:12]], lambda: _args(d))


@pytest.mark.parametrize("B,T,Hv", [(1, 1, 3), (2, 16, 6), (20, 16, 15), (2, 31, 3), (3, 40, 3), (20, 48, 15), (2, 64, 3), (20, 50, 15)])
def test_deltanet(ops, B, T, Hv):
    _, f = _dn(B, T, 3, Hv, seed=T)
    parent = trees(B, T, 4, seed=T)
    path = cuda(some_paths(parent, 0))

    def call(f):
        out, rec = _verify(ops, f, cuda(parent))
        ops.deltanet.commit_tree_([f["state"]], [f["conv_state"]], [f["mixed_qkv"]], [rec], path, Hv)
        return [out, rec, f["state"], f["conv_state"]]
    _repeats(call, lambda: {k: v.clone() for k, v in f.items()})


def test_walk(ops):
    rng = np.random.default_rng(0)
    draft, target = rng.integers(0, 2, (2, 50, 33))
    args = [cuda(target), cuda(draft), cuda(trees(50, 33, 4, 0)), cuda(rng.integers(0, 34, 50).astype(np.int32))]
    _repeats(lambda a: ops.spec.accept_tree(*a), lambda: [a.clone() for a in args])
