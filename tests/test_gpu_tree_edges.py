"""The tree-verification ops at the edges of what they allow, against oracle/tree.py."""
import numpy as np
import pytest

from oracle import fp8, tree as ot
from test_gpu_tree import _compact, _pages

pytestmark = pytest.mark.gpu


def _same_pages(got, want):
    """Scales equal, bytes of the same values."""
    assert np.array_equal(got[2], want[2]) and np.array_equal(got[3], want[3])
    for a, b in zip(got[:2], want[:2]):
        assert np.array_equal(fp8.decode_e4m3fn(a), fp8.decode_e4m3fn(b), equal_nan=True)


@pytest.mark.parametrize("scale", [2.0 ** 27, 2.0 ** 28, 2.0 ** 30, 2.0 ** 119])
def test_compact_paged_zero_rows_between_scales_far_apart(ops, scale):
    """A row of zeros (and one of zeros and NaN) that moves from a page of a large scale to one of the least, whose
    ratio passes fp32, keeps its zeros; a row that is not zero takes its new page's scale up."""
    rng = np.random.default_rng(0)
    bs, T, H = 16, 20, 2
    cache = _pages(1, 2, H, bs, rng, 1)
    for c in cache:
        for k in (2, 3):
            c[k][0], c[k][1] = 2.0 ** -100, scale
        for k, rows in ((0, c[0][1]), (1, c[1][1].transpose(0, 2, 1))):  # slots 16, 17
            rows[:, :2] = rng.choice([0x00, 0x80], (H, 2, 256))
            rows[:, 1, ::7] = 0x7F
            rows[1, 0, 5] = 0x38  # head 1: a one
    slots = np.arange(T)[None].astype(np.int64)
    path = np.full((1, T), -1, np.int32)
    path[0, :3] = [0, 16, 17]
    got = _compact(ops, cache, path, slots)
    ot.compact(path, slots, cache[0])
    assert cache[0][2][0, 0] == 2.0 ** -100 and cache[0][2][0, 1] > 2.0 ** -100
    _same_pages(got[0], cache[0])


def test_compact_paged_scales_of_zero(ops):
    """Rows that move between pages whose scale is 0 (nothing was ever appended to them) keep their bytes."""
    rng = np.random.default_rng(1)
    cache = _pages(1, 2, 1, 16, rng, 1)
    cache[0][2][:], cache[0][3][:] = 0.0, 0.0
    slots = np.arange(20)[None].astype(np.int64)
    path = np.full((1, 20), -1, np.int32)
    path[0, :4] = [0, 5, 16, 17]
    got = _compact(ops, cache, path, slots)
    ot.compact(path, slots, cache[0])
    _same_pages(got[0], cache[0])


@pytest.mark.parametrize("bs,kind", [(64, "pieces"), (128, "pieces"), (64, "rows"), (16, "blocks"), (128, "jump"), (32, "none")])
def test_compact_paged_slots_out_of_order(ops, bs, kind):
    """Slots that no block table makes: rows move up to the first that is not behind the last one, and no other page
    or row changes. (none: a block that is none in the middle, which a table may have; the path goes past it.)"""
    T, H, B = 64, 2, 3
    rng = np.random.default_rng(bs)
    N = B * 5 + 2
    cache, ids = _pages(1, N, H, bs, rng, 9), rng.permutation(N)[:B * 5].reshape(B, 5)
    at = np.array([0, 5, bs - 3])[:, None] + np.arange(T)
    slots = np.take_along_axis(ids, at // bs, 1) * bs + at % bs
    for b in range(B):
        if kind == "pieces":    # two of a block's pieces of 16 have changed places
            x, y = slots[b, :16].copy(), slots[b, 16:32].copy()
            slots[b, :16], slots[b, 16:32] = y, x
        elif kind == "rows":
            slots[b, 20], slots[b, 21] = slots[b, 21], slots[b, 20]
        elif kind == "blocks":  # begins a block where the last one has not ended
            slots[b, 30:] += 3
        elif kind == "jump" and b == 0:  # in order in each 16, far behind in the block
            slots[b, 16:32] = slots[b, 0] + 112 + np.arange(16)
        elif kind == "none":
            hole = (at[b] // bs) == at[b, 0] // bs + 1
            slots[b, hole] = -bs + at[b, hole] % bs
    path = np.full((B, T), -1, np.int32)
    for b in range(B):
        nodes = np.sort(rng.choice(np.arange(1, T), 12, replace=False))
        path[b, :13] = np.concatenate([[0], nodes])
    if kind == "none":
        path[:, :6] = [0, 2, 8, 50, 60, 63]
        path[:, 6:] = -1
    want = cache[0]
    got = _compact(ops, cache, path, slots.astype(np.int64))
    ot.compact(path, slots, want)
    _same_pages(got[0], want)
