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
