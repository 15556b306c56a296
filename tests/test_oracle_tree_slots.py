"""The rule of oracle/tree.py's compaction about slots out of order. No GPU."""
import numpy as np
import pytest

from oracle import tree as ot


@pytest.mark.parametrize("bs", [16, 32, 128])
def test_rows_in_place_of_a_table(bs):
    """Slots as a block table makes them are in place throughout, over blocks that are none (id -1) too."""
    rng = np.random.default_rng(bs)
    for off in (0, 1, bs - 1):
        ids = rng.permutation(12)
        ids[3] = -1
        at = off + np.arange(64)
        slots = ids[at // bs] * bs + at % bs
        assert ot.rows_in_place(slots, bs) == 64
        for n in (1, 7, 40):
            assert ot.rows_in_place(np.where(np.arange(64) < n, slots, -1), bs) == n or slots[n - 1] == -2
        for t in (1, 9, 63):
            wrong = slots.copy()
            wrong[t] += bs if (off + t) % bs else 1
            assert ot.rows_in_place(wrong, bs) == t


def test_compact_ends_before_a_row_out_of_place():
    """Rows 16 .. 31 of the tree in another part of their block than the first 16: each 16 are in order in themselves."""
    rng = np.random.default_rng(0)
    bs, T = 128, 32
    cache = [rng.integers(0, 0x78, (2, 1, bs, 256)).astype(np.uint8), rng.integers(0, 0x78, (2, 1, 256, bs)).astype(np.uint8),
             np.ones((2, 1), np.float32), np.ones((2, 1), np.float32)]
    slots = np.where(np.arange(T) < 16, np.arange(T), 96 + np.arange(T))[None]
    path = np.full((1, T), -1, np.int32)
    path[0, :4] = [0, 5, 15, 16]
    before = [c.copy() for c in cache]
    ot.compact(path, slots, cache)
    k = cache[0][0, 0]
    assert np.array_equal(k[1], before[0][0, 0, 5]) and np.array_equal(k[2], before[0][0, 0, 15])
    assert np.array_equal(k[3:], before[0][0, 0, 3:])
