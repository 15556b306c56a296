"""What rows of one block lose to its scale, in the oracle's append. No GPU."""
import numpy as np
import pytest

from oracle import gqa as og, paged as op, tree as ot


@pytest.mark.parametrize("top", [1, 8, 14, 20])
def test_numbers_are_off_by_their_own_rounding_and_the_largest_one_s(top):
    """Rows of magnitudes up to 2^top apart, appended tree by tree: each value is within 2^-4 of itself and 2^-16 of the
    largest that its block has had. (A number is a multiple of 2^-9 s, or has four bits; s < A / 224. It is
    rounded to 2^-10 s at most once a scale, each at least twice the one before: 2^-17.8 A and as much again.)"""
    rng = np.random.default_rng(top)
    bs, H, rows = 64, 1, 60
    cos, sin = og.rope_cos_sin(np.arange(bs))
    cache = [np.zeros((1, H, bs, 256), np.uint8), np.zeros((1, H, 256, bs), np.uint8), np.zeros((1, H), np.float32),
             np.zeros((1, H), np.float32)]
    value = rng.standard_normal((1, rows, H, 256)) * np.exp2(rng.integers(0, top, (1, rows, H, 1)))
    parent = np.array([[-1, 0, 0, 1]])
    for t in range(0, rows, 4):
        at = slice(t, t + 4)
        ot.kv_append(rng.standard_normal((1, 4, H, 256)), value[:, at], np.zeros(256), cos, sin, np.array([t]),
                     np.arange(t, t + 4)[None], parent, cache)
        _, v, _ = op.values(cache, [0], 0, t + 4)
        want = value[0, :t + 4, 0]
        assert (np.abs(v - want) <= np.abs(want) * 2.0 ** -4 + np.abs(want).max() * 2.0 ** -16).all()
