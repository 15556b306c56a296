"""The tree-verification oracle (oracle/tree.py) against what it must agree with: chains are what the
verify oracles take, a node of a tree is the last of the chain of its ancestors, committing a path is
running its chain, compacting is appending the path's rows alone. No GPU."""
import numpy as np
import pytest

from oracle import deltanet as od, gqa as og, paged as op, tree as ot
from _util import deltanet_inputs, deltanet_oracle_args

PARENT = np.array([[-1, 0, 0, 1, 1, 2, 5, 4, 4], [-1, 0, 1, 2, 3, 4, 5, 6, 7]])


def _dn(B, T, Hk=1, Hv=2, seed=0):
    return deltanet_oracle_args(deltanet_inputs(B, T, Hk, Hv, seed=seed))


def _along(d, b, nodes):
    """The arguments of request b's chain of `nodes`."""
    state, mixed, conv, w, bias, a, b_, z, A_log, dt_bias, nw = d
    at = np.ix_([b], nodes)
    return (state[b:b + 1], mixed[at], conv[b:b + 1], w, bias, a[at], b_[at], z[at], A_log, dt_bias, nw)


def test_lines():
    assert ot.line(PARENT[0], 7) == [0, 1, 4, 7] and ot.line(PARENT[0], 0) == [0]
    assert ot.depths(PARENT).tolist() == [[0, 1, 1, 2, 2, 2, 3, 3, 3], list(range(9))]
    # a parent that is none, itself or later: the committed tokens alone
    assert [ot.line([3, 1, 9, -7], t) for t in range(4)] == [[0], [1], [2], [3]]


def test_deltanet_nodes_are_the_ends_of_their_chains():
    d = _dn(2, 9)
    out, k, u, decay, states = ot.deltanet_verify(d, PARENT, 1, 2)
    for b in range(2):
        for t in range(9):
            ck, o = od.deltanet_verify(*_along(d, b, ot.line(PARENT[b], t)), 1, 2)
            np.testing.assert_allclose(o[0, -1], out[b, t], rtol=1e-10)
            np.testing.assert_allclose(ck[0, -1], states[b, t], rtol=1e-10, atol=1e-14)


def test_deltanet_commit_is_the_path_s_state():
    d = _dn(2, 9, seed=1)
    out, k, u, decay, states = ot.deltanet_verify(d, PARENT, 1, 2)
    path = np.full((2, 9), -1, np.int32)
    path[0, :4], path[1, :2] = [0, 1, 4, 7], [0, 1]
    state, conv = ot.deltanet_commit(d[0], d[2], d[1], k, u, decay, path)
    np.testing.assert_allclose(state[0], states[0, 7], rtol=1e-10, atol=1e-14)
    np.testing.assert_allclose(state[1], states[1, 1], rtol=1e-10, atol=1e-14)
    for b, nodes in ((0, [0, 1, 4, 7]), (1, [0, 1])):
        assert np.array_equal(conv[b:b + 1], od.conv_state_after(d[2][b:b + 1], d[1][b:b + 1, nodes], [len(nodes) - 1]))
    same = ot.deltanet_commit(d[0], d[2], d[1], k, u, decay, np.full((2, 9), -1))
    assert np.array_equal(same[0], d[0].astype(np.float64)) and np.array_equal(same[1], d[2])


def test_a_planted_mistake_in_the_tree_shows():
    d = _dn(1, 9)
    wrong = PARENT[:1].copy()
    wrong[0, 4] = 0
    a, b = ot.deltanet_verify(d, PARENT[:1], 1, 2)[0], ot.deltanet_verify(d, wrong, 1, 2)[0]
    diff = np.abs(a - b).max((0, 2, 3)) > 1e-6
    assert diff.tolist() == [False] * 4 + [True] + [False] * 2 + [True] * 2


def _cache(N, H, bs, rng):
    return [rng.integers(0, 0x78, (N, H, bs, 256)).astype(np.uint8), rng.integers(0, 0x78, (N, H, 256, bs)).astype(np.uint8),
            np.exp2(rng.integers(-9, -3, (N, H))).astype(np.float32), np.exp2(rng.integers(-9, -3, (N, H))).astype(np.float32)]


def _attention(rng, parent, kv=21, bs=16, H=1, grp=2):
    B, T = parent.shape
    P = -(-(kv + T) // bs)
    table = rng.permutation(B * P).reshape(B, P).astype(np.int32)
    pos = kv + np.arange(T)
    slots = table[:, pos // bs].astype(np.int64) * bs + pos % bs
    r = lambda *s: rng.standard_normal(s)  # noqa: E731
    cos, sin = og.rope_cos_sin(np.arange(kv + T))
    return dict(cache=_cache(B * P, H, bs, rng), table=table, slots=slots, kv=np.full(B, kv), n=np.full(B, T), cos=cos,
                sin=sin, q=r(B, T, H * grp, 256), gate=r(B, T, H * grp, 256), key=r(B, T, H, 256), value=r(B, T, H, 256),
                qn=r(256) * 0.1, kn=r(256) * 0.1)


def _verify(d, parent, cache):
    ot.kv_append(d["key"], d["value"], d["kn"], d["cos"], d["sin"], d["kv"], d["slots"], parent, cache)
    return ot.tree_verify(d["q"], d["gate"], d["qn"], d["cos"], d["sin"], cache, d["table"], d["kv"], d["n"], parent)


def test_attention_of_a_chain_is_the_paged_verify():
    chain = PARENT[1:]
    d = _attention(np.random.default_rng(0), chain)
    cache = [c.copy() for c in d["cache"]]
    got = _verify(d, chain, cache)
    op.kv_append(d["key"], d["value"], d["kn"], d["cos"], d["sin"], d["kv"], d["slots"], d["cache"])
    for a, b in zip(cache, d["cache"]):
        assert np.array_equal(a, b)
    want = op.tail_verify(d["q"], d["gate"], d["qn"], d["cos"], d["sin"], d["cache"], d["table"], d["kv"], d["n"])
    np.testing.assert_allclose(got, want, rtol=1e-12, atol=1e-14)


def test_attention_of_a_node_sees_its_line():
    """A node's row is that of a chain of its ancestors whose rows are copied into one place after the other."""
    d = _attention(np.random.default_rng(1), PARENT[:1])
    cache = [c.copy() for c in d["cache"]]
    got = _verify(d, PARENT[:1], cache)
    nodes = [0, 1, 4, 8]
    ot.compact(np.array([nodes + [-1] * 5]), d["slots"], cache)
    # positions 21 to 29 lie in one page, so the bytes move as they are
    sub = dict(d, q=d["q"][:, nodes], gate=d["gate"][:, nodes])
    want = op.tail_verify(sub["q"], sub["gate"], d["qn"], d["cos"], d["sin"], cache, d["table"], d["kv"], np.array([4]))
    np.testing.assert_allclose(got[0, 8], want[0, 3], rtol=1e-12, atol=1e-14)


def test_accept():
    parent = np.array([[-1, 0, 0, 1, 2, 2]] * 5)
    draft = np.array([[9, 5, 6, 7, 8, 8]] * 5)
    target = np.array([[6, 0, 8, 0, 3, 4],   # 0 -> 2 -> 4 (the first of two alike)
                       [1, 0, 0, 0, 0, 0],   # none
                       [5, 7, 0, 2, 0, 0],   # 0 -> 1 -> 3, a leaf
                       [6, 0, 8, 0, 3, 4],   # node 4 is none
                       [6, 0, 8, 0, 3, 4]])  # no node at all
    accepted, path, ids = ot.accept(target, draft, parent, np.array([6, 6, 6, 4, 0]))
    assert accepted.tolist() == [2, 0, 2, 1, -1]
    assert path.tolist() == [[0, 2, 4, -1, -1, -1], [0] + [-1] * 5, [0, 1, 3, -1, -1, -1], [0, 2] + [-1] * 4, [-1] * 6]
    assert ids.tolist() == [[6, 8, 3, -1, -1, -1], [1] + [-1] * 5, [5, 7, 2, -1, -1, -1], [6, 8] + [-1] * 4, [-1] * 6]


@pytest.mark.parametrize("off", [0, 11, 15])
def test_compact_moves_values(off):
    """Every row of the path is where it belongs, to the rounding of its new page's scale."""
    rng = np.random.default_rng(off)
    N, H, bs, T = 4, 2, 16, 20
    cache = _cache(N, H, bs, rng)
    order = rng.permutation(N)
    at = off + np.arange(T)
    slots = (order[at // bs] * bs + at % bs)[None]
    before = [c.copy() for c in cache]
    nodes = [0, 3, 4, 9, 17, 19]
    ot.compact(np.array([nodes + [-1] * (T - len(nodes))]), slots, cache)

    def rows(c, s):
        k, v, _ = op.values(c, [s // bs], 0, bs)
        return k[s % bs], v[s % bs]
    for d, node in enumerate(nodes):
        for name, got, want in zip("kv", rows(cache, int(slots[0, d])), rows(before, int(slots[0, node]))):
            scale = cache[2 if name == "k" else 3][slots[0, d] // bs, 0]
            assert (np.abs(got - want) <= np.maximum(np.abs(want) * 2.0 ** -4, scale * 2.0 ** -10)).all()
    for a, b in zip(cache[2:], before[2:]):
        assert (a >= b).all()
    # a path that is a prefix moves nothing
    again = [c.copy() for c in cache]
    ot.compact(np.array([[0, 1, 2] + [-1] * (T - 3)]), slots, again)
    assert all(np.array_equal(a, b) for a, b in zip(again, cache))
