"""GPU parity of the tree-verification ops against the oracle (oracle/tree.py), and with the chain ops
where the tree is a chain.

Tolerances. Attention: as in test_gpu_paged.py, whose kernels these are (2e-3 in the norm, BF16_U of an element's
own). DeltaNet records and states are sums in fp32 of at most 128 products and 64 nodes' terms: 192 roundings of
2^-24, 1.1e-5 of their terms' magnitude if all fall one way; 2e-5 with the exponentials' and roots' few ulps.
Its out has that and the output's own rounding to bf16, at most 2^-8 of each element and so of the norm. Walks,
windows, pages: equal."""
import numpy as np
import pytest
import torch

from oracle import fp8, gqa as og, paged as op, tree as ot
from _util import BF16_U, assert_rel_close, bits, deltanet_flat_device, deltanet_inputs, deltanet_oracle_args

pytestmark = pytest.mark.gpu
F32_TOL = 2e-5
BF, I32 = torch.bfloat16, torch.int32


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def out_close(out, ref):
    got = out.float().cpu().double().numpy().reshape(ref.shape)
    assert np.isfinite(got).all()
    assert (np.abs(got - ref) <= F32_TOL * np.abs(ref).max() + BF16_U * np.abs(ref)).all()
    assert np.linalg.norm(got - ref) <= (F32_TOL + BF16_U) * np.linalg.norm(ref)


def trees(B, T, reach, seed, wild=False):
    """parent [B, T]: among the `reach` nodes before (1: chains). wild: some that are none, itself or later."""
    rng = np.random.default_rng(seed)
    t = np.arange(T)
    parent = np.maximum(t - 1 - rng.integers(0, reach, (B, T)), 0)
    parent[:, 0] = -1
    if wild:
        odd = rng.random((B, T)) < 0.15
        parent = np.where(odd, rng.choice([-1, -2**31, 2**31 - 1, 64, 63], (B, T)), parent)
        own = rng.random((B, T)) < 0.05
        parent = np.where(own, t, parent)
    return parent.astype(np.int32)


def some_paths(parent, seed):
    """A path to a late node in each tree, node 0 first where its line begins there; -1 behind."""
    rng = np.random.default_rng(seed)
    B, T = parent.shape
    path = np.full((B, T), -1, np.int32)
    for b in range(B):
        mine = ot.line(parent[b], int(rng.integers(T // 2, T)))
        path[b, :len(mine)] = mine
    return path


# ---- DeltaNet ---------------------------------------------------------------------------------------

def _dn(B, T, Hk, Hv, seed, **kw):
    d = deltanet_inputs(B, T, Hk, Hv, seed=seed, **kw)
    return d, deltanet_flat_device(d)


def _verify(ops, f, parent):
    return ops.deltanet.verify_tree(f["state"], parent, f["mixed_qkv"], f["conv_state"], f["conv_weight"],
                                    f["conv_bias"], f["a_out"], f["b_out"], f["z"], f["A_log"], f["dt_bias"],
                                    f["norm_weight"])


def _records(rec, B, T, Hk, Hv):
    rec = rec.cpu().double().numpy()
    k, u, decay = np.split(rec, [B * T * Hk * 128, B * T * (Hk + Hv) * 128])
    return k.reshape(B, T, Hk, 128), u.reshape(B, T, Hv, 128), decay.reshape(B, T, Hv)


@pytest.mark.parametrize("B,T,Hk,Hv,reach", [
    (1, 1, 1, 1, 1), (2, 2, 1, 3, 1), (3, 5, 2, 2, 2), (1, 15, 4, 12, 4), (2, 16, 2, 6, 16), (1, 17, 1, 3, 3),
    (2, 31, 1, 2, 8), (1, 32, 2, 4, 1), (1, 33, 1, 1, 5), (2, 48, 1, 2, 12), (1, 63, 1, 3, 1), (2, 64, 1, 2, 16),
    (1, 64, 2, 2, 64),
])
def test_verify_tree_matches_oracle(ops, B, T, Hk, Hv, reach):
    d, f = _dn(B, T, Hk, Hv, seed=T + reach, state_std=0.1)
    parent = trees(B, T, reach, seed=T)
    out, rec = _verify(ops, f, cuda(parent))
    torch.cuda.synchronize()
    ref, *want, _ = ot.deltanet_verify(deltanet_oracle_args(d), parent, Hk, Hv)
    for name, got, r in zip(("k", "u", "decay"), _records(rec, B, T, Hk, Hv), want):
        assert_rel_close(got, r, tol=F32_TOL, name=name)
    out_close(out, ref)


@pytest.mark.parametrize("T,B,where", [(1, 27, "v"), (2, 27, "k"), (7, 27, "q"), (16, 27, "v"), (15, 27, "k"), (33, 9, "k"),
                                       (47, 9, "v"), (48, 9, "q"), (49, 9, "k"), (64, 9, "v")])
def test_verify_tree_many_heads(ops, T, B, where):
    """More heads than run at once, which have kernels of their own up to 16 and above 32 nodes: one request against
    the oracle, some against one by one; a node that is not a number in the middle stays on its branch."""
    Hk, Hv = 1, 29
    d, f = _dn(B, T, Hk, Hv, seed=T, state_std=0.1)
    parent = trees(B, T, 5, seed=T, wild=True)
    out, rec = _verify(ops, f, cuda(parent))
    got = _records(rec, B, T, Hk, Hv)
    out = out.reshape(B, T, Hv, 128)
    one = lambda b: {k: v[b:b + 1] if v.shape[0] == B else v for k, v in d.items()}  # noqa: E731
    ref, *want, _ = ot.deltanet_verify(deltanet_oracle_args(one(4)), parent[4:5], Hk, Hv)
    out_close(out[4:5], ref)
    for g, r in zip(got, want):
        assert_rel_close(g[4:5], r, tol=F32_TOL)
    for b in range(0, B, 4):
        o, r = _verify(ops, deltanet_flat_device(one(b)), cuda(parent[b:b + 1]))
        for g, w in zip(got, _records(r, 1, T, Hk, Hv)):
            assert_rel_close(g[b:b + 1], w, tol=2 * F32_TOL)
        assert_rel_close(out[b].float().cpu().numpy(), o.float().cpu().double().numpy().reshape(T, Hv, 128), tol=4e-3, out_unit=2 * BF16_U)
    d["mixed_qkv"][3, T // 2, {"q": 5, "k": 128 + 5, "v": 256 + 17 * 128 + 5}[where]] = float("nan")
    bad, brec = _verify(ops, deltanet_flat_device(d), cuda(parent))
    hit = torch.zeros(B, T, Hv, 128, dtype=torch.bool, device="cuda")
    # a query: the nodes whose window has it; a key: all below; a value: all below, its head
    lines = [ot.line(parent[3], t) for t in range(T)]
    below = torch.tensor([T // 2 in (mine[-4:] if where == "q" else mine) for mine in lines])
    hit[3, below, 17 if where == "v" else 0:18 if where == "v" else Hv] = True
    bad = bad.reshape(hit.shape)
    assert torch.isnan(bad[hit]).all() and torch.equal(bad[~hit], out[~hit])


def test_verify_tree_takes_odd_parents(ops):
    """Parents that are none, the node itself, later or out of range hang the node on the committed tokens."""
    B, T = 3, 40
    d, f = _dn(B, T, 1, 2, seed=5)
    parent = trees(B, T, 6, seed=5, wild=True)
    out, rec = _verify(ops, f, cuda(parent))
    ref = ot.deltanet_verify(deltanet_oracle_args(d), parent, 1, 2)[0]
    out_close(out, ref)


@pytest.mark.parametrize("T", [4, 8, 16])
def test_verify_tree_of_a_chain_is_verify_batched(ops, T):
    """Against the chain op's out and checkpoints, the states that committing each prefix gives."""
    B, Hk, Hv = 2, 2, 6
    d, f = _dn(B, T, Hk, Hv, seed=T)
    out, rec = _verify(ops, f, cuda(trees(B, T, 1, 0)))
    ck, want = ops.deltanet.verify_batched(*[f[n] for n in ("state", "mixed_qkv", "conv_state", "conv_weight",
                                             "conv_bias", "a_out", "b_out", "z", "A_log", "dt_bias", "norm_weight")])
    # two roundings to bf16 of values that are F32_TOL apart: one ulp where one of them flips
    assert_rel_close(out.float().cpu().numpy(), want.float().cpu().double().numpy(), tol=2e-3, out_unit=2 * BF16_U, name="out")
    ck = ck.reshape(B, T, Hv, 128, 128)
    for n in (1, T // 2, T):
        path = np.full((B, T), -1, np.int32)
        path[:, :n] = np.arange(n)
        state, conv = f["state"].clone(), f["conv_state"].clone()
        ops.deltanet.commit_tree_([state], [conv], [f["mixed_qkv"]], [rec], cuda(path), Hv)
        assert_rel_close(state.cpu().numpy().reshape(B, Hv, 128, 128), ck[:, n - 1].cpu().double().numpy(), tol=2 * F32_TOL)
        assert torch.equal(conv, ops.deltanet.conv_rollback(f["mixed_qkv"], f["conv_state"], cuda(np.full(B, n - 1, np.int32)), Hv))


@pytest.mark.parametrize("gate", ["wiped", "kept", "far"])
def test_verify_tree_extreme_decays(ops, gate):
    """Decays that underflow to 0 (the node forgets all before it), that are 1, and sums of g far from 0."""
    B, T, Hk, Hv = 1, 48, 1, 2
    d, f = _dn(B, T, Hk, Hv, seed=9)
    rng = np.random.default_rng(9)
    if gate == "wiped":
        a = np.where(rng.random((B, T, Hv)) < 0.2, 1e4, -3.0)
    elif gate == "kept":
        a = np.full((B, T, Hv), -200.0)
    else:
        a = np.where(rng.random((B, T, Hv)) < 0.3, 90.0, -6.0)
    d["a_out"] = torch.from_numpy(a).float()
    d["A_log"], d["dt_bias"] = torch.zeros(Hv), torch.zeros(Hv)
    f = deltanet_flat_device(d)
    parent = trees(B, T, 4, seed=9)
    out, rec = _verify(ops, f, cuda(parent))
    ref, *want, _ = ot.deltanet_verify(deltanet_oracle_args(d), parent, Hk, Hv)
    assert_rel_close(_records(rec, B, T, Hk, Hv)[1], want[1], tol=F32_TOL, name="u")
    out_close(out, ref)


@pytest.mark.parametrize("T", [9, 24, 64])
@pytest.mark.parametrize("what", ["x", "xinf", "a", "b"])
def test_verify_tree_nan_stays_on_its_branch(ops, T, what):
    """A node whose input, decay or gate is not a number makes its own and its descendants' rows NaN (an input
    also those of the two heads that share its key, and as far as the window reaches), and no others."""
    B, Hk, Hv = 2, 1, 2
    d, f = _dn(B, T, Hk, Hv, seed=T)
    parent = trees(B, T, 3, seed=T + 1)
    clean, crec = _verify(ops, f, cuda(parent))
    node = T // 2
    below = np.array([node in ot.line(parent[1], t) for t in range(T)])
    if what[0] == "x":
        d["mixed_qkv"][1, node, 128 + 5] = float("nan") if what == "x" else float("inf")  # a key's channel
    else:
        d[what + "_out"][1, node, 1] = float("nan")
    f = deltanet_flat_device(d)
    out, rec = _verify(ops, f, cuda(parent))
    hit = torch.zeros(B, T, Hv, 128, dtype=torch.bool, device="cuda")
    hit[1, torch.from_numpy(below), 0 if what[0] == "x" else 1:] = True
    out, clean = out.reshape(hit.shape), clean.reshape(hit.shape)
    assert torch.isnan(out[hit]).all()
    assert torch.equal(out[~hit], clean[~hit])
    for x, y in zip(_records(rec, B, T, Hk, Hv)[:2], _records(crec, B, T, Hk, Hv)):
        other = np.ones((B, T), bool)
        other[1] = ~below
        assert np.array_equal(x[other], y[other])
    if what != "x" and what != "xinf":
        assert torch.isnan(torch.from_numpy(_records(rec, B, T, Hk, Hv)[1])[hit.cpu()]).all()


@pytest.mark.parametrize("L,B,T,Hk,Hv", [(1, 1, 1, 1, 1), (3, 2, 9, 2, 6), (2, 3, 64, 1, 3), (70, 1, 5, 1, 1), (2, 20, 16, 1, 2)])
def test_commit_tree_matches_oracle(ops, L, B, T, Hk, Hv):
    ds = [_dn(B, T, Hk, Hv, seed=l) for l in range(L)]
    parent = trees(B, T, 3, seed=T)
    path = some_paths(parent, seed=L)
    if B > 2:
        path[1] = -1                      # a request that sits out
        path[2, :3] = [2, 1, 5][:3]       # ends where it no longer ascends
    recs = [_verify(ops, f, cuda(parent))[1] for _, f in ds]
    stack = torch.stack([torch.cat([r[:1], r]) for r in recs])  # kept in one tensor: off 16 bytes, as odd heads leave them
    recs = [r[1:] for r in stack]
    states, convs = [f["state"].clone() for _, f in ds], [f["conv_state"].clone() for _, f in ds]
    ops.deltanet.commit_tree_(states, convs, [f["mixed_qkv"] for _, f in ds], recs, cuda(path), Hv)
    torch.cuda.synchronize()
    for (d, f), rec, state, conv in zip(ds, recs, states, convs):
        a = deltanet_oracle_args(d)
        want, window = ot.deltanet_commit(a[0], a[2], a[1], *_records(rec, B, T, Hk, Hv), path)
        assert_rel_close(state.cpu().double().numpy().reshape(want.shape), want, tol=F32_TOL, name="state")
        assert np.array_equal(bits(conv).reshape(window.shape), window)
        if B > 2:
            assert torch.equal(state.reshape(B, -1)[1], f["state"].reshape(B, -1)[1])


# ---- the walk ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("B,T,reach", [(1, 1, 1), (3, 2, 1), (50, 7, 2), (64, 33, 33), (300, 64, 20), (9, 64, 1)])
def test_accept_tree_matches_oracle(ops, B, T, reach):
    rng = np.random.default_rng(B + T)
    parent = trees(B, T, reach, seed=B, wild=B > 5)
    draft, target = rng.integers(-2, 3, (2, B, T))
    draft, target = draft + (draft > 0) * 2**40, target + (target > 0) * 2**40  # past 32 bits; siblings alike; negative
    q_len = rng.integers(-1, T + 3, B).astype(np.int32)
    got = ops.spec.accept_tree(cuda(target), cuda(draft), cuda(parent), cuda(q_len))
    for g, w in zip(got, ot.accept(target, draft, parent, q_len)):
        assert np.array_equal(g.cpu().numpy(), w)


# ---- attention --------------------------------------------------------------------------------------

def _attend_inputs(B, T, H, grp, bs, kv, n, reach, seed, wild=False, spare=2):
    """Pages of finite bytes, NaN in pages that are no request's, tables with no spare entries."""
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    kv, n = np.asarray(kv, np.int32), np.asarray(n, np.int32)
    need = [-(-(int(k) + T) // bs) for k in kv]
    P, N = max(need), sum(need) + spare
    cache = [rng.integers(0, 256, (N, H, bs, 256)).astype(np.uint8) & 0xF7,
             rng.integers(0, 256, (N, H, 256, bs)).astype(np.uint8) & 0xF7,
             np.exp2(rng.integers(-9, -5, (N, H))).astype(np.float32),
             np.exp2(rng.integers(-9, -5, (N, H))).astype(np.float32)]
    ids = rng.permutation(N)
    for i in ids[sum(need):]:
        cache[0][i], cache[1][i] = 0x7F, 0xFF
    table, slots, used = np.full((B, P), -1, np.int32), np.full((B, T), -1, np.int64), 0
    for b in range(B):
        table[b, :need[b]] = ids[used:used + need[b]]
        used += need[b]
        pos = kv[b] + np.arange(max(n[b], 0))
        slots[b, :max(n[b], 0)] = table[b, pos // bs].astype(np.int64) * bs + pos % bs
    r = lambda *s: torch.randn(*s, generator=g).to(BF)  # noqa: E731
    cos, sin = og.rope_cos_sin(np.arange(max(kv) + T))
    return dict(query=r(B, T, H * grp, 256), gate=r(B, T, H * grp, 256), key=r(B, T, H, 256), value=r(B, T, H, 256),
                q_norm=torch.randn(256, generator=g) * 0.1, k_norm=torch.randn(256, generator=g) * 0.1, cos=cos, sin=sin,
                cache=cache, table=table, slots=slots, kv=kv, n=n, parent=trees(B, T, reach, seed, wild))


def _args(d):
    cache = [cuda(d["cache"][0].view(np.int8)), cuda(d["cache"][1].view(np.int8)), cuda(d["cache"][2]), cuda(d["cache"][3])]
    t = lambda *names: [d[k].cuda() for k in names]  # noqa: E731
    return [*t("query", "gate", "key", "value", "q_norm", "k_norm"), cuda(d["cos"]), cuda(d["sin"]), *cache,
            cuda(d["table"]), cuda(d["kv"]), cuda(d["slots"]), cuda(d["n"]), cuda(d["parent"])]


def _check(ops, d):
    """The pages to a step of e4m3 where fp32 and 64 bits round a key apart, the attention on the bytes that it reads."""
    args = _args(d)
    out = ops.gqa.tree_verify_paged(*args)
    torch.cuda.synchronize()
    f = lambda k: d[k].double().numpy()  # noqa: E731
    want = [c.copy() for c in d["cache"]]
    ot.kv_append(f("key"), f("value"), f("k_norm"), d["cos"], d["sin"], d["kv"], d["slots"], d["parent"], want)
    cache = [a.cpu().numpy() for a in args[8:12]]
    cache[0], cache[1] = cache[0].view(np.uint8), cache[1].view(np.uint8)
    for i in (1, 2, 3):
        assert np.array_equal(cache[i], want[i]), i
    off = np.abs((cache[0] & 0x7F).astype(int) - (want[0] & 0x7F))
    assert off.max() <= 1 and (off > 0).mean() <= 1e-3 + 2 / off.size
    ref = ot.tree_verify(f("query"), f("gate"), f("q_norm"), d["cos"], d["sin"], cache, d["table"], d["kv"], d["n"], d["parent"])
    got = out.float().cpu().double().numpy()
    assert_rel_close(got, ref, tol=2e-3, out_unit=BF16_U, name="tree_verify_paged")
    for b, n in enumerate(d["n"]):
        assert not got[b, max(int(n), 0):].any()
    return args, out


@pytest.mark.parametrize("B,T,H,grp,bs,kv,n,reach", [
    (1, 1, 1, 1, 16, [0], [1], 1),                             # one key
    (1, 1, 2, 6, 64, [300], [1], 1),
    (3, 2, 4, 6, 16, [0, 63, 62], [2, 2, 1], 2),               # 16 rows; step ends inside the tree
    (2, 5, 1, 6, 32, [5, 128], [5, 4], 3),                     # 32 rows
    (2, 8, 4, 6, 64, [37, 600], [8, 8], 4),                    # 48 rows
    (4, 8, 2, 6, 128, [127, 0, 1500, 11], [8, 0, 3, 8], 8),    # padded and idle requests
    (2, 3, 2, 16, 16, [100, 33], [3, 3], 2),                   # 48 rows of 16 a node
    (3, 9, 2, 6, 32, [250, 0, 63], [9, 4, 9], 3),              # 54 rows: two groups
    (2, 16, 1, 4, 64, [1000, 60], [16, 11], 5),                # 64 rows
    (3, 16, 2, 6, 16, [500, 0, 61], [16, 16, 9], 5),           # 96 rows
    (2, 64, 1, 6, 16, [70, 0], [64, 20], 16),                  # groups without a live node; five pages
    (1, 33, 1, 5, 64, [1000], [33], 33),                       # nodes that straddle groups
    (2, 64, 2, 2, 128, [255, 120], [64, 63], 1),               # chains of 64
    (9, 20, 4, 6, 16, [0, 5, 100, 300, 700, 1100, 64, 128, 33], [20, 19, 1, 20, 17, 20, 0, 20, 2], 6),
    (1, 63, 1, 48, 32, [40], [63], 7),                         # 24 groups
])
def test_tree_verify_paged_matches_oracle(ops, B, T, H, grp, bs, kv, n, reach):
    _check(ops, _attend_inputs(B, T, H, grp, bs, kv, n, reach, seed=B * 7 + T))


@pytest.mark.parametrize("T", [7, 40])
def test_tree_verify_paged_odd_parents(ops, T):
    _check(ops, _attend_inputs(3, T, 2, 6, 16, [20, 100, 0], [T, T, T], 4, seed=T, wild=True))


def test_tree_verify_paged_long(ops):
    """More steps than a workgroup has pages of in LDS at a time."""
    _check(ops, _attend_inputs(1, 4, 1, 4, 16, [33000], [4], 2, seed=2))
    _check(ops, _attend_inputs(2, 24, 1, 6, 128, [32768 - 8, 17000], [24, 24], 6, seed=5))


@pytest.mark.parametrize("T", [2, 5, 8, 30, 64])
def test_tree_verify_paged_of_a_chain_is_append_and_verify(ops, T):
    d = _attend_inputs(3, T, 2, 6, 16, [77, 0, 500], [T, T, T - 1], 1, seed=T)
    args, out = _check(ops, d)
    query, gate, key, value, qn, kn, cos, sin, *cache, table, kv, slots, n, _ = _args(d)
    ops.gqa.kv_append_paged(key, value, kn, cos, sin, kv, slots, *cache)
    want = ops.gqa.tail_verify_paged(query, gate, qn, cos, sin, *cache, table, kv, n)
    if T >= 30:  # another kernel's roundings: both within the tolerance of the formula, so within twice that of each other
        assert_rel_close(out.float().cpu().numpy(), want.float().cpu().numpy(), tol=4e-3, out_unit=2 * BF16_U)
    else:
        assert torch.equal(out, want)
    assert all(torch.equal(a, b) for a, b in zip(args[8:12], cache))


@pytest.mark.parametrize("T", [6, 40])
@pytest.mark.parametrize("where", ["key", "value"])
def test_tree_verify_paged_nan_stays_on_its_branch(ops, T, where):
    """A node whose key or value is not a number reaches itself and its descendants, and no others."""
    d = _attend_inputs(2, T, 2, 6, 16, [61, 30], [T, T], 3, seed=12)
    clean = ops.gqa.tree_verify_paged(*_args(d))
    node = T // 3
    below = torch.from_numpy(np.array([node in ot.line(d["parent"][0], t) for t in range(T)]))
    d[where][0, node, 1, 17] = float("nan")
    got = ops.gqa.tree_verify_paged(*_args(d))
    hit = torch.zeros_like(got, dtype=torch.bool)
    if where == "key":
        hit[0, below, 6:] = True
    else:
        hit[0, below, 6:, 17] = True
    assert torch.isnan(got[hit]).all() and 0 < int(below.sum()) < T
    # (a value that is not finite leaves its page's scale to the others, of which it was none's largest)
    assert torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("T", [6, 40])
@pytest.mark.parametrize("at", [58, 60])
def test_tree_verify_paged_nan_before_the_tree(ops, T, at):
    """A committed key's or value's NaN reaches every live row of its head, in the step that the tree begins in too."""
    for which in (0, 1):
        d = _attend_inputs(2, T, 2, 6, 16, [61, 30], [T - 1, T], 3, seed=13)
        clean = ops.gqa.tree_verify_paged(*_args(d))
        page, row = d["table"][0, at // 16], at % 16
        if which == 0:
            d["cache"][0][page, 1, row, 17] = 0x7F
        else:
            d["cache"][1][page, 1, 17, row] = 0xFF
        got = ops.gqa.tree_verify_paged(*_args(d))
        hit = torch.zeros_like(got, dtype=torch.bool)
        if which == 0:
            hit[0, :T - 1, 6:] = True
        else:
            hit[0, :T - 1, 6:, 17] = True
        assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("T", [5, 40])
def test_tree_verify_paged_missing_pages(ops, T):
    """Table entries that are none hide their positions, the tree's own among them."""
    d = _attend_inputs(3, T, 2, 6, 16, [40, 5, 100], [T, T, T], 3, seed=10)
    d["slots"][:] = -1  # nothing is appended; the pages hold finite bytes
    d["table"][0, 1] = -1
    d["table"][1] = len(d["cache"][0])
    d["table"][2, [0, 3, 6]] = [2**31 - 1, -2**31, -1]
    _check(ops, d)


@pytest.mark.parametrize("T", [5, 40])
def test_tree_verify_paged_short_table_row(ops, T):
    """Positions past what the table's row holds are none's; rows without a key are 0."""
    d = _attend_inputs(2, T, 2, 6, 16, [30, 20], [T, T], 3, seed=11)
    d["table"] = np.ascontiguousarray(d["table"][:, :2])
    d["slots"][:] = -1
    _check(ops, d)


# ---- compaction -------------------------------------------------------------------------------------

def _pages(L, N, H, bs, rng, spread):
    cache = [[rng.integers(0, 256, (N, H, bs, 256)).astype(np.uint8), rng.integers(0, 256, (N, H, 256, bs)).astype(np.uint8),
              np.exp2(rng.integers(-9, -9 + spread, (N, H))).astype(np.float32),
              np.exp2(rng.integers(-9, -9 + spread, (N, H))).astype(np.float32)] for _ in range(L)]
    return cache


def _compact(ops, caches, path, slots):
    """The op on copies of the caches; back as numpy."""
    dev = [[cuda(c[0].view(np.int8)), cuda(c[1].view(np.int8)), cuda(c[2]), cuda(c[3])] for c in caches]
    ops.gqa.compact_paged_(cuda(path), cuda(slots), *[list(x) for x in zip(*dev)])
    torch.cuda.synchronize()
    return [[c[0].cpu().numpy().view(np.uint8), c[1].cpu().numpy().view(np.uint8), c[2].cpu().numpy(), c[3].cpu().numpy()]
            for c in dev]


@pytest.mark.parametrize("L,B,T,H,bs,reach,spread", [
    (1, 1, 1, 1, 16, 1, 1), (2, 3, 8, 2, 64, 3, 1), (1, 6, 16, 4, 16, 4, 6), (3, 5, 64, 1, 16, 12, 9),
    (33, 2, 20, 1, 32, 5, 4), (2, 7, 64, 2, 128, 64, 3), (1, 8, 33, 1, 32, 2, 20),
])
def test_compact_paged_matches_oracle(ops, L, B, T, H, bs, reach, spread):
    """Random bytes, NaN among them; scales alike (bytes move), near and far apart."""
    rng = np.random.default_rng(T + L)
    parent = trees(B, T, reach, seed=T)
    path = some_paths(parent, seed=B)
    per = -(-(bs - 1 + T) // bs)
    N = B * per + 1
    caches, ids = _pages(L, N, H, bs, rng, spread), rng.permutation(N)[:B * per].reshape(B, per)
    at = rng.integers(0, bs, B)[:, None] + np.arange(T)
    slots = np.take_along_axis(ids, at // bs, 1) * bs + at % bs
    if B > 4:
        path[0] = -1                 # sits out
        slots[1, T // 2:] = -1       # granted for less than the path wants
        path[2, 1:] = path[2, :-1]   # a path that does not ascend
        slots[3, -1] = N * bs        # past the pool
    got = _compact(ops, caches, path, slots.astype(np.int64))
    for g, c in zip(got, caches):
        ot.compact(path, slots, c)
        assert np.array_equal(g[2], c[2]) and np.array_equal(g[3], c[3])
        for a, b in ((g[0], c[0]), (g[1], c[1])):
            x, y = fp8.decode_e4m3fn(a), fp8.decode_e4m3fn(b)
            assert np.array_equal(x, y, equal_nan=True)


def test_compact_paged_rows_with_no_finite_value(ops):
    """A row of NaN or zeros from a page of a larger scale leaves its new page's alone."""
    rng = np.random.default_rng(0)
    bs, T = 16, 20
    cache = _pages(1, 2, 1, bs, rng, 1)
    for c in cache:
        c[2][1], c[3][1] = 1.0, 1.0
        c[0][1, 0, :2], c[1][1, 0, :, :2] = 0x7F, 0x80  # slots 16, 17
    slots = np.arange(T)[None].astype(np.int64)
    path = np.full((1, T), -1, np.int32)
    path[0, :3] = [0, 16, 17]
    got = _compact(ops, cache, path, slots)
    assert got[0][2][0, 0] == cache[0][2][0, 0] and got[0][3][0, 0] == cache[0][3][0, 0]
    assert (got[0][0][0, 0, 1:3] == 0x7F).all() and ((got[0][1][0, 0, :, 1:3] & 0x7F) == 0).all()


# ---- refusals ---------------------------------------------------------------------------------------

def test_refusals(ops):
    d, f = _dn(1, 4, 1, 2, seed=0)
    parent = cuda(trees(1, 4, 2, 0))
    good = [f["state"], parent, *[f[n] for n in ("mixed_qkv", "conv_state", "conv_weight", "conv_bias", "a_out", "b_out",
                                                  "z", "A_log", "dt_bias", "norm_weight")]]
    for i, bad, err in ((0, good[0].double(), TypeError), (1, parent.long(), TypeError), (1, parent[0], RuntimeError),
                        (1, torch.zeros(1, 65, dtype=I32, device="cuda"), RuntimeError), (1, parent[:, :0], RuntimeError),
                        (1, parent[:0], RuntimeError), (2, good[2][:-1], RuntimeError), (6, good[6].cpu(), RuntimeError),
                        (8, good[8].float(), TypeError), (9, good[9][:1], RuntimeError)):
        with pytest.raises(err):
            ops.deltanet.verify_tree(*[bad if j == i else a for j, a in enumerate(good)])
    rec = _verify(ops, f, parent)[1]
    path = cuda(np.array([[0, 1, -1, -1]], np.int32))
    lists = [[f["state"]], [f["conv_state"]], [f["mixed_qkv"]], [rec]]
    for bad in ([[], *lists[1:]], [*lists[:3], [rec[:-1]]], [[f["state"].double()], *lists[1:]],
                [2 * l for l in lists]):  # the last: one layer's state twice
        with pytest.raises((RuntimeError, TypeError)):
            ops.deltanet.commit_tree_(*bad, path, 2)
    with pytest.raises(RuntimeError):
        ops.deltanet.commit_tree_(*lists, path, 1)
    with pytest.raises(RuntimeError, match="requires grad"):
        ops.deltanet.commit_tree_([f["state"].clone().requires_grad_()], *lists[1:], path, 2)
    ops.deltanet.commit_tree_([], [], [], [], path, 2)
    ids = torch.zeros(1, 4, dtype=torch.int64, device="cuda")
    one = torch.ones(1, dtype=I32, device="cuda")
    for bad in ((ids.int(), ids, parent, one), (ids, ids[:, :3], parent, one), (ids, ids, parent, one.long()),
                (ids, ids, parent.cpu(), one)):
        with pytest.raises((RuntimeError, TypeError)):
            ops.spec.accept_tree(*bad)
    a = _attend_inputs(1, 4, 1, 6, 16, [5], [4], 2, seed=1)
    args = _args(a)
    for i, bad, err in ((0, args[0].float(), TypeError), (2, args[2][:, :3], RuntimeError), (9, args[9].transpose(2, 3), RuntimeError),
                        (14, args[14].int(), TypeError), (16, args[16][:, :2], RuntimeError), (16, args[16].long(), TypeError),
                        (13, args[13].cpu(), RuntimeError)):
        with pytest.raises(err):
            ops.gqa.tree_verify_paged(*[bad if j == i else x for j, x in enumerate(args)])
    slots = args[14]
    for bad in ([[], args[9:10], args[10:11], args[11:12]], [2 * [x] for x in args[8:12]],
                [[args[8].float()], *[[x] for x in args[9:12]]]):
        with pytest.raises((RuntimeError, TypeError)):
            ops.gqa.compact_paged_(path, slots, *bad)
    with pytest.raises(RuntimeError):
        ops.gqa.compact_paged_(path, slots[:, :3].contiguous(), *[[x] for x in args[8:12]])
