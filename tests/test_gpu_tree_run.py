"""The tree-verification operators together, as a serving loop uses them: plan, DeltaNet and attention over a tree,
walk, commit, compact, give back, over many steps against the oracle; captured and replayed; on two
streams and another stream than the tensors'; compiled; and as the verify slice's step."""
import numpy as np
import pytest
import torch

from oracle import gqa as og, paged as op, tree as ot
from _util import BF16_U, assert_rel_close, bits, deltanet_flat_device, deltanet_inputs, deltanet_oracle_args
from test_gpu_tree import F32_TOL, cuda, out_close, trees

pytestmark = pytest.mark.gpu
BF, I32 = torch.bfloat16, torch.int32
HK, HV, H, GRP, T = 1, 3, 2, 6, 12
QKV = (2 * HK + HV) * 128


def _world(B, P, N, bs, seed):
    """Device state of B requests: one DeltaNet layer's and two attention layers' over one block table."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    d = deltanet_flat_device(deltanet_inputs(B, T, HK, HV, seed=seed))
    w = dict(d, table=torch.full((B, P), -1, dtype=I32), held=torch.zeros(B, dtype=I32),
             free=torch.randperm(N, generator=g).int(), count=torch.tensor([N], dtype=I32), kv_len=torch.zeros(B, dtype=I32),
             last=torch.zeros(B, dtype=I32), committed=torch.zeros(B, dtype=I32), k_norm=r(256) * 0.1, q_norm=r(256) * 0.1)
    cos, sin = og.rope_cos_sin(np.arange(P * bs))
    w["cos"], w["sin"] = torch.from_numpy(cos), torch.from_numpy(sin)
    for l in range(2):
        w[f"k{l}"], w[f"v{l}"] = (torch.zeros(N, H, *s, dtype=torch.int8) for s in ((bs, 256), (256, bs)))
        w[f"ks{l}"], w[f"vs{l}"] = torch.zeros(2, N, H)
    return {k: v.contiguous().cuda() for k, v in w.items()}


def _inputs(B, seed, sizes=True):
    """A step's rows, trees and tokens; some requests with fewer nodes or none."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    rng = np.random.default_rng(seed)
    parent = trees(B, T, 4, seed)
    draft = rng.integers(0, 3, (B, T))
    n = rng.integers(0, T + 1, B) if sizes else np.full(B, T)
    return dict(mixed=r(B * T * QKV).to(BF), a=r(B * T * HV), b=r(B * T * HV), z=r(B * T * HV, 128).to(BF),
                query=r(2, B, T, H * GRP, 256).to(BF), gate=r(2, B, T, H * GRP, 256).to(BF),
                key=(r(2, B, T, H, 256) * (1 + 7 * torch.rand(2, B, T, 1, 1, generator=g, device="cuda"))).to(BF),
                value=(r(2, B, T, H, 256) * (1 + 7 * torch.rand(2, B, T, 1, 1, generator=g, device="cuda"))).to(BF),
                parent=cuda(parent), draft=cuda(draft), target=cuda(rng.integers(0, 3, (B, T))), n=cuda(n.astype(np.int32)))


def _step(ops, w, x, bs):
    slots, granted = ops.paged.update_blocks_(w["kv_len"], x["n"], w["table"], w["held"], w["free"], w["count"], bs, T)
    out, rec = ops.deltanet.verify_tree(w["state"], x["parent"], x["mixed"], w["conv_state"], w["conv_weight"], w["conv_bias"],
                                        x["a"], x["b"], x["z"], w["A_log"], w["dt_bias"], w["norm_weight"])
    attn = [ops.gqa.tree_verify_paged(x["query"][l], x["gate"][l], x["key"][l], x["value"][l], w["q_norm"], w["k_norm"], w["cos"],
                                      w["sin"], w[f"k{l}"], w[f"v{l}"], w[f"ks{l}"], w[f"vs{l}"], w["table"], w["kv_len"],
                                      slots, granted, x["parent"]) for l in range(2)]
    accepted, path, ids = ops.spec.accept_tree(x["target"], x["draft"], x["parent"], granted)
    ops.deltanet.commit_tree_([w["state"]], [w["conv_state"]], [x["mixed"]], [rec], path, HV)
    ops.gqa.compact_paged_(path, slots, *[[w[f"{k}{l}"] for l in range(2)] for k in ("k", "v", "ks", "vs")])
    ops.spec.commit_(accepted, w["last"], w["kv_len"], w["committed"])
    return slots, granted, out, rec, *attn, accepted, path, ids


def _oracle_step(w, x, bs):
    """The step on numpy copies of w before it; what it leaves, and its outputs."""
    c = {k: v.cpu().numpy().copy() if v.dtype != BF else bits(v).copy() for k, v in w.items()}
    B = len(c["kv_len"])
    parent, n = x["parent"].cpu().numpy(), x["n"].cpu().numpy()
    slots, granted, free = op.update_blocks(c["kv_len"], n, c["table"], c["held"], c["free"], c["count"][0], bs, T)
    shaped = lambda v, *s: v.reshape(*s)  # noqa: E731
    d = (shaped(c["state"], B, HV, 128, 128), shaped(bits(x["mixed"]), B, T, QKV), shaped(c["conv_state"], B, QKV, 3),
         c["conv_weight"], c["conv_bias"], shaped(x["a"].cpu().numpy(), B, T, HV), shaped(x["b"].cpu().numpy(), B, T, HV),
         shaped(bits(x["z"]), B, T, HV, 128), c["A_log"], c["dt_bias"], c["norm_weight"])
    out, k, u, decay, _ = ot.deltanet_verify(d, parent, HK, HV)
    accepted, path, ids = ot.accept(x["target"].cpu().numpy(), x["draft"].cpu().numpy(), parent, granted)
    state, conv = ot.deltanet_commit(d[0], d[2], d[1], k, u, decay, path)
    return dict(c=c, slots=slots, granted=granted, free=free, out=out, accepted=accepted, path=path, ids=ids, state=state,
                conv=conv, parent=parent)


@pytest.mark.parametrize("N,short", [(22, False), (6, True)])
def test_serving_loop_matches_oracle(ops, N, short):
    """Thirty steps with requests that end and sit out, a pool with room and one that refuses some: every output, the
    states and the pages themselves. The pages' bytes of K are checked to a step and then taken over, so that each step
    is checked on the bytes it reads."""
    B, P, bs = 4, 7, 16
    w = _world(B, P, N, bs, seed=3)
    rng = np.random.default_rng(5)
    refused = moved = 0
    for step in range(30):
        x = _inputs(B, 100 + step)
        room = P * bs - w["kv_len"] - T
        x["n"] = torch.where(room >= 0, x["n"], 0)
        o = _oracle_step(w, x, bs)
        slots, granted, out, rec, a0, a1, accepted, path, ids = _step(ops, w, x, bs)
        torch.cuda.synchronize()
        refused += int((granted < x["n"]).sum())
        for got, want in ((slots, "slots"), (granted, "granted"), (accepted, "accepted"), (path, "path"), (ids, "ids")):
            assert np.array_equal(got.cpu().numpy(), o[want]), (step, want)
        c = o["c"]
        assert np.array_equal(w["table"].cpu().numpy(), c["table"]) and int(w["count"]) == o["free"]
        out_close(out.reshape(B, T, HV, 128), o["out"])
        assert_rel_close(w["state"].cpu().numpy().reshape(o["state"].shape), o["state"], tol=F32_TOL)
        assert np.array_equal(bits(w["conv_state"]).reshape(o["conv"].shape), o["conv"])
        f = lambda t: t.double().cpu().numpy()  # noqa: E731
        for l, got in enumerate((a0, a1)):
            cache = [c[f"k{l}"].view(np.uint8), c[f"v{l}"].view(np.uint8), c[f"ks{l}"], c[f"vs{l}"]]
            ot.kv_append(f(x["key"][l]), f(x["value"][l]), f(w["k_norm"]), c["cos"], c["sin"], c["kv_len"], o["slots"],
                         o["parent"], cache)
            ref = ot.tree_verify(f(x["query"][l]), f(x["gate"][l]), f(w["q_norm"]), c["cos"], c["sin"], cache, c["table"],
                                 c["kv_len"], o["granted"], o["parent"])
            # K's bytes that fp32 and 64 bits round apart move a score by at most a step of one of 256 products: within
            # the tolerance of the attention's own roundings
            assert_rel_close(f(got.float()), ref, tol=2e-3, out_unit=BF16_U, name=f"step {step}")
            ot.compact(o["path"], o["slots"], cache)
            assert np.array_equal(w[f"v{l}"].cpu().numpy().view(np.uint8), cache[1])
            assert np.array_equal(w[f"ks{l}"].cpu().numpy(), cache[2]) and np.array_equal(w[f"vs{l}"].cpu().numpy(), cache[3])
            k = w[f"k{l}"].cpu().numpy().view(np.uint8)
            assert np.abs((k & 0x7F).astype(int) - (cache[0] & 0x7F)).max() <= 1
        moved += int((o["path"] > np.arange(T)).sum())
        kv = c["kv_len"] + o["accepted"] + 1
        assert np.array_equal(w["kv_len"].cpu().numpy(), kv)
        kv = kv.copy()
        kv[rng.random(B) < 0.1] = 0
        w["kv_len"].copy_(torch.from_numpy(kv.astype(np.int32)))
    assert (refused > 0) == short and moved > 30


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_steps_equal_eager_ones(ops):
    """Two graphs of a step on one state, replayed in turn with other work and synchronisations between, against eager
    steps on a copy of the state."""
    B, P, bs = 3, 20, 16
    a, b = _world(B, P, 60, bs, seed=7), _world(B, P, 60, bs, seed=7)
    inputs = [_inputs(B, 200 + k, sizes=False) for k in range(2)]
    for w in (a, b):
        _step(ops, w, inputs[0], bs)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(ops, a, x, bs))
        graphs.append(g)
    for n in range(24):
        for k, v in _inputs(B, 300 + n, sizes=n % 3 > 0).items():
            inputs[n % 2][k].copy_(v)
        graphs[n % 2].replay()
        torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")
        if n % 3 == 0:
            torch.cuda.synchronize()
        want = _step(ops, b, inputs[n % 2], bs)
        torch.cuda.synchronize()
        assert _same(outs[n % 2], want), n
        assert all(torch.equal(a[k], b[k]) for k in a), n


def test_two_streams_at_once(ops):
    """The same steps on two streams, neither the tensors' own, with states of their own give what they give alone."""
    B, P, bs = 3, 20, 32
    inputs = [_inputs(B, 400 + k, sizes=False) for k in range(6)]
    alone = [[_step(ops, w, x, bs) for x in inputs] for w in (_world(B, P, 60, bs, seed=k) for k in (9, 10))]
    worlds = [_world(B, P, 60, bs, seed=k) for k in (9, 10)]
    torch.cuda.synchronize()
    both = []
    for w in worlds:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            both.append([_step(ops, w, x, bs) for x in inputs])
    torch.cuda.synchronize()
    assert all(_same(p, q) for x, y in zip(alone, both) for p, q in zip(x, y))


def test_compiled_step_equals_eager(ops):
    import torch._dynamo
    torch._dynamo.reset()
    B, P, bs = 2, 10, 16
    a, b, x = _world(B, P, 20, bs, seed=12), _world(B, P, 20, bs, seed=12), _inputs(B, 500)
    want, got = _step(torch.ops, a, x, bs), torch.compile(lambda w: _step(torch.ops, w, x, bs), fullgraph=True,
                                                          backend="aot_eager")(b)
    torch.cuda.synchronize()
    assert _same(got, want) and all(torch.equal(a[k], b[k]) for k in a)


def test_verify_slice_steps_over_trees():
    """A chain's step_tree against step (within the roundings of DeltaNet's two ways to its states, through the layers
    behind it), then trees: replays equal eager steps bit for bit, pages and lengths agree, and a slice takes steps of one kind."""
    from spec_verify_step import HIDDEN, VerifySlice
    B, K, kv = 3, 7, [37, 300, 5]
    make = lambda: VerifySlice(B, K, kv, 512, pattern="DDG", seed=1, paged_block=16)  # noqa: E731
    chain, one, two = make(), make(), make()
    x = torch.randn(B * (K + 1), HIDDEN, device="cuda").to(BF)
    parent = torch.arange(-1, K, dtype=I32, device="cuda").expand(B, -1).contiguous()
    ids = torch.randint(0, 9, (B, K + 1), device="cuda")
    target = torch.full_like(ids, 99)
    target[0, :3], target[1, :K] = ids[0, 1:4], ids[1, 1:]
    want = chain.forward(x)
    hidden, accepted, path, out = one.step_tree(x, parent, ids, target)
    # the first DeltaNet layer's output is the chain's but for its last fp32 digits, which flips some of its roundings to
    # bf16: 2^-8 of some elements, carried through three layers
    assert_rel_close(hidden.float().cpu().numpy(), want.float().cpu().double().numpy(), tol=1e-2, out_unit=2 * BF16_U)
    assert accepted.tolist() == [3, K, 0] and one.kv_len.tolist() == [37 + 4, 300 + K + 1, 6]
    assert out[0].tolist()[:4] == ids[0, 1:4].tolist() + [99] and path[1].tolist() == list(range(K + 1))
    two.step_tree(x, parent, ids, target)
    args = (x, parent, ids, target, torch.full((B,), K + 1, dtype=I32, device="cuda"))
    two.capture_tree(*args)
    rng = np.random.default_rng(0)
    for n in range(8):
        x.copy_(torch.randn(x.shape, device="cuda").to(BF))
        parent.copy_(cuda(trees(B, K + 1, 3, seed=n)))
        ids.copy_(torch.randint(0, 2, ids.shape, device="cuda"))
        target.copy_(torch.randint(0, 2, ids.shape, device="cuda"))
        args[4].copy_(cuda(rng.integers(0, K + 2, B).astype(np.int32)))
        want, got = one.step_tree(*args), two.replay_tree()
        torch.cuda.synchronize()
        assert _same(got, want), n
        assert torch.equal(one.kv_len, two.kv_len) and torch.equal(one.committed, two.committed)
        for k in ("table", "held", "free", "count"):
            assert torch.equal(one.pages[k], two.pages[k])
        for p, q in zip(one.layers, two.layers):
            names = ("state", "conv_state") if p["kind"] == "D" else ("cache_k", "cache_v", "k_scale", "v_scale")
            assert all(torch.equal(p[k], q[k]) for k in names)
    with pytest.raises(RuntimeError, match="checkpoints"):
        chain.prev_accepted = accepted
        chain.step_tree(*args)


def test_verify_slice_of_deltanet_layers_alone():
    """A slice without attention layers has no pages: its tree steps take every node, or as many as they are told."""
    from spec_verify_step import HIDDEN, VerifySlice
    B, K = 2, 4
    one = VerifySlice(B, K, [9, 30], 64, pattern="DD", seed=2)
    x = torch.randn(B * (K + 1), HIDDEN, device="cuda").to(BF)
    parent = torch.tensor([[-1, 0, 0, 1, 2], [-1, 0, 1, 2, 3]], dtype=I32, device="cuda")
    ids = torch.tensor([[0, 5, 6, 7, 8], [0, 1, 2, 3, 4]], device="cuda")
    target = torch.tensor([[6, 1, 8, 1, 9], [1, 2, 3, 4, 5]], device="cuda")
    before = [L["state"].clone() for L in one.layers]
    _, accepted, path, out = one.step_tree(x, parent, ids, target)
    assert accepted.tolist() == [2, 4] and path[0].tolist() == [0, 2, 4, -1, -1] and out[0].tolist() == [6, 8, 9, -1, -1]
    assert one.kv_len.tolist() == [12, 35] and all(not torch.equal(L["state"], s) for L, s in zip(one.layers, before))
    before = [L["state"].clone() for L in one.layers]
    n = torch.tensor([0, 3], dtype=I32, device="cuda")
    _, accepted, _, _ = one.step_tree(x, parent, ids, target, n)
    assert accepted.tolist() == [-1, 2] and one.kv_len.tolist() == [12, 38]
    half = before[0].shape[0] // 2
    assert all(torch.equal(L["state"][:half], s[:half]) for L, s in zip(one.layers, before))
