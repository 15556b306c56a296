"""The paged operators together, as a serving loop uses them: plan, append, attend, sample, give back,
over many steps against the oracle; captured and replayed; on two streams; compiled; and as the KV
cache of the verify slice."""
import numpy as np
import pytest
import torch

from oracle import gqa as og, paged as op, sample as osm
from _util import BF16_U, assert_rel_close

pytestmark = pytest.mark.gpu
BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32
H, GRP = 2, 6


def _world(B, P, N, bs, V, seed):
    """Device state of B requests on N blocks, and a head from attention rows to V logits."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    cos, sin = og.rope_cos_sin(np.arange(P * bs))
    w = dict(table=torch.full((B, P), -1, dtype=I32), held=torch.zeros(B, dtype=I32),
             free=torch.randperm(N, generator=g).int(), count=torch.tensor([N], dtype=I32),
             cache_k=torch.zeros(N, H, bs, 256, dtype=torch.int8), cache_v=torch.zeros(N, H, 256, bs, dtype=torch.int8),
             k_scale=torch.zeros(N, H), v_scale=torch.zeros(N, H), kv_len=torch.zeros(B, dtype=I32),
             k_norm=r(256) * 0.1, q_norm=r(256) * 0.1, cos=torch.from_numpy(cos), sin=torch.from_numpy(sin),
             head=r(H * GRP * 256, V) * 0.05)
    return {k: v.cuda() for k, v in w.items()}


def _settings(B, gen):
    pick = lambda v, t: torch.tensor(v, dtype=t, device="cuda")[  # noqa: E731
        torch.randint(0, len(v), (B,), generator=gen, device="cuda")]
    return (pick([0.0, 0.7, 1.0], F32), pick([0, 5, 50], I32), pick([1.0, 0.9], F32), pick([0.0, 0.05], F32),
            torch.rand(B, generator=gen, device="cuda"))


def _rows(B, T, gen):
    r = lambda n: torch.randn(B, T, n, 256, generator=gen, device="cuda").to(BF)  # noqa: E731
    return r(H * GRP), r(H * GRP), r(H), r(H)


def _step(ops, w, new, rows, settings, bs, T):
    """Plan, append, attend, and a token from the last row that each request was granted."""
    query, gate, key, value = rows
    pages = (w["cache_k"], w["cache_v"], w["k_scale"], w["v_scale"])
    slots, granted = ops.paged.update_blocks_(w["kv_len"], new, w["table"], w["held"], w["free"], w["count"], bs, T)
    ops.gqa.kv_append_paged(key, value, w["k_norm"], w["cos"], w["sin"], w["kv_len"], slots, *pages)
    out = ops.gqa.tail_verify_paged(query, gate, w["q_norm"], w["cos"], w["sin"], *pages, w["table"], w["kv_len"],
                                    granted)
    at = (granted - 1).clamp(min=0).long()
    last = out[torch.arange(len(at), device="cuda"), at].reshape(len(at), -1).float()
    ids = ops.spec.sample(last @ w["head"], *settings)
    return slots, granted, out, ids


@pytest.mark.parametrize("N,short", [(24, False), (9, True)])
def test_serving_loop_matches_oracle(ops, N, short):
    """Prompts, plain decode and verify steps with some rows not kept, requests that end, a pool
    with room and one that is too small now and then: every output and the pages themselves, step by step."""
    B, P, bs, T, V = 5, 8, 16, 20, 997
    w = _world(B, P, N, bs, V, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(4)
    rng = np.random.default_rng(5)
    refused = 0
    for step in range(40):
        left = P * bs - w["kv_len"].cpu().numpy() - T
        new = rng.integers(0, T + 1, B) if step % 3 == 0 else rng.integers(0, 2, B) if step % 3 == 1 else rng.integers(0, 6, B)
        new = torch.from_numpy(np.where(left > 0, new, 0).astype(np.int32)).cuda()
        before = {k: w[k].cpu().numpy().copy() for k in ("table", "held", "free", "count", "kv_len")}
        cache = [w[k].cpu().numpy().copy() for k in ("cache_k", "cache_v", "k_scale", "v_scale")]
        cache[0], cache[1] = cache[0].view(np.uint8), cache[1].view(np.uint8)
        rows, settings = _rows(B, T, gen), _settings(B, gen)
        slots, granted, out, ids = _step(ops, w, new, rows, settings, bs, T)
        torch.cuda.synchronize()
        s_ref, g_ref, free = op.update_blocks(before["kv_len"], new.cpu().numpy(), before["table"], before["held"],
                                              before["free"], before["count"][0], bs, T)
        refused += int((g_ref < new.cpu().numpy()).sum())
        assert np.array_equal(slots.cpu().numpy(), s_ref) and np.array_equal(granted.cpu().numpy(), g_ref)
        assert np.array_equal(w["table"].cpu().numpy(), before["table"]) and int(w["count"]) == free
        q, gate, key, value = (x.double().cpu().numpy() for x in rows)
        kn, qn = w["k_norm"].double().cpu().numpy(), w["q_norm"].double().cpu().numpy()
        cos, sin = w["cos"].cpu().numpy(), w["sin"].cpu().numpy()
        op.kv_append(key, value, kn, cos, sin, before["kv_len"], s_ref, cache)
        assert np.array_equal(w["cache_v"].cpu().numpy().view(np.uint8), cache[1])
        k = w["cache_k"].cpu().numpy().view(np.uint8)
        assert np.abs((k & 0x7F).astype(int) - (cache[0] & 0x7F)).max() <= 1
        assert np.array_equal(w["k_scale"].cpu().numpy(), cache[2]) and np.array_equal(w["v_scale"].cpu().numpy(), cache[3])
        cache[0] = k  # the attention is checked on the bytes that it reads
        ref = op.tail_verify(q, gate, qn, cos, sin, cache, before["table"], before["kv_len"], g_ref)
        assert_rel_close(out.float().cpu().double().numpy(), ref, tol=2e-3, out_unit=BF16_U, name=f"step {step}")
        last = out[torch.arange(B), (granted - 1).clamp(min=0).long()].reshape(B, -1).float()
        want = osm.sample((last @ w["head"]).double().cpu().numpy(), *[x.cpu().numpy() for x in settings])
        assert np.array_equal(ids.cpu().numpy(), want)
        kept = (g_ref * rng.random(B) + 0.999).astype(np.int32).clip(0, g_ref)
        kv = before["kv_len"] + kept
        kv[rng.random(B) < 0.12] = 0
        w["kv_len"].copy_(torch.from_numpy(kv.astype(np.int32)))
    assert (refused > 0) == short


def test_captured_steps_equal_eager_ones(ops):
    """Two graphs of a step, on one state at fixed addresses, replayed in turn with other work and
    synchronisations between, against the same steps run eagerly on a copy of the state."""
    B, P, N, bs, T, V = 4, 40, 160, 16, 3, 5003
    gen = torch.Generator(device="cuda").manual_seed(6)
    a, b = _world(B, P, N, bs, V, seed=7), _world(B, P, N, bs, V, seed=7)
    inputs = [dict(new=torch.full((B,), T, dtype=I32, device="cuda"), rows=_rows(B, T, gen), settings=_settings(B, gen))
              for _ in range(2)]
    for w in (a, b):  # a few rows to begin with, and the library's first launches outside the capture
        _step(ops, w, inputs[0]["new"], inputs[0]["rows"], inputs[0]["settings"], bs, T)
        w["kv_len"] += 2
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = _step(ops, a, i["new"], i["rows"], i["settings"], bs, T)
            a["kv_len"] += 2
        graphs.append(g)
        outs.append(o)
    for n in range(40):
        i = inputs[n % 2]
        for x in i["rows"]:
            x.copy_(torch.randn(x.shape, generator=gen, device="cuda").to(BF))
        i["settings"][4].copy_(torch.rand(B, generator=gen, device="cuda"))
        graphs[n % 2].replay()
        torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")
        if n % 3 == 0:
            torch.cuda.synchronize()
        want = _step(ops, b, i["new"], i["rows"], i["settings"], bs, T)
        b["kv_len"] += 2
        torch.cuda.synchronize()
        for x, y in zip(outs[n % 2], want):
            assert torch.equal(x, y), n
        for k in ("table", "held", "count", "cache_k", "cache_v", "k_scale", "v_scale", "kv_len"):
            assert torch.equal(a[k], b[k]), (n, k)


def test_two_streams_at_once(ops):
    """The same calls on two streams with states of their own give what they give alone."""
    B, P, N, bs, T, V = 6, 30, 180, 32, 4, 20011
    gen = torch.Generator(device="cuda").manual_seed(8)
    new = torch.full((B,), T, dtype=I32, device="cuda")
    rows, settings = [_rows(B, T, gen) for _ in range(6)], [_settings(B, gen) for _ in range(6)]

    def run(w):
        got = []
        for r, s in zip(rows, settings):
            got.append(_step(ops, w, new, r, s, bs, T))
            w["kv_len"] += T
        return got

    alone = [run(_world(B, P, N, bs, V, seed=i)) for i in (9, 10)]
    worlds = [_world(B, P, N, bs, V, seed=i) for i in (9, 10)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in worlds]
    both = []
    for s, w in zip(streams, worlds):
        with torch.cuda.stream(s):
            both.append(run(w))
    torch.cuda.synchronize()
    for x, y in zip(alone, both):
        for a, b in zip(x, y):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_compiled_step_equals_eager(ops):
    """torch.compile(fullgraph=True) traces the step through the ops' fakes, in-place state included."""
    import torch._dynamo
    torch._dynamo.reset()
    B, P, N, bs, T, V = 3, 10, 30, 16, 2, 1009
    gen = torch.Generator(device="cuda").manual_seed(11)
    a, b = _world(B, P, N, bs, V, seed=12), _world(B, P, N, bs, V, seed=12)
    new, rows, settings = torch.full((B,), T, dtype=I32, device="cuda"), _rows(B, T, gen), _settings(B, gen)
    fn = lambda w: _step(torch.ops, w, new, rows, settings, bs, T)  # noqa: E731
    want, got = fn(a), torch.compile(fn, fullgraph=True, backend="aot_eager")(b)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("bs", [16, 64])
def test_verify_slice_with_a_paged_cache(bs):
    """The verify step over the paged cache: replays of its graphs equal eager steps bit for bit, the
    table holds what the lengths need and no block twice."""
    from spec_verify_step import HIDDEN, VerifySlice, synthetic_logits
    B, K, V, kv = 3, 3, 1000, [37, 300, 5]
    slices = [VerifySlice(B, K, kv, 512, pattern="DG", seed=1, paged_block=bs) for _ in range(2)]
    x = torch.randn(B * (K + 1), HIDDEN, device="cuda").to(BF)
    sets = [synthetic_logits(B, K, V, 20 + i, "cuda") for i in range(2)]
    for m in slices:
        m.step(x, *sets[0])
        m.make_persistent()
    eager, graph = slices
    graph.capture(x, sets)
    for n in range(10):
        x.copy_(torch.randn(x.shape, device="cuda").to(BF))
        want = eager.step(x, *sets[n % 2])
        got = graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n
        for k in ("table", "held", "free", "count"):
            assert torch.equal(eager.pages[k], graph.pages[k]), (n, k)
        for k in ("cache_k", "cache_v", "k_scale", "v_scale"):
            assert torch.equal(eager.layers[1][k], graph.layers[1][k]), (n, k)
        table, held = graph.pages["table"].cpu(), graph.pages["held"].cpu()
        ids = [i for b in range(B) for i in table[b, :held[b]].tolist()]
        ids += graph.pages["free"][:int(graph.pages["count"])].tolist()
        assert sorted(ids) == list(range(B * -(-512 // bs)))
    assert torch.equal(eager.kv_len, graph.kv_len)


@pytest.mark.parametrize("replayed", [False, True])
@pytest.mark.parametrize("s_max", [64, 72])
def test_verify_slice_stops_where_its_pages_end(s_max, replayed):
    """A step whose rows would pass s_max is refused before it runs, eager or replayed: every step that
    runs has all its rows granted, and the refused one changes nothing."""
    from spec_verify_step import HIDDEN, VerifySlice, synthetic_logits
    B, K, V = 2, 3, 500
    m = VerifySlice(B, K, [s_max - 12, 5], s_max, pattern="DG", seed=1, paged_block=16)
    x = torch.randn(B * (K + 1), HIDDEN, device="cuda").to(BF)
    sets = [synthetic_logits(B, K, V, 30 + i, "cuda") for i in range(2)]
    m.step(x, *sets[0])
    if replayed:
        m.capture(x, sets)
    for n in range(20):
        before = [m.kv_len.clone()] + [m.pages[k].clone() for k in ("table", "held", "free", "count")]
        full = int(m.kv_len.max()) + K + 1 > s_max
        if full:
            with pytest.raises(RuntimeError, match="s_max"):
                m.replay() if replayed else m.step(x, *sets[n % 2])
            torch.cuda.synchronize()
            after = [m.kv_len] + [m.pages[k] for k in ("table", "held", "free", "count")]
            assert all(torch.equal(a, b) for a, b in zip(before, after))
            break
        m.replay() if replayed else m.step(x, *sets[n % 2])
        assert torch.equal(m.pages["held"], (before[0] + K + 1 + 15) // 16)  # granted, which is to have its blocks
    assert full


def test_chunk_and_sampling_replayed_beside_each_other(ops):
    """A prompt chunk's attention captured in one graph and sampling in another, replayed on two streams
    at once with lengths, pages and settings that change in place, against eager calls."""
    from test_gpu_paged import _attend_inputs, _cuda_cache
    from test_gpu_sample import _settings
    T, V = 70, 30011
    inputs = [_attend_inputs(3, T, 2, 6, 32, kv, n, seed=5 + k, spare_pages=spare) for k, (kv, n, spare) in enumerate(
        [([300, 0, 77], [70, 70, 3], 30), ([0, 900, 0], [0, 70, 70], 6), ([5, 5, 640], [70, 1, 64], 25)])]
    N = min(len(d["cache"][0]) for d in inputs)
    P = max(d["table"].shape[1] for d in inputs)
    cases = []
    for d in inputs:
        assert d["table"].max() < len(d["cache"][0])
        table = np.full((3, P), -1, np.int32)
        table[:, :d["table"].shape[1]] = np.where(d["table"] < N, d["table"], -1)
        cases.append([d["query"].cuda(), d["gate"].cuda(), *(c[:N].clone() for c in _cuda_cache(d["cache"])),
                      *(torch.from_numpy(a).cuda() for a in (table, d["kv"], d["n"]))])
    cos, sin = (torch.from_numpy(np.ascontiguousarray(inputs[1][k])).float().cuda() for k in ("cos", "sin"))
    norm = inputs[0]["q_norm"].cuda()
    rng = np.random.default_rng(3)
    rows = []
    for _ in range(3):
        s = _settings(40, rng)
        rows.append([torch.randn(40, V, device="cuda")] + [torch.from_numpy(s[k]).cuda() for k in
                                                           ("temperature", "top_k", "top_p", "min_p", "u")])
    live, srow = [t.clone() for t in cases[0]], [t.clone() for t in rows[0]]
    attend = lambda c: ops.gqa.tail_verify_paged(c[0], c[1], norm, cos, sin, *c[2:])  # noqa: E731
    want = [(attend(c), ops.spec.sample(*r)) for c, r in zip(cases, rows)]
    torch.cuda.synchronize()
    ga, gs = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        out = attend(live)
    with torch.cuda.graph(gs):
        ids = ops.spec.sample(*srow)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for k in (0, 1, 2, 1, 0):
        for dst, src in zip(live + srow, cases[k] + rows[k]):
            dst.copy_(src)
        torch.cuda.synchronize()
        with torch.cuda.stream(one):
            ga.replay()
        with torch.cuda.stream(two):
            gs.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[k][0]) and torch.equal(ids, want[k][1])
