"""GPU parity of the paged e4m3 KV cache ops against the oracle (oracle/paged.py): block tables
bit for bit, appended pages byte for byte (V) or within one code where fp32 and 64 bits round a
normed K value apart, attention within its roundings.

Attention's tolerance: the kernel rounds q' to f16 relative to the row's largest element (at most
2^-11, 0.0002 in the root mean square), the softmax weights to f16 (2^-11 as well) and its output to
bf16, at most 2^-8 relative and 0.43 * 2^-8 = 0.0017 in the root mean square over a binade:
2e-3 in the norm, and for an element its own rounding (BF16_U) beside 2e-3 of the largest. Above
48 rows of a kv head q' has three e4m3 parts (2^-13 at most) and a weight three parts over its 32 keys'
largest (2^-13, or 2^-26 of that largest): less than f16's.
"""
import numpy as np
import pytest
import torch

from oracle import gqa as og, paged as op
from _util import BF16_U, assert_rel_close

pytestmark = pytest.mark.gpu
TOL = 2e-3
BF = torch.bfloat16


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


# ---- block tables -----------------------------------------------------------------------------------

def _state(B, P, N, rng):
    return dict(table=np.full((B, P), -1, np.int32), held=np.zeros(B, np.int32),
                stack=rng.permutation(N).astype(np.int32), free=N)


def _step(ops, s, d, kv, new, bs, T):
    """One call on the device state d and on the oracle's state s; everything compared."""
    got = ops.paged.update_blocks_(cuda(kv), cuda(new), d["table"], d["held"], d["stack"], d["free"], bs, T)
    slots, granted, s["free"] = op.update_blocks(kv, new, s["table"], s["held"], s["stack"], s["free"], bs, T)
    torch.cuda.synchronize()
    assert np.array_equal(got[1].cpu().numpy(), granted)
    assert np.array_equal(got[0].cpu().numpy(), slots)
    for k in ("table", "held", "stack"):
        assert np.array_equal(d[k].cpu().numpy(), s[k]), k
    assert int(d["free"]) == s["free"]
    return slots, granted


def _device(s):
    d = {k: cuda(v) for k, v in s.items() if k != "free"}
    d["free"] = torch.tensor([s["free"]], dtype=torch.int32, device="cuda")
    return d


@pytest.mark.parametrize("B,P,N,bs,T", [
    (1, 1, 1, 16, 1),          # the smallest pool
    (7, 6, 20, 16, 40),        # refusals
    (64, 40, 1200, 64, 8),     # a verify step's
    (3, 300, 500, 16, 4097),   # odd T: the slots' own launch, unaligned rows
    (1024, 4, 3000, 32, 5),    # one thread per request
    (1025, 4, 2500, 128, 3),   # requests in two groups
    (2500, 3, 5000, 16, 2),
])
def test_update_blocks(ops, B, P, N, bs, T):
    """A run of calls: random growth past the pool, ends of requests, and calls in which some
    requests give back while others are granted."""
    rng = np.random.default_rng(B + T)
    s = _state(B, P, N, rng)
    d = _device(s)
    kv = np.zeros(B, np.int32)
    for _ in range(6):
        new = rng.integers(0, T + 1, B).astype(np.int32)
        _, granted = _step(ops, s, d, kv, new, bs, T)
        kv = kv + (granted * rng.random(B)).astype(np.int32)
        kv[rng.random(B) < 0.2] = 0
    _step(ops, s, d, np.zeros(B, np.int32), np.zeros(B, np.int32), bs, T)
    assert s["free"] == N


def test_update_blocks_out_of_range_values(ops):
    """Negative lengths and counts count as 0, new_len past T as T, counts past the row or the pool
    as full; a request longer than its table row is refused without counting; the last free block
    goes to the first that needs one."""
    rng = np.random.default_rng(3)
    s = _state(6, 3, 8, rng)
    s["table"][:] = 7
    s["held"][:] = [-5, 0, 9, 0, 0, 0]
    s["free"] = 4
    d = _device(s)
    kv = np.array([-3, 100, 40, 0, 16, 2**31 - 1], np.int32)
    new = np.array([-1, 5, 8, 99, 1, 8], np.int32)
    _step(ops, s, d, kv, new, 16, 8)
    s["free"], d["free"] = 99, torch.tensor([99], dtype=torch.int32, device="cuda")
    _step(ops, s, d, kv, new, 16, 8)
    s["free"], d["free"] = -4, torch.tensor([-4], dtype=torch.int32, device="cuda")
    _step(ops, s, d, np.zeros(6, np.int32), new, 16, 8)


# ---- append ---------------------------------------------------------------------------------------------

def _empty_cache(N, H, bs, rng):
    """Pages of random bytes (NaN among them) and scales: what an append does not write must stay."""
    return [rng.integers(0, 256, (N, H, bs, 256)).astype(np.uint8),
            rng.integers(0, 256, (N, H, 256, bs)).astype(np.uint8),
            np.exp2(rng.integers(-9, -3, (N, H))).astype(np.float32),
            np.exp2(rng.integers(-9, -3, (N, H))).astype(np.float32)]


def _cuda_cache(c):
    return [cuda(c[0].view(np.int8)), cuda(c[1].view(np.int8)), cuda(c[2]), cuda(c[3])]


def _slots(kv, n, T, bs, N, rng):
    """Slots of n[b] rows at positions kv[b] + t in distinct random pages, -1 behind; (slots, table)."""
    B = len(kv)
    P = max(1, max(-(-(int(kv[b]) + int(n[b])) // bs) for b in range(B)))
    table = np.full((B, P), -1, np.int32)
    ids, slots = rng.permutation(N), np.full((B, T), -1, np.int64)
    used = 0
    for b in range(B):
        m = -(-(int(kv[b]) + int(n[b])) // bs)
        table[b, :m] = ids[used:used + m]
        used += m
        pos = int(kv[b]) + np.arange(int(n[b]))
        slots[b, :int(n[b])] = table[b, pos // bs].astype(np.int64) * bs + pos % bs
    return slots, table


def _same_cache(dev, ref):
    for name, got, want in (("k_scale", dev[2], ref[2]), ("v_scale", dev[3], ref[3])):
        assert np.array_equal(got.cpu().numpy(), want), name
    k, v = dev[0].cpu().numpy().view(np.uint8), dev[1].cpu().numpy().view(np.uint8)
    assert np.array_equal(v, ref[1]), f"{(v != ref[1]).sum()} V bytes differ"
    off = np.abs((k & 0x7F).astype(int) - (ref[0] & 0x7F))
    sign = (k ^ ref[0]) >> 7
    assert off.max() <= 1 and not (sign & ((k & 0x7F) > 0)).any()
    # fp32 norm and rotation are off by a few 2^-24 relative; a step is 2^-4 to 2^-3: codes differ
    # where a value lies that near a border, in one of some 10^5
    assert (off > 0).mean() <= 1e-3 + 2 / off.size


def _append(ops, key, value, k_norm, cos, sin, kv, slots, cache):
    ops.gqa.kv_append_paged(key, value, k_norm, cos, sin, kv, slots, *cache)


@pytest.mark.parametrize("bs,T,H,kv,n", [
    (16, 1, 4, [0, 1, 15, 16, 17], [1, 1, 1, 1, 1]),      # plain decode at every edge of a page
    (64, 8, 4, [60, 0, 57, 64], [8, 8, 8, 8]),            # verify rows that cross a page end
    (16, 8, 1, [5, 12, 16], [8, 0, 3]),                   # padded rows, an idle request
    (32, 3, 2, [31, 30], [3, 2]),
    (128, 300, 2, [5, 128], [300, 129]),                  # prompts over several pages
    (16, 65, 1, [3], [65]),
    (64, 129, 1, [0, 7], [129, 100]),
    (128, 20, 1, [100], [20]),
])
def test_kv_append_paged(ops, bs, T, H, kv, n):
    rng = np.random.default_rng(T + bs)
    B = len(kv)
    kv = np.array(kv, np.int32)
    N = sum(-(-(int(a) + int(b)) // bs) for a, b in zip(kv, n)) + 3
    slots, _ = _slots(kv, n, T, bs, N, rng)
    cache = _empty_cache(N, H, bs, rng)
    dev = _cuda_cache(cache)
    g = torch.Generator().manual_seed(T)
    key = (torch.randn(B, T, H, 256, generator=g) * 3).to(BF)
    value = (torch.randn(B, T, H, 256, generator=g) * torch.rand(B, T, H, 1, generator=g) * 9).to(BF)
    k_norm = torch.randn(256, generator=g) * 0.1
    cos, sin = og.rope_cos_sin(np.arange(int(kv.max()) + T - 1))  # one short: the last row clamps
    _append(ops, key.cuda(), value.cuda(), k_norm.cuda(), cuda(cos), cuda(sin), cuda(kv), cuda(slots), dev)
    torch.cuda.synchronize()
    op.kv_append(key.double().numpy(), value.double().numpy(), k_norm.double().numpy(), cos, sin, kv, slots,
                 cache)
    _same_cache(dev, cache)


def test_kv_append_paged_scale_grows_and_shrinks(ops):
    """Row after row into one page: tiny, zero, huge, then small values again (the scale stays),
    and a new first row, which sets the scale anew whatever the stale rows held."""
    rng = np.random.default_rng(5)
    H, bs, N = 2, 16, 3
    cache = _empty_cache(N, H, bs, rng)
    dev = _cuda_cache(cache)
    k_norm = np.zeros(256)
    cos, sin = og.rope_cos_sin(np.arange(64))
    seen = []
    for pos, size in ((0, 1e-3), (1, 0.0), (2, 1e-30), (3, 7.0), (4, 3e4), (5, 1e38), (6, 1.0), (0, 1e-3), (1, 2.0)):
        kv = np.array([pos], np.int32)
        key = torch.randn(1, 1, H, 256).to(BF)
        value = (torch.rand(1, 1, H, 256) * size).to(BF)
        slots = np.array([[bs + pos]], np.int64)
        _append(ops, key.cuda(), value.cuda(), cuda(k_norm.astype(np.float32)), cuda(cos), cuda(sin), cuda(kv),
                cuda(slots), dev)
        torch.cuda.synchronize()
        op.kv_append(key.double().numpy(), value.double().numpy(), k_norm, cos, sin, kv, slots, cache)
        _same_cache(dev, cache)
        seen.append(float(cache[3][1, 0]))
    assert seen[0] == seen[1] == seen[2] < seen[3] < seen[4] < seen[5] == seen[6] > seen[7] < seen[8]


def test_kv_append_paged_non_finite_and_foreign_slots(ops):
    """NaN and infinities become NaN bytes and leave the scale; slots past the pool or negative, and
    rows behind a break in a request's slots, are skipped."""
    rng = np.random.default_rng(6)
    H, bs, N, T = 1, 16, 4, 4
    cache = _empty_cache(N, H, bs, rng)
    dev = _cuda_cache(cache)
    key = torch.randn(4, T, H, 256).to(BF)
    value = torch.randn(4, T, H, 256).to(BF)
    value[0, 0, 0, 3], value[0, 1, 0, 4], value[0, 2, 0, 5] = float("nan"), float("inf"), -float("inf")
    value[1] = float("nan")
    key[0, 1, 0, 7] = float("nan")
    kv = np.array([3, 14, 0, 0], np.int32)
    slots = np.array([[3, 4, 5, 6], [30, 31, -1, -1], [N * bs, N * bs + 1, -1, -1], [-7, 50, 51, 52]], np.int64)
    cos, sin = og.rope_cos_sin(np.arange(64))
    z = torch.zeros(256)
    _append(ops, key.cuda(), value.cuda(), z.cuda(), cuda(cos), cuda(sin), cuda(kv), cuda(slots), dev)
    torch.cuda.synchronize()
    slots[3] = -1  # a request without a first slot appends nothing
    op.kv_append(key.double().numpy(), value.double().numpy(), z.double().numpy(), cos, sin, kv, slots, cache)
    _same_cache(dev, cache)


def test_kv_append_paged_rows_behind_a_block_that_is_none(ops):
    """A request's first block is none in its table: its rows there go nowhere, those in the blocks behind
    it are appended, as where a block's id is past the pool."""
    rng = np.random.default_rng(8)
    H, bs, N, T = 2, 16, 8, 40
    for none in (-1, N):
        for kv0 in (0, 5, 15):
            cache = _empty_cache(N, H, bs, rng)
            dev = _cuda_cache(cache)
            table = np.array([[none, 3, 1, 6], [none, none, 2, none]], np.int32)
            kv = np.array([kv0, kv0], np.int32)
            pos = kv[:, None] + np.arange(T)
            slots = np.take_along_axis(table, pos // bs, 1).astype(np.int64) * bs + pos % bs
            key, value = torch.randn(2, T, H, 256).to(BF), torch.randn(2, T, H, 256).to(BF)
            cos, sin = og.rope_cos_sin(np.arange(64))
            z = torch.zeros(256)
            _append(ops, key.cuda(), value.cuda(), z.cuda(), cuda(cos), cuda(sin), cuda(kv), cuda(slots), dev)
            torch.cuda.synchronize()
            op.kv_append(key.double().numpy(), value.double().numpy(), z.double().numpy(), cos, sin, kv, slots, cache)
            _same_cache(dev, cache)


def test_kv_append_paged_negative_length(ops):
    """A negative length counts as 0 here too, so that the rows that update_blocks_ places from position
    0 on are rotated by these positions."""
    rng = np.random.default_rng(9)
    H, bs, N, T = 1, 16, 3, 20
    slots = np.arange(T, dtype=np.int64)[None]
    key, value = torch.randn(1, T, H, 256).to(BF), torch.randn(1, T, H, 256).to(BF)
    cos, sin = og.rope_cos_sin(np.arange(64))
    z = torch.zeros(256)
    cache = _empty_cache(N, H, bs, rng)
    for kv in (-3, -2**31):
        dev = _cuda_cache(cache)
        kv = np.array([kv], np.int32)
        _append(ops, key.cuda(), value.cuda(), z.cuda(), cuda(cos), cuda(sin), cuda(kv), cuda(slots), dev)
        torch.cuda.synchronize()
        ref = [a.copy() for a in cache]
        op.kv_append(key.double().numpy(), value.double().numpy(), z.double().numpy(), cos, sin, np.zeros(1, np.int32),
                     slots, ref)
        _same_cache(dev, ref)


# ---- attention -----------------------------------------------------------------------------------------------

def _attend_inputs(B, T, H, grp, bs, kv, n, seed, spare_pages=2):
    rng = np.random.default_rng(seed)
    kv = np.array(kv, np.int32)
    N = sum(-(-(int(a) + int(b)) // bs) for a, b in zip(kv, n)) + spare_pages
    _, table = _slots(kv, n, T, bs, N, rng)
    # random finite e4m3 values up to 4 (code 0x48), in pages of different scales; and NaN wherever
    # no row may look: whole spare pages, and the rows behind each request's last
    code = lambda *s: (rng.integers(0, 0x49, s) | (rng.integers(0, 2, s) << 7)).astype(np.uint8)  # noqa: E731
    cache = [code(N, H, bs, 256), code(N, H, 256, bs),
             np.exp2(rng.integers(-2, 1, (N, H))).astype(np.float32),
             np.exp2(rng.integers(-3, 2, (N, H))).astype(np.float32)]
    used = set(table[table >= 0].tolist())
    for i in set(range(N)) - used:
        cache[0][i], cache[1][i], cache[2][i], cache[3][i] = 0x7F, 0xFF, np.nan, np.nan
    for b in range(B):
        end = int(kv[b]) + int(n[b])
        if end % bs and end:
            last = table[b, end // bs]
            cache[0][last, :, end % bs:], cache[1][last, :, :, end % bs:] = 0xFF, 0x7F
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    cos, sin = og.rope_cos_sin(np.arange(max(int(kv.max()) + T, 1)))
    return dict(query=r(B, T, H * grp, 256).to(BF), gate=r(B, T, H * grp, 256).to(BF), q_norm=r(256) * 0.1,
                cos=cos, sin=sin, cache=cache, table=table, kv=kv, n=np.array(n, np.int32))


def _attend(ops, d, dev=None):
    dev = dev or _cuda_cache(d["cache"])
    return ops.gqa.tail_verify_paged(d["query"].cuda(), d["gate"].cuda(), d["q_norm"].cuda(), cuda(d["cos"]),
                                     cuda(d["sin"]), *dev, cuda(d["table"]), cuda(d["kv"]), cuda(d["n"]))


def _oracle(d):
    return op.tail_verify(d["query"].double().numpy(), d["gate"].double().numpy(), d["q_norm"].double().numpy(),
                          d["cos"], d["sin"], d["cache"], d["table"], d["kv"], d["n"])


def _check(ops, d):
    out = _attend(ops, d)
    torch.cuda.synchronize()
    got, ref = out.float().cpu().double().numpy(), _oracle(d)
    assert_rel_close(got, ref, tol=TOL, out_unit=BF16_U, name="tail_verify_paged")
    for b, n in enumerate(d["n"]):
        assert not got[b, max(int(n), 0):].any()


@pytest.mark.parametrize("B,T,H,grp,bs,kv,n", [
    (1, 1, 1, 1, 16, [0], [1]),                         # one key, one head
    (1, 1, 1, 6, 64, [300], [1]),                       # one 16-row tile
    (3, 1, 4, 6, 16, [0, 63, 64], [1, 1, 1]),           # step ends
    (2, 8, 4, 6, 64, [37, 600], [8, 8]),                # three tiles
    (3, 8, 4, 6, 32, [0, 1, 2000], [8, 8, 8]),
    (4, 5, 2, 6, 128, [127, 128, 1500, 11], [5, 0, 3, 1]),  # two tiles, padded and idle requests
    (2, 4, 2, 4, 16, [100, 33], [4, 4]),
    (1, 7, 1, 48, 16, [50], [7]),                       # a token's heads fill a group: many groups
    (2, 33, 2, 6, 16, [70, 0], [33, 20]),               # a prompt's chunk: groups without a live token
    (1, 150, 1, 5, 64, [500], [150]),                   # tokens that straddle groups (48 rows, 5 heads)
])
def test_tail_verify_paged_matches_oracle(ops, B, T, H, grp, bs, kv, n):
    _check(ops, _attend_inputs(B, T, H, grp, bs, kv, n, seed=B * 7 + T))


def test_tail_verify_paged_ragged_batches(ops):
    """More pairs than workgroups, some without a step; then one long request among short ones, so
    that one pair has most workgroups."""
    rng = np.random.default_rng(41)
    kv, n = rng.integers(0, 301, 70), rng.integers(0, 4, 70)
    _check(ops, _attend_inputs(70, 3, 4, 6, 16, kv, n, seed=41))
    kv = rng.integers(0, 60, 40)
    kv[7] = 9000
    _check(ops, _attend_inputs(40, 5, 2, 6, 64, kv, [5] * 40, seed=43))


def test_tail_verify_paged_long(ops):
    """Chunks of pages beyond what a workgroup keeps in LDS at a time, alone and beside a neighbour."""
    _check(ops, _attend_inputs(1, 1, 1, 6, 16, [33000], [1], seed=2))
    _check(ops, _attend_inputs(2, 8, 4, 6, 128, [32768 - 8, 17000], [8, 8], seed=5))


def test_tail_verify_paged_more_requests_than_the_plan_keeps(ops):
    """4300 units, some without a step: the plan reads the lengths past its 4096 again."""
    rng = np.random.default_rng(4)
    kv, n = rng.integers(0, 50, 4300), rng.integers(0, 2, 4300)
    kv[4200] = 700
    _check(ops, _attend_inputs(4300, 1, 1, 2, 16, kv, n, seed=44))


def test_tail_verify_paged_all_idle(ops):
    d = _attend_inputs(3, 2, 2, 6, 16, [5, 0, 40], [0, 0, 0], seed=9)
    assert not _attend(ops, d).any()


def test_tail_verify_paged_missing_pages(ops):
    """Table entries that are none or past the pool hide their positions; a row with none left is 0,
    whatever its gate."""
    d = _attend_inputs(3, 3, 2, 6, 16, [40, 5, 100], [3, 3, 3], seed=10)
    d["table"][0, 1] = -1
    d["table"][1, 0] = len(d["cache"][0])
    d["table"][2, [0, 3, 6]] = [2**31 - 1, -2**31, -1]
    d["gate"][1] = float("nan")
    got, ref = _attend(ops, d).float().cpu().double().numpy(), None
    d["gate"][1] = 0
    ref = _oracle(d)
    assert not got[1].any()
    assert_rel_close(got, ref, tol=TOL, out_unit=BF16_U, name="missing pages")


@pytest.mark.parametrize("B,T,n", [(2, 1, [1, 1]), (2, 8, [8, 5]), (1, 40, [40])])
def test_tail_verify_paged_scales_far_apart(ops, B, T, n):
    """Value scales from 2^-100 to 2^20 among a request's pages, row by row against the oracle's row: a
    row's largest product of weight and scale may lie in any page.

    Keys' codes up to 0x48 have a root mean square of 1.17, |q'| is 16: over key scales of up to 8 a
    score, their product over 16, deviates by 9.4. Rounding q' to f16 (0.0002 relative in the root mean
    square) moves it by 0.0019, the difference of two keys' by 0.0027, and with it in full a row that
    lies in two keys. Of 480 rows with a few such pairs each the largest is near 3.5 deviations; four
    are 0.0108, with the output's own 0.0017 added 0.0125."""
    kv = [700, 131][:B]
    d = _attend_inputs(B, T, 2, 6, 16, kv, n, seed=77 + T)
    rng = np.random.default_rng(T)
    live = d["cache"][3][np.isfinite(d["cache"][3])]
    d["cache"][2][:] *= 8
    d["cache"][3][np.isfinite(d["cache"][3])] = np.exp2(rng.choice([-100, -60, -12, -3, 0, 5, 20], live.shape))
    got, ref = _attend(ops, d).float().cpu().double().numpy(), _oracle(d)
    err, size = np.linalg.norm(got - ref, axis=-1), np.linalg.norm(ref, axis=-1)
    for b in range(B):
        assert (size[b, :n[b]] > 0).all() and (err[b, :n[b]] <= 0.0125 * size[b, :n[b]]).all()


@pytest.mark.parametrize("where", ["k", "v"])
def test_tail_verify_paged_nan_stays_with_its_rows(ops, where):
    """A NaN among the new rows' keys or values reaches the rows that see it and no others."""
    B, T, H, grp, bs = 2, 6, 2, 6, 16
    d = _attend_inputs(B, T, H, grp, bs, [61, 30], [6, 6], seed=12)
    clean = _attend(ops, d)
    pos = 61 + 3
    page, row = d["table"][0, pos // bs], pos % bs
    if where == "k":
        d["cache"][0][page, 1, row, 17] = 0x7F
    else:
        d["cache"][1][page, 1, 17, row] = 0xFF
    got = _attend(ops, d)
    hit = torch.zeros_like(got, dtype=torch.bool)
    if where == "k":
        hit[0, 3:, grp:] = True
    else:
        hit[0, 3:, grp:, 17] = True
    assert torch.isnan(got[hit]).all()
    assert torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("B,T,H,grp,bs,kv,n", [
    (1, 9, 1, 6, 16, [0], [9]),                          # 54 rows, one step
    (3, 25, 2, 5, 128, [127, 128, 1000], [25, 0, 7]),    # 125 rows, idle and padded requests
    (2, 64, 1, 6, 32, [255, 2], [64, 63]),               # tokens that straddle groups of 128 rows
    (1, 3, 1, 43, 64, [513], [3]),                       # 129 rows
    (8, 40, 4, 6, 16, [0, 5, 100, 300, 700, 1100, 64, 128], [40, 39, 1, 40, 17, 40, 0, 22]),  # 64 pairs
    (5, 90, 4, 5, 16, [900, 0, 1500, 33, 260], [90, 90, 90, 90, 2]),  # 80 pairs: one round or two
    (33, 30, 2, 9, 32, [7 * k for k in range(33)], [30] * 33),        # 198: some pairs cut, some not
])
def test_tail_verify_paged_many_rows(ops, B, T, H, grp, bs, kv, n):
    _check(ops, _attend_inputs(B, T, H, grp, bs, kv, n, seed=B * 11 + T))


def test_tail_verify_paged_many_rows_long(ops):
    """Parts of more steps than a workgroup has pages of in LDS at a time; against the formula in 64-bit
    torch on the device, which decodes the pages once for all tokens."""
    T, H, grp, bs, kv = 340, 4, 6, 16, 17000
    d = _attend_inputs(1, T, H, grp, bs, [kv], [T], seed=3)
    f64 = lambda a: torch.as_tensor(a).cuda().double()  # noqa: E731
    e4m3 = lambda c: cuda(c).view(torch.float8_e4m3fn).double()  # noqa: E731
    table = cuda(d["table"][0]).long()
    k = (e4m3(d["cache"][0]) * f64(d["cache"][2])[..., None, None])[table].transpose(0, 1).reshape(H, -1, 256)
    v = (e4m3(d["cache"][1]) * f64(d["cache"][3])[..., None, None])[table].permute(1, 0, 3, 2).reshape(H, -1, 256)
    k, v = k[:, :kv + T].contiguous(), v[:, :kv + T].contiguous()
    q = f64(d["query"])[0]
    q = (1 + f64(d["q_norm"])) * q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6)
    cos, sin = (f64(d[n])[kv:kv + T, None] for n in ("cos", "sin"))
    rot = torch.cat([-q[..., 32:64], q[..., :32]], -1)
    q = torch.cat([q[..., :64] * cos + rot * sin, q[..., 64:]], -1)
    hidden = torch.arange(kv + T, device="cuda") > kv + torch.arange(T, device="cuda")[:, None]
    ref = torch.empty_like(q)
    for h in range(H * grp):
        s = (q[:, h] @ k[h // grp].t().contiguous() / 16).masked_fill(hidden, -torch.inf)
        ref[:, h] = torch.softmax(s, -1) @ v[h // grp]
    ref *= torch.sigmoid(f64(d["gate"])[0])
    assert_rel_close(_attend(ops, d)[0].double().cpu().numpy(), ref.cpu().numpy(), tol=TOL, out_unit=BF16_U)


@pytest.mark.parametrize("T", [8, 40])
@pytest.mark.parametrize("at", [0, 9001])
def test_tail_verify_paged_dominating_key(ops, T, at):
    """One key 11 to 18 nats above 16000 others that are all alike, its value 0: a row's output is what
    the small weights leave, row by row against the formula in 64 bits. As many pairs as leave each
    whole (T = 40), requests over the same pages.

    Beside the output's rounding (0.43 * 2^-8 = 0.0017 of a row in the root mean square, 0.0023 where all
    its elements lie at the bottom of a binade) such a row has, in full, the weights' rounding, alike for
    equal weights: 2^-11 in f16, 2^-13 in three parts. Those of the key's own 32 in the parts are off by
    up to 2^-3, 31 of 16000: 0.0002. And the key's score, at most 18 nats of 128 products of one sign, each
    with q's rounding of 0.0002: 18 * 0.0002 / (0.8 * sqrt(128)) = 0.0004, four deviations 0.0016. In all
    0.0046."""
    B, grp, bs, kv = 264, 6, 64, 16000 - 17
    S = kv + T
    P = -(-S // bs)
    g = torch.Generator().manual_seed(T + at)
    cache = [np.zeros((P, 1, bs, 256), np.uint8),
             torch.randint(0x30, 0x41, (P, 1, 256, bs), generator=g).numpy().astype(np.uint8),  # 0.5 to 2
             np.ones((P, 1), np.float32), np.exp2(np.arange(P) % 3).astype(np.float32).reshape(P, 1)]
    cache[0][at // bs, 0, at % bs, 128:] = 0x41  # 2.25
    cache[1][at // bs, 0, :, at % bs] = 0
    q = torch.randn(1, T, grp, 256, generator=g).abs().to(BF)
    gate = torch.randn(1, T, grp, 256, generator=g).to(BF)
    i32 = lambda v: torch.full((B,), v, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.arange(P, dtype=torch.int32, device="cuda").expand(B, P).contiguous()
    out = ops.gqa.tail_verify_paged(q.cuda().expand(B, -1, -1, -1).contiguous(),
                                    gate.cuda().expand(B, -1, -1, -1).contiguous(), torch.zeros(256).cuda(),
                                    *(cuda(a) for a in og.rope_cos_sin(np.arange(S))), *_cuda_cache(cache), table,
                                    i32(kv), i32(T))
    v = cuda(cache[1]).view(torch.float8_e4m3fn).double() * cuda(cache[3]).double()[..., None, None]
    v = v[:, 0].transpose(1, 2).reshape(-1, 256).cumsum(0)[kv:kv + T]  # up to each token's last key
    x = q[0].double()
    gap = (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6))[..., 128:].sum(-1) * 2.25 / 16  # [T, grp]
    assert 10 < gap.min() and gap.max() < 18
    z = torch.arange(kv, kv + T)[:, None] + gap.exp()
    ref = v.cpu()[:, None] / z[..., None] * torch.sigmoid(gate[0].double())
    for b in (0, B - 1):
        err = (out[b].cpu().double() - ref).norm(dim=-1) / ref.norm(dim=-1)
        assert err.max() <= 0.0046, float(err.max())


@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("at", [500, 503, 520])
def test_tail_verify_paged_many_rows_nan(ops, where, at):
    """Keys past the first token's: a NaN reaches the rows that see it and no others. Before it: all."""
    B, T, H, grp, bs = 2, 24, 2, 6, 16
    d = _attend_inputs(B, T, H, grp, bs, [501, 30], [22, 24], seed=15)
    clean = _attend(ops, d)
    page, row = d["table"][0, at // bs], at % bs
    if where == "k":
        d["cache"][0][page, 1, row, 17] = 0x7F
    else:
        d["cache"][1][page, 1, [17, 200], row] = 0xFF
        d["cache"][1][page, 1, 200, row - 1] = 0x7F
    got = _attend(ops, d)
    hit = torch.zeros_like(got, dtype=torch.bool)
    if where == "k":
        hit[0, max(at - 501, 0):22, grp:] = True
    else:
        hit[0, max(at - 501, 0):22, grp:, 17] = True
        hit[0, max(at - 502, 0):22, grp:, 200] = True
    assert torch.isnan(got[hit]).all()
    assert torch.equal(got[~hit], clean[~hit])


def test_tail_verify_paged_many_rows_missing_pages(ops):
    d = _attend_inputs(3, 30, 2, 6, 16, [400, 5, 700], [30, 30, 30], seed=16)
    d["table"][0, 1] = -1
    d["table"][1] = len(d["cache"][0])
    d["table"][2, [0, 3, 20, 44]] = [2**31 - 1, -2**31, -1, -1]
    d["gate"][1] = float("nan")
    got = _attend(ops, d).float().cpu().double().numpy()
    d["gate"][1] = 0
    assert not got[1].any()
    assert_rel_close(got, _oracle(d), tol=TOL, out_unit=BF16_U, name="missing pages")


@pytest.mark.parametrize("T", [1, 8, 30])
@pytest.mark.parametrize("which", [2, 3])
def test_tail_verify_paged_nan_scale(ops, T, which):
    """A page without a valid scale makes its head's rows that see it NaN, and no others."""
    d = _attend_inputs(2, T, 2, 6, 16, [100, 40], [T, T], seed=21)
    clean = _attend(ops, d)
    d["cache"][which][d["table"][0, 2], 1] = float("nan")
    got = _attend(ops, d)
    assert torch.isnan(got[0, :, 6:]).all()
    assert torch.equal(got[0, :, :6], clean[0, :, :6]) and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("T,grp,bs", [(8, 2, 16), (8, 4, 16), (8, 6, 16), (40, 6, 16), (40, 6, 64), (100, 2, 32)])
def test_tail_verify_paged_nan_scale_behind_the_first_rows(ops, which, T, grp, bs):
    """A page without a valid scale that only a request's later tokens reach: NaN from its first position
    on, and the tokens before it as they were, in every tile width."""
    kv = 2 * bs - 4
    d = _attend_inputs(2, T, 2, grp, bs, [kv, 40], [T, T], seed=23)
    clean = _attend(ops, d)
    d["cache"][which][d["table"][0, 2], 1] = float("nan")  # positions from 2 bs on: the tokens from 4 on
    got = _attend(ops, d)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[0, 4:, grp:] = True
    assert torch.isnan(got[hit]).all()
    assert torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("T", [1, 8, 40])
def test_tail_verify_paged_rotates_by_the_length_past_the_table(ops, T):
    """A length past what the table's row holds: all of the row's positions are seen, and the query's
    RoPE rows are those of its own position (clamped to the RoPE tables alone)."""
    d = _attend_inputs(2, T, 2, 6, 16, [70, 20], [T, T], seed=24)
    d["cos"], d["sin"] = og.rope_cos_sin(np.arange(70 + T - 1))  # the last token's clamps
    d["table"] = np.ascontiguousarray(d["table"][:, :3])  # 48 positions
    d["cache"][0] &= 0xF7  # finite bytes throughout
    d["cache"][1] &= 0xF7
    _check(ops, d)


def test_tail_verify_paged_equals_dense_op_in_values(ops):
    """The same positions through gqa::tail_verify's dense bf16 cache of the dequantised rows."""
    B, T, H, grp, bs = 2, 8, 4, 6, 32
    d = _attend_inputs(B, T, H, grp, bs, [100, 517], [8, 8], seed=14)
    S = 544
    k, v = torch.zeros(2, B, H, S, 256, dtype=BF)
    for b in range(B):
        for h in range(H):
            n = int(d["kv"][b]) + T
            kk, vv, _ = op.values(d["cache"], d["table"][b, :-(-n // bs)], h, n)
            k[b, h, :n], v[b, h, :n] = torch.from_numpy(kk).to(BF), torch.from_numpy(vv).to(BF)
    cos, sin = cuda(d["cos"]), cuda(d["sin"])
    at = cuda(d["kv"]).long()[:, None] + torch.arange(T, device="cuda")
    ref = ops.gqa.tail_verify(d["query"].cuda(), d["gate"].cuda(), d["q_norm"].cuda(), cos[at].contiguous(),
                              sin[at].contiguous(), k.cuda(), v.cuda(), cuda(d["kv"]))
    assert_rel_close(_attend(ops, d).float().cpu().numpy(), ref.float().cpu().numpy(), tol=TOL, out_unit=BF16_U)


def test_refusals(ops):
    d = _attend_inputs(1, 1, 1, 6, 16, [5], [1], seed=1)
    args = [d["query"].cuda(), d["gate"].cuda(), d["q_norm"].cuda(), cuda(d["cos"]), cuda(d["sin"]),
            *_cuda_cache(d["cache"]), cuda(d["table"]), cuda(d["kv"]), cuda(d["n"])]
    for i, bad, err in ((0, args[0].float(), TypeError), (1, args[1][:, :, :3], RuntimeError),
                        (5, args[5].float(), TypeError), (6, args[6].transpose(2, 3), RuntimeError),
                        (7, args[7][:1], RuntimeError), (9, args[9].long(), TypeError),
                        (10, args[10].cpu(), RuntimeError), (11, torch.cat([args[11]] * 2), RuntimeError)):
        with pytest.raises(err):
            ops.gqa.tail_verify_paged(*[bad if j == i else a for j, a in enumerate(args)])
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    plan = [i32(0), i32(1), i32(-1, -1).reshape(1, 2), i32(0), i32(0, 1), i32(2)]
    for bs, T in ((8, 1), (16, 0)):
        with pytest.raises(RuntimeError):
            ops.paged.update_blocks_(*plan, bs, T)
    with pytest.raises(TypeError):
        ops.paged.update_blocks_(plan[0].long(), *plan[1:], 16, 1)
    with pytest.raises(RuntimeError):
        ops.paged.update_blocks_(i32(0, 1), *plan[1:], 16, 1)


def test_update_blocks_refuses_sizes_past_the_limits(ops):
    """T past 32 bits: refused before anything is allocated, not taken modulo 2^32."""
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    plan = [i32(0), i32(1), i32(-1, -1).reshape(1, 2), i32(0), i32(0, 1), i32(2)]
    torch.cuda.reset_peak_memory_stats()  # of the tests before
    held = torch.cuda.memory_allocated()
    for T in (2**32 + 8, 2**31, 2**30 + 1):
        with pytest.raises(RuntimeError):
            ops.paged.update_blocks_(*plan, 16, T)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() < held + 2**33 and int(plan[3]) == 0


def test_refuses_gradients(ops):
    """No backward pass: inputs that require grad are refused unless gradients are off."""
    d = _attend_inputs(1, 2, 1, 6, 16, [20], [2], seed=22)
    q = d["query"].cuda().requires_grad_()
    args = (d["gate"].cuda(), d["q_norm"].cuda(), cuda(d["cos"]), cuda(d["sin"]), *_cuda_cache(d["cache"]),
            cuda(d["table"]), cuda(d["kv"]), cuda(d["n"]))
    with pytest.raises(RuntimeError, match="requires grad"):
        ops.gqa.tail_verify_paged(q, *args)
    with torch.no_grad():
        out = ops.gqa.tail_verify_paged(q, *args)
    assert not out.requires_grad and torch.equal(out, ops.gqa.tail_verify_paged(q.detach(), *args))
    r = torch.ones(2).cuda()
    with pytest.raises(RuntimeError, match="requires grad"):
        ops.spec.sample(torch.zeros(2, 9).cuda().requires_grad_(), r, r.int(), r, r, r)


def test_refuses_gradients_under_transforms(ops):
    """The same through torch.func, forward mode and compiled code; without a gradient of theirs these run."""
    import torch._dynamo
    torch._dynamo.reset()
    d = _attend_inputs(1, 2, 1, 6, 16, [20], [2], seed=22)
    q = d["query"].cuda()
    args = (d["gate"].cuda(), d["q_norm"].cuda(), cuda(d["cos"]), cuda(d["sin"]), *_cuda_cache(d["cache"]),
            cuda(d["table"]), cuda(d["kv"]), cuda(d["n"]))
    fn = lambda x: ops.gqa.tail_verify_paged(x, *args)  # noqa: E731
    want, compiled = fn(q), torch.compile(fn, fullgraph=True, backend="aot_eager")
    with pytest.raises(RuntimeError, match="requires grad"):
        torch.func.grad(lambda x: fn(x).float().sum())(q)
    with pytest.raises(RuntimeError, match="tangent"):
        torch.func.jvp(fn, (q,), (q,))
    with pytest.raises(Exception, match="requires grad"):
        compiled(q.clone().requires_grad_())
    assert torch.equal(compiled(q), want)
    w = torch.ones((), device="cuda")
    assert torch.equal(torch.func.grad(lambda x: (x * fn(q)).sum())(w), want.sum())
    with torch.inference_mode():
        assert torch.equal(fn(q), want) and torch.equal(fn(q.clone()), want)
    # an append counts as a write of the cache
    old = args[6]._version
    key = torch.randn(1, 2, 1, 256, device="cuda").to(BF)
    ops.gqa.kv_append_paged(key, key, *args[1:4], args[9], torch.full((1, 2), -1, device="cuda"), *args[4:8])
    assert args[6]._version > old


@pytest.mark.parametrize("T", [1, 8, 40])
def test_pages_past_32_bit_offsets(ops, T):
    """A pool of 5 GB for K and for V, of which the request holds the last blocks: the appended bytes and
    the attention over them are those of a pool with these blocks alone."""
    H, bs, N, held = 4, 128, 40000, 4
    g = torch.Generator(device="cuda").manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    kv = torch.tensor([held * bs - T - 3], dtype=torch.int32, device="cuda")
    n = torch.tensor([T], dtype=torch.int32, device="cuda")
    cos, sin = (cuda(a) for a in og.rope_cos_sin(np.arange(held * bs)))
    norm = r(256) * 0.1
    past = [r(1, held * bs - T - 3, H, 256).to(BF) for _ in range(2)]
    new = [r(1, T, H, 256).to(BF) for _ in range(2)]
    q, gate = r(1, T, 6 * H, 256).to(BF), r(1, T, 6 * H, 256).to(BF)
    outs, pages = [], []
    for blocks in (N, held):
        cache = (torch.zeros(blocks, H, bs, 256, dtype=torch.int8, device="cuda"),
                 torch.zeros(blocks, H, 256, bs, dtype=torch.int8, device="cuda"),
                 torch.ones(blocks, H, device="cuda"), torch.ones(blocks, H, device="cuda"))
        table = torch.arange(blocks - held, blocks, dtype=torch.int32, device="cuda")[None]
        slots = (blocks - held) * bs + torch.arange(held * bs, device="cuda")[None]
        ops.gqa.kv_append_paged(*past, norm, cos, sin, torch.zeros_like(kv), slots[:, :-T - 3].contiguous(), *cache)
        ops.gqa.kv_append_paged(*new, norm, cos, sin, kv, slots[:, -T - 3:-3].contiguous(), *cache)
        outs.append(ops.gqa.tail_verify_paged(q, gate, norm, cos, sin, *cache, table, kv, n))
        pages.append([c[-held:].clone() for c in cache])
        assert not cache[0][:-held].any() and not cache[1][:-held].any()
    assert all(torch.equal(a, b) for a, b in zip(*pages))
    assert torch.equal(*outs) and outs[0].isfinite().all() and outs[0].any()
