"""The paged-cache oracle (oracle/paged.py) against independent statements of the same things:
torch's e4m3fn cast, the dense verify attention's oracle, a block allocator's invariants; and the
host-side refusals of the paged entry points, which reach no GPU."""
import numpy as np
import pytest
import torch

from oracle import gqa as og, paged as op
from oracle.numerics import f32_to_bf16_bits, bf16_bits_to_f32


def test_to_e4m3_matches_torch():
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(4000) * np.exp2(rng.integers(-12, 8, 4000)),
                        np.arange(-448, 449, 0.5), np.arange(-64, 64) * 2.0 ** -11])
    x = np.clip(x, -448, 448).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(op.to_e4m3(x), want)
    assert op.to_e4m3([np.nan, np.inf, -np.inf]).tolist() == [0x7F] * 3


@pytest.mark.parametrize("amax,scale", [(448.0, 1.0), (448.0 * (1 + 2.0 ** -20), 2.0), (224.0, 0.5),
                                        (0.0, 2.0 ** -100), (1e-38, 2.0 ** -100), (1.0, 2.0 ** -8),
                                        (3.3e38, 2.0 ** 120)])
def test_scale_of(amax, scale):
    assert op.scale_of(amax) == scale


def test_update_blocks_keeps_every_block_once():
    """Random admissions, growth, refusals and releases over a small pool: every block is held by
    one request or free, a granted request's slots are its table's, and giving back what a call
    granted restores the stack."""
    rng = np.random.default_rng(1)
    B, P, N, bs, T = 7, 6, 20, 16, 40
    table = np.full((B, P), -1, np.int32)
    held = np.zeros(B, np.int32)
    stack = rng.permutation(N).astype(np.int32)
    free, kv = N, np.zeros(B, np.int32)
    refused = 0
    for step in range(200):
        new = rng.integers(0, T + 1, B).astype(np.int32)
        before = (table.copy(), held.copy(), stack.copy(), free)
        slots, granted, free = op.update_blocks(kv, new, table, held, stack, free, bs, T)
        if step % 3 == 0:
            _, _, free = op.update_blocks(kv, np.zeros(B, np.int32), table, held, stack, free, bs, T)
            assert free == before[3] and np.array_equal(stack[:free], before[2][:free])
            assert np.array_equal(table, before[0]) and np.array_equal(held, before[1])
            continue
        refused += int((granted < new).sum())
        ids = np.concatenate([table[b, :held[b]] for b in range(B)] + [stack[:free]])
        assert sorted(ids.tolist()) == list(range(N))
        for b in range(B):
            assert (table[b, held[b]:] == -1).all() and granted[b] in (0, new[b])
            pos = kv[b] + np.arange(granted[b])
            assert np.array_equal(slots[b, :granted[b]], table[b, pos // bs] * bs + pos % bs)
            assert (slots[b, granted[b]:] == -1).all()
        # accept part of the new rows; now and then a request ends
        kv = kv + (granted * rng.random(B)).astype(np.int32)
        done = rng.random(B) < 0.15
        kv[done] = 0
        _, _, free = op.update_blocks(kv, np.zeros(B, np.int32), table, held, stack, free, bs, T)
    assert refused > 50


def test_append_then_attend_matches_dense_oracle():
    """Rows appended in pieces to shuffled pages, attended over the table, against the dense verify
    oracle on the dequantised rows; the appended values stay within half an e4m3 step of what was
    appended (a step of 2^-3 relative, or 2^-9 of the block's scale below the normals)."""
    rng = np.random.default_rng(2)
    B, H, grp, bs, N, T = 2, 2, 3, 16, 9, 5
    cache = [np.zeros((N, H, bs, 256), np.uint8), np.zeros((N, H, 256, bs), np.uint8),
             np.zeros((N, H), np.float32), np.zeros((N, H), np.float32)]
    table = rng.permutation(N)[:8].reshape(B, 4).astype(np.int32)
    cos, sin = og.rope_cos_sin(np.arange(80))
    k_norm, q_norm = rng.standard_normal(256) * 0.1, rng.standard_normal(256) * 0.1
    kv = np.zeros(B, np.int64)
    dense = [np.zeros((B, H, 64, 256)), np.zeros((B, H, 64, 256))]
    for n in (16, 9, 13, 2):
        key, value = rng.standard_normal((2, B, n, H, 256)) * rng.uniform(0.2, 5)
        pos = kv[:, None] + np.arange(n)
        slots = np.take_along_axis(table, pos // bs, 1).astype(np.int64) * bs + pos % bs
        op.kv_append(key, value, k_norm, cos, sin, kv, slots, cache)
        for b in range(B):
            dense[0][b, :, pos[b]] = op.norm_rope(key[b], k_norm, cos[pos[b]][:, None], sin[pos[b]][:, None])
            dense[1][b, :, pos[b]] = value[b]
        kv = kv + n
    L = int(kv[0])
    for b in range(B):
        for h in range(H):
            k, v, ok = op.values(cache, table[b], h, L)
            assert ok.all()
            for got, want, sc in ((k, dense[0][b, h, :L], cache[2]), (v, dense[1][b, h, :L], cache[3])):
                step = np.repeat(sc[table[b], h], bs)[:L, None] * 2.0 ** -10
                assert (np.abs(got - want) <= np.abs(want) * 2.0 ** -4 + 2 * step).all()
            dense[0][b, h, :L], dense[1][b, h, :L] = k, v
    q, gate = (bf16_bits_to_f32(f32_to_bf16_bits(rng.standard_normal((B, T, H * grp, 256)).astype(np.float32)))
               for _ in range(2))
    got = op.tail_verify(q, gate, q_norm, cos, sin, cache, table, kv - T, np.full(B, T))
    pos = (kv - T)[:, None] + np.arange(T)
    bits = [f32_to_bf16_bits(x.astype(np.float32)) for x in (q, gate, *dense)]
    want = og.gqa_tail_verify(bits[0], bits[1], q_norm, cos[pos], sin[pos], bits[2], bits[3], kv - T)
    np.testing.assert_allclose(got, want, rtol=1e-10, atol=1e-12)
    part = op.tail_verify(q, gate, q_norm, cos, sin, cache, table, kv - T, np.array([2, 0]))
    assert np.array_equal(part[0, :2], got[0, :2]) and not part[0, 2:].any() and not part[1].any()


# ---- refusals on the host: no entry point reaches a launch with these ------------------------------

def _status(name, *args):
    import npn_native
    return getattr(npn_native.lib(), name)(*args)


ADDR = 1 << 20  # a 16-byte aligned address that is never read: every call below is refused first


def test_update_blocks_refusals():
    def st(ptrs=[ADDR] * 8, B=2, P=4, N=8, bs=16, T=1):
        return _status("npn_paged_update_blocks", *ptrs, B, P, N, bs, T, None)
    for i in range(8):
        assert st([0 if j == i else ADDR for j in range(8)]) == 1
    for bad in (dict(B=0), dict(B=65536), dict(P=0), dict(N=0), dict(bs=8), dict(bs=48), dict(bs=256),
                dict(T=0), dict(B=65535, T=1 << 16), dict(B=65535, P=1 << 16)):
        assert st(**bad) == 2, bad
    assert st([ADDR] * 6 + [ADDR + 8, ADDR]) == 3


def test_kv_append_paged_refusals():
    def st(ptrs=[ADDR] * 11, positions=10, B=2, T=1, H=4, N=8, bs=16):
        return _status("npn_gqa_kv_append_paged", *ptrs[:5], positions, *ptrs[5:], B, T, H, N, bs, None)
    for i in range(11):
        assert st([0 if j == i else ADDR for j in range(11)]) == 1
    for bad in (dict(positions=0), dict(B=0), dict(B=65536), dict(T=0), dict(H=0), dict(N=0), dict(bs=24),
                dict(T=(1 << 24) + 1)):
        assert st(**bad) == 2, bad
    for i in (0, 1, 2, 3, 4, 7, 8):
        assert st([ADDR + (2 if j == i else 0) for j in range(11)]) == 3, i


def test_tail_verify_paged_refusals():
    from npn_native import query

    def st(ptrs=[ADDR] * 13, positions=10, B=2, T=1, hq=24, H=4, N=8, P=4, bs=16, ws=ADDR, n=1 << 40):
        return _status("npn_gqa_tail_verify_paged", *ptrs[:5], positions, *ptrs[5:], B, T, hq, H, N, P, bs,
                       ws, n, None)
    for i in range(13):
        assert st([0 if j == i else ADDR for j in range(13)]) == 1
    for bad in (dict(positions=0), dict(B=0), dict(T=0), dict(hq=23), dict(hq=196), dict(H=0), dict(N=0),
                dict(P=0), dict(bs=20), dict(B=65536), dict(T=1 << 19), dict(P=1 << 27)):
        assert st(**bad) == 2, bad
    for i in (0, 1, 2, 3, 4, 5, 6, 12):
        assert st([ADDR + (2 if j == i else 0) for j in range(13)]) == 3, i
    n = query("npn_gqa_tail_verify_paged_workspace_size", 2, 1, 24, 4, 4, 16)
    assert n > 0 and st(n=n - 1) == 4 and st(ws=None) == 4
    assert query("npn_gqa_tail_verify_paged_workspace_size", 2, 1, 23, 4, 4, 16) == 0
    assert query("npn_gqa_tail_verify_paged_workspace_size", 2, 1, 24, 4, 4, 17) == 0


def test_ops_refuse_cpu_tensors_and_propagate_shapes():
    import npn_ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    i32, bf = torch.int32, torch.bfloat16
    with pytest.raises((NotImplementedError, RuntimeError)):
        z = torch.zeros(2, dtype=i32)
        torch.ops.paged.update_blocks_(z, z.clone(), torch.zeros(2, 4, dtype=i32), z.clone(),
                                       torch.zeros(8, dtype=i32), torch.zeros(1, dtype=i32), 16, 1)
    with FakeTensorMode():
        e = torch.empty
        B, T, H, N, bs, P = 3, 4, 2, 10, 32, 5
        s, g = torch.ops.paged.update_blocks_(e(B, dtype=i32), e(B, dtype=i32), e(B, P, dtype=i32),
                                              e(B, dtype=i32), e(N, dtype=i32), e(1, dtype=i32), bs, T)
        assert s.shape == (B, T) and s.dtype == torch.int64 and g.shape == (B,) and g.dtype == i32
        ck, cv = e(N, H, bs, 256, dtype=torch.int8), e(N, H, 256, bs, dtype=torch.int8)
        kv = e(B, T, H, 256, dtype=bf)
        assert torch.ops.gqa.kv_append_paged(kv, kv, e(256), e(50, 64), e(50, 64), e(B, dtype=i32), s, ck, cv,
                                             e(N, H), e(N, H)) is None
        q = e(B, T, 6 * H, 256, dtype=bf)
        o = torch.ops.gqa.tail_verify_paged(q, q, e(256), e(50, 64), e(50, 64), ck, cv, e(N, H), e(N, H),
                                            e(B, P, dtype=i32), e(B, dtype=i32), g)
        assert o.shape == q.shape and o.dtype == bf
