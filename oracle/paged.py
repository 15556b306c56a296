"""CPU restatement of the paged 8-bit KV cache ops in 64 bits (numpy): the block tables' plan, the
e4m3 append and the attention over the pages. The definitions are those of
include/npn_spec_verify.h; a cache is (cache_k [N, Hkv, bs, 256] uint8, cache_v [N, Hkv, 256, bs]
uint8, k_scale [N, Hkv], v_scale [N, Hkv])."""
import numpy as np

from . import fp8, gqa

DH = 256
MIN_EXP = -100


def update_blocks(kv_len, new_len, table, held, stack, free, bs, T):
    """In place on table [B, P], held [B] and stack [N]; returns (slots [B, T], granted [B],
    free count)."""
    B, P = table.shape
    kv = [max(int(n), 0) for n in kv_len]
    new = [min(max(int(n), 0), T) for n in new_len]
    want = [-(-(n + m) // bs) for n, m in zip(kv, new)]
    free = min(max(int(free), 0), len(stack))
    had = [min(max(int(n), 0), P) for n in held]
    for b in range(B - 1, -1, -1):
        for j in range(had[b] - 1, want[b] - 1, -1):
            if free < len(stack):
                stack[free] = table[b, j]
            free = min(free + 1, len(stack))
            table[b, j] = -1
    slots = np.full((B, T), -1, np.int64)
    granted = np.zeros(B, np.int32)
    asked, left = 0, free
    for b in range(B):
        need = max(want[b] - had[b], 0) if want[b] <= P else 0
        asked += need
        ok = want[b] <= P and (need == 0 or asked <= free)
        held[b] = want[b] if ok else had[b]
        if not ok:
            continue
        for j in range(had[b], want[b]):
            left -= 1
            table[b, j] = stack[left]
        granted[b] = new[b]
        for t in range(new[b]):
            pos = kv[b] + t
            slots[b, t] = int(table[b, pos // bs]) * bs + pos % bs
    return slots, granted, left


def scale_of(amax):
    """The least power of two s >= 2^-100 with amax <= 448 s."""
    if amax == 0:
        return 2.0 ** MIN_EXP
    e = int(np.ceil(np.log2(amax / 448.0)))
    while amax > 448.0 * 2.0 ** e:
        e += 1
    while e > MIN_EXP and amax <= 448.0 * 2.0 ** (e - 1):
        e -= 1
    return 2.0 ** max(e, MIN_EXP)


def to_e4m3(x):
    """Nearest-even e4m3fn bytes of |x| <= 448 (NaN and infinities: 0x7F)."""
    x = np.asarray(x, np.float64)
    ok = np.isfinite(x)
    return np.where(ok, fp8.encode_e4m3fn(np.where(ok, x, 0.0)), np.uint8(0x7F))


def norm_rope(x, w, cos, sin):
    with np.errstate(all="ignore"):
        return gqa.rope_partial(gqa.rms_norm_1p(x, w), cos, sin)


def kv_append(key, value, k_norm, cos_table, sin_table, kv_len, slots, cache):
    """key, value [B, T, Hkv, 256] (values); in place on the cache's four arrays."""
    cache_k, cache_v, k_scale, v_scale = cache
    N, H, bs, _ = cache_k.shape
    B, T = slots.shape
    for b in range(B):
        pos = np.minimum(max(int(kv_len[b]), 0) + np.arange(T), len(cos_table) - 1)
        k = norm_rope(key[b], k_norm, cos_table[pos][:, None].astype(np.float64),
                      sin_table[pos][:, None].astype(np.float64))
        rows = {}
        for t in range(T):
            if 0 <= slots[b, t] < N * bs:
                rows.setdefault(int(slots[b, t]) // bs, []).append(t)
        for blk, ts in rows.items():
            off = [int(slots[b, t]) % bs for t in ts]
            for h in range(H):
                for x, page, scale in ((k[ts, h], cache_k[blk, h], k_scale),
                                       (value[b, ts, h].astype(np.float64), cache_v[blk, h].T, v_scale)):
                    fin = np.abs(x[np.isfinite(x)])
                    now = need = scale_of(fin.max() if fin.size else 0.0)
                    if off[0] > 0:
                        old = float(scale[blk, h])
                        now = max(old, need)
                        if now > old:
                            older = page[:off[0]]
                            val = fp8.decode_e4m3fn(older).astype(np.float64)
                            page[:off[0]] = to_e4m3(val * (old / now))
                    page[off] = to_e4m3(x / now)
                    scale[blk, h] = now


def values(cache, blocks, h, n):
    """K and V rows [n, 256] of the positions in `blocks` for head h; (K, V, which exist)."""
    cache_k, cache_v, k_scale, v_scale = cache
    N, _, bs, _ = cache_k.shape
    k, v, ok = np.zeros((len(blocks) * bs, DH)), np.zeros((len(blocks) * bs, DH)), []
    for j, blk in enumerate(blocks):
        there = 0 <= blk < N
        ok += [there] * bs
        if there:
            at = slice(j * bs, (j + 1) * bs)
            k[at] = fp8.decode_e4m3fn(cache_k[blk, h]).astype(np.float64) * float(k_scale[blk, h])
            v[at] = fp8.decode_e4m3fn(cache_v[blk, h]).astype(np.float64).T * float(v_scale[blk, h])
    return k[:n], v[:n], np.array(ok, bool)[:n]


def tail_verify(query, gate, q_norm, cos_table, sin_table, cache, table, kv_len, q_len):
    """query, gate [B, T, Hq, 256] values -> out [B, T, Hq, 256]."""
    B, T, Hq, _ = query.shape
    H, bs = cache[0].shape[1], cache[0].shape[2]
    grp = Hq // H
    out = np.zeros(query.shape)
    for b in range(B):
        n, m = max(int(kv_len[b]), 0), min(int(q_len[b]), T)
        cap = min(n + max(m, 0), table.shape[1] * bs)
        for t in range(max(m, 0)):
            pos = min(n + t, len(cos_table) - 1)
            q = norm_rope(query[b, t], q_norm, cos_table[pos].astype(np.float64),
                          sin_table[pos].astype(np.float64))
            seen = min(n + t + 1, cap)
            for h in range(H):
                k, v, ok = values(cache, table[b, :-(-seen // bs)], h, seen)
                if not ok.any():
                    continue
                s = (q[h * grp:(h + 1) * grp] @ k[ok].T) / 16.0
                e = np.exp(s - s.max(-1, keepdims=True))
                o = (e @ v[ok]) / e.sum(-1, keepdims=True)
                g = gate[b, t, h * grp:(h + 1) * grp].astype(np.float64)
                out[b, t, h * grp:(h + 1) * grp] = o / (1.0 + np.exp(-g))
    return out
