"""CPU restatement of the tree-verification ops in 64 bits (numpy), from the definitions of
include/npn_spec_verify.h. parent [B, T]: node t hangs on node parent[b, t] where that lies in [0, t), else on
the committed tokens alone. Every node is computed along its own line of ancestors."""
import numpy as np

from . import deltanet, fp8, paged
from .numerics import bf16_bits_to_f32

D = 128


def line(parent, t):
    """Node t's ancestors and itself, the first one first; parent [T]."""
    out = [t]
    while 0 <= parent[out[-1]] < out[-1]:
        out.append(int(parent[out[-1]]))
    return out[::-1]


def depths(parent):
    """[B, T]: how many ancestors each node has."""
    return np.array([[len(line(p, t)) - 1 for t in range(len(p))] for p in np.asarray(parent)])


# ---- DeltaNet ---------------------------------------------------------------------------------------

def deltanet_verify(d, parent, Hk, Hv):
    """d: the numpy arguments of oracle.deltanet.deltanet_verify. Returns (out [B, T, Hv, D], k [B, T, Hk, D],
    u [B, T, Hv, D], decay [B, T, Hv], states [B, T, Hv, D, D]), each node from the state and window of its parent."""
    state, mixed, conv, w, bias, a, b_, z, A_log, dt_bias, nw = d
    B, T = np.asarray(parent).shape
    g, beta = deltanet.gates(a, b_, A_log, dt_bias)
    out, us = np.zeros((2, B, T, Hv, D))
    ks, states = np.zeros((B, T, Hk, D)), np.zeros((B, T, Hv, D, D))
    for b in range(B):
        cs = bf16_bits_to_f32(conv[b]).astype(np.float64)
        x = bf16_bits_to_f32(mixed[b]).astype(np.float64)
        for t in range(T):
            mine = line(parent[b], t)
            window = np.concatenate([cs, x[mine].T], axis=1)[:, -4:]
            y = (window * w.astype(np.float64)).sum(-1) + bias.astype(np.float64)
            y = y / (1.0 + np.exp(-y))
            q, k, v = deltanet._split_qkv(y, Hk, Hv, D)
            ks[b, t] = deltanet.l2_normalize(k)
            q = np.repeat(deltanet.l2_normalize(q, 1.0 / np.sqrt(D)), Hv // Hk, axis=0)
            k = np.repeat(ks[b, t], Hv // Hk, axis=0)
            S = (states[b, mine[-2]] if len(mine) > 1 else np.asarray(state[b], np.float64))
            S = S * np.exp(g[b, t])[:, None, None]
            u = (v - np.einsum("hkv,hk->hv", S, k)) * beta[b, t][:, None]
            S = S + k[:, :, None] * u[:, None, :]
            us[b, t], states[b, t] = u, S
            out[b, t] = deltanet.gated_rms_norm(np.einsum("hkv,hk->hv", S, q), z[b, t], nw)
    return out, ks, us, np.exp(g), states


def path_length(path, T):
    n, before = 0, -1
    while n < T and before < path[n] < T:
        before = path[n]
        n += 1
    return n


def deltanet_commit(state, conv, mixed, k, u, decay, path):
    """state [B, Hv, D, D], conv [B, QKV, 3] bits, mixed [B, T, QKV] bits -> (state, conv) along the paths."""
    state, conv = np.asarray(state, np.float64).copy(), conv.copy()
    B, T = path.shape
    rep = state.shape[1] // k.shape[2]
    for b in range(B):
        for t in path[b, :path_length(path[b], T)]:
            key = np.repeat(k[b, t].astype(np.float64), rep, axis=0)
            state[b] = state[b] * decay[b, t].astype(np.float64)[:, None, None]
            state[b] += key[:, :, None] * u[b, t].astype(np.float64)[:, None, :]
            conv[b] = np.concatenate([conv[b, :, 1:], mixed[b, t][:, None]], axis=1)
    return state, conv


# ---- attention --------------------------------------------------------------------------------------

def kv_append(key, value, k_norm, cos_table, sin_table, kv_len, slots, parent, cache):
    """paged.kv_append with node t's rotation at kv_len + its number of ancestors, in place on the cache."""
    B, T = slots.shape
    pos = np.minimum(np.maximum(kv_len, 0)[:, None].astype(np.int64) + depths(parent), len(cos_table) - 1)
    # each request's own table of its nodes' rows
    for b in range(B):
        at = slice(b, b + 1)
        paged.kv_append(key[at], value[at], k_norm, cos_table[pos[b]], sin_table[pos[b]], np.zeros(1, np.int64),
                        slots[at], cache)


def tree_verify(query, gate, q_norm, cos_table, sin_table, cache, table, kv_len, q_len, parent):
    B, T, Hq, _ = query.shape
    H, bs = cache[0].shape[1], cache[0].shape[2]
    grp = Hq // H
    out = np.zeros(query.shape)
    for b in range(B):
        n, m = max(int(kv_len[b]), 0), min(max(int(q_len[b]), 0), T)
        cap = min(n + m, table.shape[1] * bs)
        for h in range(H):
            k, v, ok = paged.values(cache, table[b, :-(-cap // bs)], h, cap)
            for t in range(m):
                mine = line(parent[b], t)
                pos = min(n + len(mine) - 1, len(cos_table) - 1)
                q = paged.norm_rope(query[b, t, h * grp:(h + 1) * grp], q_norm, cos_table[pos].astype(np.float64),
                                    sin_table[pos].astype(np.float64))
                see = ok & (np.arange(cap) < n)
                at = np.array([n + s for s in mine if n + s < cap], int)
                see[at] = ok[at]
                if not see.any():
                    continue
                s = (q @ k[see].T) / 16.0
                e = np.exp(s - s.max(-1, keepdims=True))
                g = gate[b, t, h * grp:(h + 1) * grp].astype(np.float64)
                out[b, t, h * grp:(h + 1) * grp] = (e @ v[see]) / e.sum(-1, keepdims=True) / (1.0 + np.exp(-g))
    return out


# ---- the walk and the pages -------------------------------------------------------------------------

def accept(target, draft, parent, q_len):
    B, T = parent.shape
    accepted, path, ids = np.zeros(B, np.int32), np.full((B, T), -1, np.int32), np.full((B, T), -1, np.int64)
    for b in range(B):
        n, node, count = min(max(int(q_len[b]), 0), T), 0, 0
        while n > 0:
            path[b, count], ids[b, count] = node, target[b, node]
            count += 1
            after = [c for c in range(node + 1, n) if parent[b, c] == node and draft[b, c] == target[b, node] >= 0]
            if not after:
                break
            node = after[0]
        accepted[b] = count - 1
    return accepted, path, ids


def rows_in_place(slots, bs):
    """How many of a request's rows, from the first on, lie one behind the other, in a block to its end and from the
    next one's begin; slots [T]."""
    for t in range(1, len(slots)):
        last, at = int(slots[t - 1]), int(slots[t])
        if (last + 1) % bs != 0 if at % bs == 0 else at != last + 1:
            return t
    return len(slots)


def compact(path, slots, cache):
    """In place on one layer's (cache_k, cache_v, k_scale, v_scale)."""
    N, H, bs, _ = cache[0].shape
    B, T = path.shape
    inside = lambda s: 0 <= s < N * bs  # noqa: E731
    for b in range(B):
        n, rows_held = path_length(path[b], T), rows_in_place(slots[b], bs)
        for d in range(n):
            if path[b, d] >= rows_held or not (inside(slots[b, d]) and inside(slots[b, path[b, d]])):
                n = d
                break
        src, dst = [int(slots[b, p]) for p in path[b, :n]], [int(s) for s in slots[b, :n]]
        for page, scale, is_v in ((cache[0], cache[2], False), (cache[1], cache[3], True)):
            for h in range(H):
                rows = lambda blk: page[blk, h].T if is_v else page[blk, h]  # noqa: E731
                come = [(rows(s // bs)[s % bs].copy(), float(scale[s // bs, h])) for s in src]
                for blk in dict.fromkeys(s // bs for s in dst):
                    here = [d for d in range(n) if dst[d] // bs == blk]
                    old = now = float(scale[blk, h])
                    for d in here:
                        if src[d] != dst[d]:
                            x = np.abs(fp8.decode_e4m3fn(come[d][0]).astype(np.float64)) * come[d][1]
                            x = x[np.isfinite(x)]
                            if x.size and x.max() > 0:
                                now = max(now, paged.scale_of(x.max()))
                    into = rows(blk)
                    if now > old:
                        upto = max(dst[d] % bs for d in here) + 1
                        into[:upto] = paged.to_e4m3(fp8.decode_e4m3fn(into[:upto]).astype(np.float64) * (old / now))
                        scale[blk, h] = now
                    for d in here:
                        row, s = come[d]
                        if src[d] != dst[d]:
                            into[dst[d] % bs] = row if s == now else paged.to_e4m3(
                                fp8.decode_e4m3fn(row).astype(np.float64) * (s / now))
