"""The operators that verify a tree of drafted tokens: what is measured of them, in plain torch and by
the kernels.

A tree has T <= 64 nodes a request, node 0 the last committed token, the others drafts behind their
parent (parent [B, T]). Verifying one runs the target model over all nodes at once, each seeing the
committed tokens and its own ancestors, walks the tree by the target's tokens and commits the path.
Kinds of cases:

  attend   the attention layer: the nodes' K/V rows into the paged e4m3 cache, and attention of each
           node over the committed rows and its ancestors (gqa::tree_verify_paged)
  recur    the gated DeltaNet layer: every node's output from the committed state along its own
           ancestors, and the rows to commit from (deltanet::verify_tree)
  accept   the walk (spec::accept_tree)
  commit   the DeltaNet layers' states and conv windows moved along the path (deltanet::commit_tree_)
  compact  the path's K/V rows moved to the front of the tree's in all layers (gqa::compact_paged_)

Cache pages: cache_k [N, Hkv, bs, 256] and cache_v [N, Hkv, 256, bs] e4m3fn bytes, one power-of-two
scale per block and head each; attention heads of 256 with a 64-dim partial RoPE, DeltaNet heads of 128.
`own` selects the framework's kernels; the plain form is elementary torch in 32 bits, in 64 for the
sums of decays.
"""
import math

import torch

own = False

DEV = "cuda"
DH, ROPE, THETA, EPS = 256, 64, 1e7, 1e-6
D = 128
E4M3, BF, F32, F64 = torch.float8_e4m3fn, torch.bfloat16, torch.float32, torch.float64
I32, I64 = torch.int32, torch.int64
MAX_E4M3, MIN_EXP = 448.0, -100


def listed():
    return [
        # one user's long conversation, a small tree
        {"name": "attend_b1_t16", "kind": "attend", "B": 1, "T": 16, "reach": 4, "q_lo": 16, "hkv": 4,
         "grp": 6, "bs": 64, "kv_lo": 32768, "kv_hi": 32768},
        # a serving batch of mixed lengths, trees as small as a chain's verify step, small pages
        {"name": "attend_b32_t8", "kind": "attend", "B": 32, "T": 8, "reach": 3, "q_lo": 4, "hkv": 4,
         "grp": 6, "bs": 16, "kv_lo": 100, "kv_hi": 16384},
        # large trees
        {"name": "attend_b16_t64", "kind": "attend", "B": 16, "T": 64, "reach": 16, "q_lo": 64, "hkv": 4,
         "grp": 6, "bs": 64, "kv_lo": 1024, "kv_hi": 8192},
        # one user
        {"name": "recur_b1_t16", "kind": "recur", "B": 1, "T": 16, "reach": 4, "hk": 16, "hv": 48},
        # a serving batch
        {"name": "recur_b32_t16", "kind": "recur", "B": 32, "T": 16, "reach": 4, "hk": 16, "hv": 48},
        # large trees
        {"name": "recur_b8_t64", "kind": "recur", "B": 8, "T": 64, "reach": 16, "hk": 16, "hv": 48},
        # one user, and a large batch of large trees
        {"name": "accept_b1_t16", "kind": "accept", "B": 1, "T": 16, "reach": 4, "q_lo": 16},
        {"name": "accept_b256_t64", "kind": "accept", "B": 256, "T": 64, "reach": 16, "q_lo": 0},
        # all 48 DeltaNet layers of one user's model
        {"name": "commit_b1_l48", "kind": "commit", "L": 48, "B": 1, "T": 16, "reach": 4, "hk": 16, "hv": 48},
        # the three DeltaNet layers of a slice, a serving batch
        {"name": "commit_b32_l3", "kind": "commit", "L": 3, "B": 32, "T": 16, "reach": 4, "hk": 16, "hv": 48},
        # the attention layer of a slice, one user
        {"name": "compact_b1_l1", "kind": "compact", "L": 1, "B": 1, "T": 16, "reach": 4, "hkv": 4, "bs": 64},
        # all 16 attention layers, a serving batch of large trees over small pages
        {"name": "compact_b64_l16", "kind": "compact", "L": 16, "B": 64, "T": 64, "reach": 16, "hkv": 4,
         "bs": 16},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "recur", "recur", "accept", "commit", "compact"])
    T = _log_int(rng, 1, 64)
    # 1: a chain; T: bushes
    reach = _log_int(rng, 1, T)
    c = {"kind": kind, "T": T, "reach": reach}
    if kind == "attend":
        c["hkv"], c["grp"] = rng.choice([(1, 6), (2, 4), (4, 6), (1, 8)])
        c["bs"] = rng.choice([16, 32, 64, 128])
        c["B"] = _log_int(rng, 1, min(64, 1024 // (T * c["grp"] // 24 + 1)))
        hi = min(32768, 1000000 // (c["B"] * c["hkv"]), 100000000 // (c["B"] * c["hkv"] * c["grp"] * T))
        hi = _log_int(rng, 16, hi)
        # q_lo 0: some requests sit out
        return {**c, "q_lo": rng.choice([0, T // 2, T]), "kv_lo": rng.choice([0, hi // 8, hi]), "kv_hi": hi}
    if kind == "accept":
        return {**c, "B": _log_int(rng, 1, 256), "q_lo": rng.choice([0, T // 2, T])}
    if kind == "compact":
        return {**c, "L": _log_int(rng, 1, 16), "B": _log_int(rng, 1, 64), "hkv": rng.choice([1, 2, 4]),
                "bs": rng.choice([16, 32, 64, 128])}
    c["hk"], c["hv"] = rng.choice([(16, 48), (16, 32), (4, 12), (2, 6), (3, 3), (1, 5)])
    if kind == "recur":
        return {**c, "B": _log_int(rng, 1, max(1, 24576 // (c["hv"] * max(T, 16))))}
    c["L"] = _log_int(rng, 1, 48)
    return {**c, "B": _log_int(rng, 1, max(1, 4608 // (c["hv"] * c["L"])))}


# ---- inputs ---------------------------------------------------------------------------------

def _lens(lo, hi, n):
    """n lengths spread evenly over [lo, hi]; which request has which comes from the seed."""
    return [lo + (hi - lo) * (2 * i + 1) // (2 * n) for i in range(n)]


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen, device=DEV)
    return torch.tensor(values, dtype=I32, device=DEV)[order]


def _trees(B, T, reach, gen):
    """parent [B, T]: each node's among the `reach` nodes before it."""
    t = torch.arange(T, device=DEV)
    lo = (t - reach).clamp(min=0)
    parent = lo + (torch.rand(B, T, generator=gen, device=DEV) * (t - lo)).long()
    return torch.where(t > 0, torch.minimum(parent, (t - 1).clamp(min=0)), -1).int()


def _ancestors(parent):
    """[B, T, T] truth values: s is t or one of t's ancestors."""
    T = parent.shape[1]
    eye = torch.eye(T, device=DEV)
    step = (parent[:, :, None] == torch.arange(T, device=DEV)).float() + eye
    return torch.linalg.matrix_power(step, max(T - 1, 1)) > 0


def _path(on):
    """Nodes of the truth values [B, T] in order, -1 behind."""
    T = on.shape[1]
    order = torch.where(on, torch.arange(T, device=DEV), T).sort(-1).values
    return torch.where(order < T, order, -1).int()


def _tables(positions):
    inv = THETA ** (-torch.arange(0, ROPE, 2, device=DEV, dtype=F64) / ROPE)
    ang = torch.arange(positions, device=DEV, dtype=F64)[:, None] * inv
    ang = torch.cat([ang, ang], -1)
    return ang.cos().float(), ang.sin().float()


def _paged(total, bs, gen):
    """Distinct random pages for `total` [B] tokens each: (table [B, P] with -1 behind, N)."""
    need = (total.long() + bs - 1) // bs
    P = max(1, int(need.max()))
    held = torch.arange(P, device=DEV)[None] < need[:, None]
    N = max(1, int(need.sum()))
    ids = torch.full((len(need), P), -1, dtype=I32, device=DEV)
    ids[held] = torch.randperm(N, generator=gen, device=DEV)[:int(need.sum())].int()
    return ids, N


def _pages(N, hkv, bs, gen, value):
    """Random e4m3 pages and their scales, as appends of N(0, 1) rows leave them."""
    shape = (N, hkv, DH, bs) if value else (N, hkv, bs, DH)
    cache = torch.empty(shape, dtype=torch.int8, device=DEV)
    scale = torch.empty(N, hkv, device=DEV)
    for i in range(0, N, 1024):
        x = torch.randn(cache[i:i + 1024].shape, generator=gen, device=DEV)
        scale[i:i + 1024] = _scale_of(x.abs().amax((-2, -1)))
        cache[i:i + 1024] = (x / scale[i:i + 1024, :, None, None]).to(E4M3).view(torch.int8)
    return cache, scale


def _slots(table, at, live, bs):
    """Slots of the positions `at` [B, T] where `live`, -1 elsewhere."""
    P = table.shape[1]
    slots = table.long().gather(1, (at // bs).clamp(max=P - 1)) * bs + at % bs
    return torch.where(live, slots, -1)


def _some_path(parent, gen):
    """A path from node 0 to one of the later nodes, as an accepted one."""
    B, T = parent.shape
    last = (T // 2 + torch.rand(B, generator=gen, device=DEV) * (T - T // 2)).long().clamp(max=T - 1)
    return _path(_ancestors(parent)[torch.arange(B, device=DEV), last])


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *n: torch.randn(*n, generator=gen, device=DEV)  # noqa: E731
    s = dict(case)
    kind, B, T = case["kind"], case["B"], case["T"]
    s["parent"] = _trees(B, T, case["reach"], gen)
    t = torch.arange(T, device=DEV)
    if kind in ("attend", "accept"):
        s["q_len"] = _shuffled(_lens(case["q_lo"], T, B), gen)

    if kind == "accept":
        # the target's token is the draft of one of the node's children in three of four
        s["draft_ids"] = torch.randint(0, 151936, (B, T), generator=gen, device=DEV)
        other = torch.randint(0, 151936, (B, T), generator=gen, device=DEV)
        child = s["parent"][:, None, :] == t[:, None]
        pick = (child * (0.1 + torch.rand(B, T, T, generator=gen, device=DEV))).argmax(-1)
        hit = child.any(-1) & (torch.rand(B, T, generator=gen, device=DEV) < 0.75)
        s["target_ids"] = torch.where(hit, s["draft_ids"].gather(1, pick), other)
        return s

    if kind in ("recur", "commit"):
        hk, hv, L = case["hk"], case["hv"], case.get("L", 1)
        qkv = (2 * hk + hv) * D
        s["state"] = rnd(L, B * hv * D, D) * 0.1
        s["mixed_qkv"] = rnd(L, B * T * qkv).to(BF)
        s["conv_state"] = rnd(L, B * qkv, 3).to(BF)
        if kind == "recur":
            for k in ("state", "mixed_qkv", "conv_state"):
                s[k] = s[k][0]
            s["conv_weight"], s["conv_bias"] = rnd(qkv, 4) * 0.5, rnd(qkv) * 0.1
            s["a_out"], s["b_out"], s["z"] = rnd(B * T * hv), rnd(B * T * hv), rnd(B * T * hv, D).to(BF)
            s["A_log"], s["dt_bias"] = rnd(hv) * 0.5, rnd(hv)
            s["norm_weight"] = 1 + 0.1 * rnd(D)
            return s
        # what a verify leaves: unit keys, rows u, decays below 1
        k = rnd(L, B, T, hk, D)
        k = k / k.square().sum(-1, keepdim=True).sqrt()
        decay = torch.exp(-torch.log1p(torch.exp(rnd(L, B, T, hv))))
        s["records"] = torch.cat([k.reshape(L, -1), rnd(L, B * T * hv * D) * 0.5, decay.reshape(L, -1)], 1)
        s["path"] = _some_path(s["parent"], gen)
        for k in ("state", "conv_state", "mixed_qkv", "records"):
            s[k + "s"] = list(s[k].unbind())
        return s

    hkv, bs = case["hkv"], case["bs"]
    if kind == "compact":
        # the trees' own pages, the first of them begun by older rows
        L = case["L"]
        off = _shuffled(_lens(0, bs - 1, B), gen)
        table, N = _paged(off + T, bs, gen)
        at = off.long()[:, None] + t
        s["slots"] = _slots(table, at, torch.ones_like(at, dtype=torch.bool), bs)
        s["path"] = _some_path(s["parent"], gen)
        for name, value in (("k", False), ("v", True)):
            cache, scale = _pages(L * N, hkv, bs, gen, value)
            # some layers' pages have larger values than their neighbours
            scale *= torch.exp2(torch.randint(-1, 2, scale.shape, generator=gen, device=DEV).float())
            s["cache_" + name] = cache.view(L, N, *cache.shape[1:])
            s[name + "_scale"] = scale.view(L, N, hkv)
        for k in ("cache_k", "cache_v", "k_scale", "v_scale"):
            s[k + "s"] = list(s[k].unbind())
        return s

    kv = _shuffled(_lens(case["kv_lo"], case["kv_hi"], B), gen)
    s["kv_len"] = kv
    s["cos"], s["sin"] = _tables(case["kv_hi"] + T)
    s["block_table"], N = _paged(kv + T, bs, gen)  # the pool does not depend on who drafts how much
    s["slots"] = _slots(s["block_table"], kv.long()[:, None] + t, t < s["q_len"][:, None], bs)
    hq = hkv * case["grp"]
    s["query"], s["gate"] = rnd(B, T, hq, DH).to(BF), rnd(B, T, hq, DH).to(BF)
    s["key"], s["value"] = rnd(B, T, hkv, DH).to(BF), rnd(B, T, hkv, DH).to(BF)
    s["q_norm"], s["k_norm"] = rnd(DH) * 0.1, rnd(DH) * 0.1
    s["cache_k"], s["k_scale"] = _pages(N, hkv, bs, gen, False)
    s["cache_v"], s["v_scale"] = _pages(N, hkv, bs, gen, True)
    return s


# ---- the plain forms --------------------------------------------------------------------------

def _scale_of(amax):
    """The smallest 2^e >= amax / 448, e >= -100 (448 = 0.875 * 2^9; frexp's fraction is exact)."""
    f, e = torch.frexp(amax)
    e = torch.where(f <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, MIN_EXP).clamp(min=MIN_EXP)
    return ((e + 127) << 23).view(F32)


def _e4m3(x):
    x = torch.where(x.isfinite(), x.clamp(-MAX_E4M3, MAX_E4M3), math.nan)
    return x.to(E4M3).view(torch.int8)


def _norm_rope(x, w, cos, sin):
    """(1 + w) RMSNorm over the last axis and the rotation of dims [0, 64); cos, sin [.., 64]."""
    x = (1 + w) * (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS))
    a, b, rest = x.split([ROPE // 2, ROPE // 2, DH - ROPE], -1)
    rot = torch.cat([a, b], -1) * cos + torch.cat([-b, a], -1) * sin
    return torch.cat([rot, rest], -1)


def _append(s, k, v):
    """Rows k, v [B, T, Hkv, 256] (f32) into the pages of their slots."""
    bs, slots = s["bs"], s["slots"]
    ok = slots >= 0
    blk, off = slots[ok] // bs, slots[ok] % bs
    N, hkv = s["k_scale"].shape
    first = torch.full((N,), bs, device=DEV).scatter_reduce(0, blk, off, "amin")
    head = slots[:, 0][ok[:, 0]] // bs  # only a request's first page holds older rows
    older = torch.arange(bs, device=DEV) < first[head][:, None]

    def into(x, cache, scale, rows_last):
        size = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
        amax = torch.zeros(N, hkv, device=DEV).scatter_reduce(0, blk[:, None].expand(-1, hkv), size, "amax")
        need = _scale_of(amax)
        grown = torch.where((first > 0)[:, None], torch.maximum(scale, need), need)
        grown = torch.where((first < bs)[:, None], grown, scale)
        page = cache[head]
        by = (scale[head] / grown[head])[:, :, None, None]
        mask = (older[:, None, None, :] if rows_last else older[:, None, :, None]) & (by != 1)
        cache[head] = torch.where(mask, _e4m3(page.view(E4M3).float() * by), page)
        scale.copy_(grown)
        q = _e4m3(x / grown[blk][:, :, None])
        if rows_last:
            cache[blk, :, :, off] = q
        else:
            cache[blk, :, off] = q

    into(k[ok], s["cache_k"], s["k_scale"], False)
    into(v[ok], s["cache_v"], s["v_scale"], True)


def _plain_attend(s):
    B, T, hq, _ = s["query"].shape
    table, bs = s["block_table"].long(), s["bs"]
    (N, hkv), P = s["k_scale"].shape, table.shape[1]
    grp, S = hq // hkv, P * bs
    kv = s["kv_len"].long()
    anc = _ancestors(s["parent"])
    at = (kv[:, None] + anc.sum(-1) - 1).clamp(max=s["cos"].shape[0] - 1)
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    _append(s, _norm_rope(s["key"].float(), s["k_norm"], cos, sin), s["value"].float())
    page = table.clamp(min=0)
    q = _norm_rope(s["query"].float(), s["q_norm"], cos, sin) / 16.0
    q = q.view(B, T, hkv, grp, DH).transpose(1, 2).reshape(B, hkv, T * grp, DH)
    k = s["cache_k"][page].view(E4M3).float() * s["k_scale"][page][..., None, None]
    k = k.transpose(1, 2).reshape(B, hkv, S, DH)
    score = (q @ k.transpose(-1, -2)).view(B, hkv, T, grp, S)
    del k
    node = torch.arange(S, device=DEV) - kv[:, None]  # of a position; negative: committed
    of = node.clamp(0, T - 1)[:, None].expand(-1, T, -1)
    seen = (node < 0)[:, None] | (anc.gather(2, of) & (node < T)[:, None])
    score = torch.where(seen[:, None, :, None], score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    del score
    v = s["cache_v"][page].view(E4M3).float() * s["v_scale"][page][..., None, None]
    v = v.permute(0, 2, 1, 4, 3).reshape(B, hkv, S, DH)
    o = (p.view(B, hkv, T * grp, S) @ v).view(B, hkv, T, grp, DH).transpose(1, 2).reshape(B, T, hq, DH)
    o = o / (1 + torch.exp(-s["gate"].float()))
    live = torch.arange(T, device=DEV) < s["q_len"][:, None]
    return torch.where(live[:, :, None, None], o, 0.0).to(BF)


def _plain_recur(s):
    B, T, hk, hv = s["B"], s["T"], s["hk"], s["hv"]
    qkv, grp = (2 * hk + hv) * D, hv // hk
    parent = s["parent"].long()
    anc = _ancestors(s["parent"])
    # the conv's window: positions 0..2 are the committed inputs', 3 + t is node t's
    x = torch.cat([s["conv_state"].float().view(B, qkv, 3).transpose(1, 2),
                   s["mixed_qkv"].float().view(B, T, qkv)], 1)
    up = torch.cat([parent.new_tensor([[0, 0, 1]]).expand(B, -1), torch.where(parent < 0, 2, parent + 3)], 1)
    e0 = torch.arange(3, 3 + T, device=DEV).expand(B, -1)
    e1 = up.gather(1, e0)
    e2 = up.gather(1, e1)
    e3 = up.gather(1, e2)
    tap = lambda e, j: x.gather(1, e[:, :, None].expand(-1, -1, qkv)) * s["conv_weight"][:, j]  # noqa: E731
    y = tap(e3, 0) + tap(e2, 1) + tap(e1, 2) + tap(e0, 3) + s["conv_bias"]
    y = y / (1 + torch.exp(-y))
    q, k, v = y.split([hk * D, hk * D, hv * D], -1)
    unit = lambda r: r * torch.rsqrt(r.square().sum(-1, keepdim=True) + EPS)  # noqa: E731
    q, k = unit(q.reshape(B, T, hk, D)) / math.sqrt(D), unit(k.reshape(B, T, hk, D))
    v = v.reshape(B, T, hv, D).transpose(1, 2)
    a = s["a_out"].view(B, T, hv) + s["dt_bias"]
    g = -torch.exp(s["A_log"]) * (torch.clamp(a, min=0) + torch.log1p(torch.exp(-a.abs())))
    beta = (1 / (1 + torch.exp(-s["b_out"].view(B, T, hv)))).transpose(1, 2)[..., None]
    total = (anc.double() @ g.double()).transpose(1, 2)  # [B, hv, T], along each node's ancestors
    decay = torch.exp((total[..., :, None] - total[..., None, :]).float())
    decay = torch.where(anc[:, None], decay, 0.0)
    heads = lambda r: r.repeat_interleave(grp, 2).transpose(1, 2)  # noqa: E731
    qh, kh = heads(q), heads(k)
    S0 = s["state"].view(B, hv, D, D)
    begun = torch.exp(total.float())[..., None]
    low = -beta * decay * (kh @ kh.transpose(-1, -2))
    low = torch.where(torch.eye(T, device=DEV, dtype=torch.bool), 0.0, low)
    u = beta * (v - begun * (kh @ S0))
    for _ in range(max(1, (T - 1).bit_length())):  # (1 - low)^-1 = (1 + low)(1 + low^2)(1 + low^4)..
        u = u + low @ u
        low = low @ low
    o = begun * (qh @ S0) + (decay * (qh @ kh.transpose(-1, -2))) @ u
    o = o.transpose(1, 2) * torch.rsqrt(o.transpose(1, 2).square().mean(-1, keepdim=True) + EPS)
    z = s["z"].float().view(B, T, hv, D)
    out = o * s["norm_weight"] * (z / (1 + torch.exp(-z)))
    records = torch.cat([k.reshape(-1), u.transpose(1, 2).reshape(-1), torch.exp(g).reshape(-1)])
    return out.to(BF).view(B * T * hv, D), records


def _plain_accept(s):
    B, T = s["parent"].shape
    t = torch.arange(T, device=DEV)
    parent, live = s["parent"].long(), t < s["q_len"][:, None]
    match = live & (parent >= 0) & (s["draft_ids"] == s["target_ids"].gather(1, parent.clamp(min=0)))
    # of siblings with the same token the first
    twin = (parent[:, :, None] == parent[:, None, :]) & match[:, None, :] & (t[None, :] < t[:, None])
    match &= ~twin.any(-1)
    match[:, 0] = live[:, 0]
    on = live & ~(_ancestors(s["parent"]) & ~match[:, None, :]).any(-1)
    path = _path(on)
    n = on.sum(-1)
    # the accepted drafts, then the target's token at the last of them
    nodes = path.long().roll(-1, 1)
    ids = torch.where(t < (n - 1)[:, None], s["draft_ids"].gather(1, nodes.clamp(min=0)), -1)
    last = path.long().gather(1, (n - 1).clamp(min=0)[:, None]).clamp(min=0)
    end = (t == (n - 1)[:, None]) & (n > 0)[:, None]
    return (n - 1).int(), path, torch.where(end, s["target_ids"].gather(1, last), ids)


def _plain_commit(s):
    L, B, T, hk, hv = s["L"], s["B"], s["T"], s["hk"], s["hv"]
    qkv, grp = (2 * hk + hv) * D, hv // hk
    k, u, decay = s["records"].split([B * T * hk * D, B * T * hv * D, B * T * hv], 1)
    path = s["path"].long()
    on, at = (path >= 0)[None, :, :, None], path.clamp(min=0)
    take = lambda r, n: r.reshape(L, B, T, n).gather(  # noqa: E731
        2, at[None, :, :, None].expand(L, -1, -1, n))
    decay = torch.where(on, take(decay, hv), 1.0)
    upto = decay.flip(2).cumprod(2).flip(2)  # a node's decay and those after it
    later = torch.cat([upto[:, :, 1:], torch.ones_like(upto[:, :, :1])], 2)
    k = torch.where(on, take(k, hk * D), 0.0).view(L, B, T, hk, D).repeat_interleave(grp, 3)
    u = torch.where(on, take(u, hv * D), 0.0).view(L, B, T, hv, D) * later[..., None]
    S = s["state"].view(L, B, hv, D, D)
    S.copy_(S * upto[:, :, 0, :, None, None] + k.permute(0, 1, 3, 4, 2) @ u.transpose(2, 3))
    conv = s["conv_state"].view(L, B, qkv, 3)
    x = s["mixed_qkv"].view(L, B, T, qkv).gather(2, at[None, :, :, None].expand(L, -1, -1, qkv))
    window = torch.cat([conv.transpose(2, 3), x], 2)
    n = (path >= 0).sum(-1)
    last = n[:, None] + torch.arange(3, device=DEV)
    conv.copy_(window.gather(2, last[None, :, :, None].expand(L, -1, -1, qkv)).transpose(2, 3))


def _plain_compact(s):
    bs, path, slots = s["bs"], s["path"].long(), s["slots"]
    on = (path >= 0) & (slots >= 0)
    src, dst = slots.gather(1, path.clamp(min=0))[on], slots[on]
    moved = src != dst
    sb, so, db, do = src // bs, src % bs, dst // bs, dst % bs
    L, N, hkv = s["k_scale"].shape
    upto = torch.full((N,), -1, device=DEV).scatter_reduce(0, db, do, "amax")[db]
    older = torch.arange(bs, device=DEV) <= upto[:, None]  # [rows, bs]

    def within(cache, scale, rows_last):
        rows = (cache[:, sb, :, :, so] if rows_last else cache[:, sb, :, so]).transpose(0, 1)  # [L, n, hkv, 256]
        x = rows.view(E4M3).float()
        size = torch.where(x.isfinite() & moved[:, None, None], x.abs(), 0.0).amax(-1) * scale[:, sb]
        amax = torch.zeros(L, N, hkv, device=DEV).scatter_reduce(
            1, db[None, :, None].expand(L, -1, hkv), size, "amax")
        now = torch.maximum(scale, torch.where(amax > 0, _scale_of(amax), 0.0))
        by = (scale / now)[:, db, :, None, None]
        page = cache[:, db]
        mask = (older[:, None, None, :] if rows_last else older[:, None, :, None]) & (by != 1)
        cache[:, db] = torch.where(mask, _e4m3(page.view(E4M3).float() * by), page)
        by = (scale[:, sb] / now[:, db])[..., None]
        row = torch.where(by != 1, _e4m3(x * by), rows)
        if rows_last:
            cache[:, db, :, :, do] = row.transpose(0, 1)
        else:
            cache[:, db, :, do] = row.transpose(0, 1)
        scale.copy_(now)

    within(s["cache_k"], s["k_scale"], False)
    within(s["cache_v"], s["v_scale"], True)


# ---- one pass -----------------------------------------------------------------------------------

def _ops():
    import os
    import sys
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "neuron-pytorch-native_amd", "kernels")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import npn_ops  # noqa: F401  (registers the torch.ops)
    return torch.ops


def _own(s):
    ops, kind = _ops(), s["kind"]
    if kind == "attend":
        return ops.gqa.tree_verify_paged(
            s["query"], s["gate"], s["key"], s["value"], s["q_norm"], s["k_norm"], s["cos"], s["sin"],
            s["cache_k"], s["cache_v"], s["k_scale"], s["v_scale"], s["block_table"], s["kv_len"],
            s["slots"], s["q_len"], s["parent"])
    if kind == "recur":
        return ops.deltanet.verify_tree(
            s["state"], s["parent"], s["mixed_qkv"], s["conv_state"], s["conv_weight"], s["conv_bias"],
            s["a_out"], s["b_out"], s["z"], s["A_log"], s["dt_bias"], s["norm_weight"])
    if kind == "accept":
        return ops.spec.accept_tree(s["target_ids"], s["draft_ids"], s["parent"], s["q_len"])
    if kind == "commit":
        return ops.deltanet.commit_tree_(s["states"], s["conv_states"], s["mixed_qkvs"], s["recordss"],
                                         s["path"], s["hv"])
    return ops.gqa.compact_paged_(s["path"], s["slots"], s["cache_ks"], s["cache_vs"], s["k_scales"],
                                  s["v_scales"])


def _plain(s):
    return {"attend": _plain_attend, "recur": _plain_recur, "accept": _plain_accept,
            "commit": _plain_commit, "compact": _plain_compact}[s["kind"]](s)


def _caches(s):
    """The e4m3 values, and the scales that they are multiples of."""
    return {"k": s["cache_k"].view(E4M3), "v": s["cache_v"].view(E4M3), "k_scale": s["k_scale"],
            "v_scale": s["v_scale"]}


def run(s):
    """One pass; what it updates in place it may update again."""
    got = _own(s) if own else _plain(s)
    if s["kind"] == "attend":
        return {"attn": got, **_caches(s)}
    if s["kind"] == "recur":
        return {"out": got[0], "records": got[1]}
    if s["kind"] == "accept":
        return {"accepted": got[0], "path": got[1], "out_ids": got[2]}
    if s["kind"] == "commit":
        return {"state": s["state"], "conv_state": s["conv_state"]}
    return _caches(s)


# ---- what a pass cannot do without ----------------------------------------------------------------

def _depth(T, reach):
    """About how many nodes a path has: each step goes back (reach + 1) / 2 nodes."""
    return 1 + (T - 1) / ((min(reach, T) + 1) / 2)


def work(case):
    B, T = case["B"], case["T"]
    deep = _depth(T, case["reach"])
    if case["kind"] == "accept":
        return {"bytes": B * (T * 20 + 4 + 4 + T * 12), "flops": B * T}
    if case["kind"] == "recur":
        hk, hv = case["hk"], case["hv"]
        nodes = B * T
        return {"bytes": 4 * B * hv * D * D + 2 * nodes * (2 * hk + hv) * D + 2 * 2 * nodes * hv * D
                + 4 * nodes * ((hk + hv) * D + 3 * hv),
                "flops": nodes * hv * D * (4 * D + 8 * deep / 2)}
    if case["kind"] == "commit":
        hk, hv, n = case["hk"], case["hv"], 0.75 * deep
        heads = case["L"] * B * hv
        return {"bytes": heads * (8 * D * D + 4 * n * D) + case["L"] * B * (4 * n * hk * D + 4 * 3 * (2 * hk + hv) * D),
                "flops": heads * D * D * (1 + 2 * n)}
    if case["kind"] == "compact":
        rows = case["L"] * B * case["hkv"] * 0.75 * deep
        return {"bytes": rows * 4 * DH + 12 * B * T, "flops": rows * 2 * DH}
    hkv, hq = case["hkv"], case["hkv"] * case["grp"]
    kv, q = _lens(case["kv_lo"], case["kv_hi"], B), _lens(case["q_lo"], T, B)
    keys = sum(kv) + sum(q)
    seen = sum(kv) / B * sum(q) + sum(q) * _depth(T, case["reach"]) / 2
    return {"bytes": keys * hkv * (2 * DH + 8 / case["bs"]) + 3 * sum(q) * hq * DH * 2
            + sum(q) * hkv * DH * 2 * 3,
            "flops": 4 * DH * hq * seen}


# ---- the same in 64 bits ----------------------------------------------------------------------------

def _lines(parent):
    """Each node's ancestors and itself, node by node on the host."""
    lines = []
    for row in parent.tolist():
        mine = []
        for t, p in enumerate(row):
            mine.append((mine[p] if p >= 0 else []) + [t])
        lines.append(mine)
    return lines


def _turn64(x, w, pos):
    """Normed and rotated rows in 64 bits; the rotation as complex products, its angles from the
    32-bit table that the operators are given."""
    x = x.double()
    x = x / (x.pow(2).sum(-1, keepdim=True) / DH + EPS).sqrt() * (w.double() + 1)
    cos, sin = _tables(int(pos.max()) + 1)
    turn = torch.complex(cos[pos][..., :ROPE // 2].double(), sin[pos][..., :ROPE // 2].double())
    z = torch.complex(x[..., :ROPE // 2], x[..., ROPE // 2:ROPE]) * turn[:, None]
    return torch.cat([z.real, z.imag, x[..., ROPE:]], -1)


def _power64(big):
    """The least power of two s >= 2^-100 with big <= 448 s."""
    return torch.exp2(torch.ceil(torch.log2(big / MAX_E4M3)).clamp(min=MIN_EXP))


def _round64(x):
    return x.float().to(E4M3).double()


def _exact_attend(s):
    """Request by request: its rows into the pages, page by page, then each node over its own keys."""
    B, T, hq, _ = s["query"].shape
    hkv, bs = s["hkv"], s["bs"]
    out = torch.zeros(B, T, hq, DH, dtype=F64, device=DEV)
    k8, v8 = s["cache_k"].view(E4M3).float(), s["cache_v"].view(E4M3).float()  # exact in 32 bits
    ks, vs = s["k_scale"].double(), s["v_scale"].double()
    lines = _lines(s["parent"])
    for b in range(B):
        n, m = int(s["kv_len"][b]), int(s["q_len"][b])
        if m == 0:
            continue
        pos = torch.tensor([n + len(lines[b][t]) - 1 for t in range(m)], device=DEV)
        rows = (_turn64(s["key"][b, :m], s["k_norm"], pos), s["value"][b, :m].double())
        pages = s["block_table"][b, :-(-(n + m) // bs)].long()
        t = 0
        while t < m:
            block, off = int(pages[(n + t) // bs]), (n + t) % bs
            many = min(bs - off, m - t)
            for x, cache, scale, dim in ((rows[0], k8, ks, 1), (rows[1], v8, vs, 2)):
                x = x[t:t + many].transpose(0, 1)  # [hkv, many, 256]
                now = _power64(x.abs().amax((-2, -1)))
                page = cache[block]
                if off:
                    now = torch.maximum(scale[block], now)
                    lead = page.narrow(dim, 0, off)
                    lead.copy_(_round64(lead.double() * (scale[block] / now)[:, None, None]))
                x = _round64(x / now[:, None, None])
                page.narrow(dim, off, many).copy_(x if dim == 1 else x.transpose(-1, -2))
                scale[block] = now
            t += many
        see = torch.zeros(m, n + m, dtype=torch.bool, device=DEV)
        see[:, :n] = True
        for t in range(m):
            see[t, [n + a for a in lines[b][t]]] = True
        q = _turn64(s["query"][b, :m], s["q_norm"], pos)
        for h in range(hkv):
            k = (k8[pages, h].double() * ks[pages, h][:, None, None]).reshape(-1, DH)[:n + m].t().contiguous()
            v = (v8[pages, h].double() * vs[pages, h][:, None, None]).transpose(1, 2).reshape(-1, DH)[:n + m]
            for j in range(h * s["grp"], (h + 1) * s["grp"]):
                e = (q[:, j] @ k / 16.0).masked_fill(~see, -math.inf)
                e = (e - e.amax(-1, keepdim=True)).exp()
                out[b, :m, j] = e @ v / e.sum(-1, keepdim=True)
    return {"attn": out * torch.sigmoid(s["gate"].double()), "k": k8.double(), "v": v8.double(),
            "k_scale": ks, "v_scale": vs}


def _exact_recur(s):
    """Node by node, each from its parent's state and window."""
    B, T, hk, hv = s["B"], s["T"], s["hk"], s["hv"]
    qkv, grp = (2 * hk + hv) * D, hv // hk
    row = torch.arange(B, device=DEV)
    parent = s["parent"].long()
    states = torch.empty(B, T + 1, hv, D, D, dtype=F64, device=DEV)  # 0: the committed one, t + 1: node t's
    windows = torch.empty(B, T + 1, qkv, 3, dtype=F64, device=DEV)
    states[:, 0] = s["state"].double().view(B, hv, D, D)
    windows[:, 0] = s["conv_state"].double().view(B, qkv, 3)
    x = s["mixed_qkv"].double().view(B, T, qkv)
    w, bias = s["conv_weight"].double(), s["conv_bias"].double()
    gate = torch.nn.functional.softplus(s["a_out"].double().view(B, T, hv) + s["dt_bias"].double())
    decay = torch.exp(-s["A_log"].double().exp() * gate)
    beta = torch.sigmoid(s["b_out"].double().view(B, T, hv))
    ks, us, out = [], [], []
    for t in range(T):
        up = parent[:, t] + 1
        window = torch.cat([windows[row, up], x[:, t, :, None]], -1)
        windows[:, t + 1] = window[..., 1:]
        y = (window * w).sum(-1) + bias
        y = y * torch.sigmoid(y)
        q, k = y[:, :hk * D].view(B, hk, D), y[:, hk * D:2 * hk * D].view(B, hk, D)
        q = q / (q.pow(2).sum(-1, keepdim=True) + EPS).sqrt() / D ** 0.5
        k = k / (k.pow(2).sum(-1, keepdim=True) + EPS).sqrt()
        ks.append(k)
        q, k = q.repeat_interleave(grp, 1), k.repeat_interleave(grp, 1)
        S = states[row, up] * decay[:, t, :, None, None]
        u = (y[:, 2 * hk * D:].view(B, hv, D) - (S * k[..., None]).sum(-2)) * beta[:, t, :, None]
        S = S + k[..., None] * u[..., None, :]
        states[:, t + 1] = S
        us.append(u)
        o = (S * q[..., None]).sum(-2)
        out.append(o / (o.pow(2).mean(-1, keepdim=True) + EPS).sqrt())
    z = s["z"].double().view(B, T, hv, D)
    out = torch.stack(out, 1) * s["norm_weight"].double() * z * torch.sigmoid(z)
    return {"out": out.view(B * T * hv, D),
            "records": torch.cat([torch.stack(ks, 1).flatten(), torch.stack(us, 1).flatten(), decay.flatten()])}


def _exact_accept(s):
    """Request by request, from child to child on host lists."""
    T = s["T"]
    accepted, paths, out = [], [], []
    rows = zip(s["parent"].tolist(), s["draft_ids"].tolist(), s["target_ids"].tolist(), s["q_len"].tolist())
    for parent, draft, target, n in rows:
        path, ids = ([0] if n > 0 else []), []
        while path:
            token = target[path[-1]]
            ids.append(token)
            child = [c for c in range(path[-1] + 1, n) if parent[c] == path[-1] and draft[c] == token]
            if not child:
                break
            path.append(child[0])
        accepted.append(len(path) - 1)
        paths.append(path + [-1] * (T - len(path)))
        out.append(ids + [-1] * (T - len(ids)))
    return {"accepted": torch.tensor(accepted, dtype=I32, device=DEV),
            "path": torch.tensor(paths, dtype=I32, device=DEV), "out_ids": torch.tensor(out, device=DEV)}


def _exact_commit(s):
    """Layer by layer, request by request, one token step after the other."""
    L, B, T, hk, hv = s["L"], s["B"], s["T"], s["hk"], s["hv"]
    qkv, grp = (2 * hk + hv) * D, hv // hk
    state, conv = s["state"].double(), s["conv_state"].double()
    nodes = s["path"].tolist()
    for l in range(L):
        k, u, decay = s["records"][l].double().split([B * T * hk * D, B * T * hv * D, B * T * hv])
        k, u, decay = k.view(B, T, hk, D), u.view(B, T, hv, D), decay.view(B, T, hv)
        x = s["mixed_qkv"][l].double().view(B, T, qkv)
        S, win = state[l].view(B, hv, D, D), conv[l].view(B, qkv, 3)
        for b in range(B):
            for t in nodes[b]:
                if t < 0:
                    break
                key = k[b, t].repeat_interleave(grp, 0)
                S[b] = S[b] * decay[b, t][:, None, None] + key[:, :, None] * u[b, t][:, None, :]
                win[b] = torch.cat([win[b][:, 1:], x[b, t][:, None]], 1)
    return {"state": state, "conv_state": conv}


def _exact_compact(s):
    """Request by request and page by page, on values in 64 bits."""
    bs, T = s["bs"], s["T"]
    slots, nodes = s["slots"].tolist(), s["path"].tolist()
    got = {}
    for name, dim in (("k", -2), ("v", -1)):
        cache, scale = s["cache_" + name].view(E4M3).double(), s[name + "_scale"].double()
        for b in range(s["B"]):
            path = [p for p in nodes[b] if p >= 0]
            rows = [(cache[:, slots[b][p] // bs].select(dim, slots[b][p] % bs).clone(),
                     scale[:, slots[b][p] // bs].clone()) for p in path]  # all read before any is written
            d = 0
            while d < len(path):
                block, off = divmod(slots[b][d], bs)
                many = min(bs - off, len(path) - d)
                comes = [e for e in range(d, d + many) if path[e] != e]
                now = scale[:, block].clone()
                for e in comes:
                    now = torch.maximum(now, _power64((rows[e][0] * rows[e][1][..., None]).abs().amax(-1)))
                page = cache[:, block]
                lead = page.narrow(dim, 0, off + many)
                lead.copy_(_round64(lead * (scale[:, block] / now)[..., None, None]))
                for e in comes:
                    page.select(dim, off + e - d).copy_(_round64(rows[e][0] * (rows[e][1] / now)[..., None]))
                scale[:, block] = now
                d += many
        got[name], got[name + "_scale"] = cache, scale
    return {"k": got["k"], "v": got["v"], "k_scale": got["k_scale"], "v_scale": got["v_scale"]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "recur": _exact_recur, "accept": _exact_accept,
            "commit": _exact_commit, "compact": _exact_compact}[case["kind"]](s)
