"""The paged serving operators: what is measured of them, in plain torch and by the kernels.

A decode or verify step over a paged 8-bit KV cache plans its pages, appends its new K/V rows,
attends and, for plain decode, samples a token. Kinds of cases:

  blocks  one scheduling cycle of the block tables (paged::update_blocks_): blocks and slots for
          the new tokens of B requests, then the blocks that the step did not keep given back
  append  the new K/V rows of B requests into the e4m3 pages (gqa::kv_append_paged)
  attend  attention of T new tokens per request over those pages (gqa::tail_verify_paged); T = 1
          is plain decode, a long T a chunk of a prompt
  sample  one token per row of logits with temperature, top-k, top-p and min-p (spec::sample)

The cache: cache_k [N, Hkv, bs, 256] and cache_v [N, Hkv, 256, bs] e4m3fn bytes, one power-of-two
scale per block and head each; attention heads of 256 with a 64-dim partial RoPE.
`own` selects the framework's kernels; the plain form is elementary torch in 32 bits, in 64 for
the sampler's sums.
"""
import math

import torch

own = False

DEV = "cuda"
DH, ROPE, THETA, EPS = 256, 64, 1e7, 1e-6
E4M3, BF, F32, F64 = torch.float8_e4m3fn, torch.bfloat16, torch.float32, torch.float64
I32, I64 = torch.int32, torch.int64
MAX_E4M3, MIN_EXP = 448.0, -100
U_TOP = 1.0 - 2.0 ** -24


def listed():
    return [
        # a verify step's plan at a serving batch: at most one new block per request
        {"name": "blocks_step_b64", "kind": "blocks", "B": 64, "T": 8, "bs": 64, "kv_lo": 0,
         "kv_hi": 32768, "new_lo": 0, "spare": 1.0},
        # a batch of prompts admitted at once into small pages
        {"name": "blocks_prompts_b256", "kind": "blocks", "B": 256, "T": 2048, "bs": 16,
         "kv_lo": 0, "kv_hi": 8192, "new_lo": 0, "spare": 1.0},
        # plain decode: one row per request
        {"name": "append_token_b32", "kind": "append", "B": 32, "T": 1, "hkv": 4, "bs": 64,
         "kv_lo": 1, "kv_hi": 32768},
        # a verify step: eight rows per request, pages that end inside them
        {"name": "append_verify_b32", "kind": "append", "B": 32, "T": 8, "hkv": 4, "bs": 16,
         "kv_lo": 1, "kv_hi": 32768},
        # prompts of 4096 tokens into the pages
        {"name": "append_prompt_4x4096", "kind": "append", "B": 4, "T": 4096, "hkv": 4, "bs": 64,
         "kv_lo": 0, "kv_hi": 100},
        # one user's long conversation, one token at a time
        {"name": "attend_token_b1", "kind": "attend", "B": 1, "T": 1, "hkv": 4, "grp": 6,
         "bs": 64, "kv_lo": 32768, "kv_hi": 32768},
        # plain decode of a mixed batch on one of four ranks, small pages
        {"name": "attend_token_b64", "kind": "attend", "B": 64, "T": 1, "hkv": 1, "grp": 6,
         "bs": 16, "kv_lo": 100, "kv_hi": 16384},
        # a verify step over mixed long caches at full width
        {"name": "attend_verify_b16", "kind": "attend", "B": 16, "T": 8, "hkv": 4, "grp": 6,
         "bs": 64, "kv_lo": 4096, "kv_hi": 32768},
        # a chunk of two long prompts
        {"name": "attend_chunk_2x256", "kind": "attend", "B": 2, "T": 256, "hkv": 4, "grp": 6,
         "bs": 64, "kv_lo": 4096, "kv_hi": 8192},
        # one user's next token
        {"name": "sample_b1", "kind": "sample", "R": 1, "V": 151936, "bf16": False},
        # a serving batch, each request with its own settings
        {"name": "sample_b32", "kind": "sample", "R": 32, "V": 151936, "bf16": False},
        # a large batch over the larger vocabulary, straight from a bf16 head
        {"name": "sample_b256", "kind": "sample", "R": 256, "V": 248320, "bf16": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["blocks", "append", "attend", "attend", "sample", "sample"])
    bs = rng.choice([16, 32, 64, 128])
    if kind == "blocks":
        B = _log_int(rng, 1, 256)
        T = _log_int(rng, 1, min(2048, 524288 // B))
        # spare below 1: the pool cannot serve every request
        return {"kind": kind, "B": B, "T": T, "bs": bs, "kv_lo": 0,
                "kv_hi": _log_int(rng, 16, 8192), "new_lo": rng.choice([0, 1, T]),
                "spare": rng.choice([1.0, 1.0, 0.5])}
    if kind == "append":
        hkv = rng.choice([1, 2, 4])
        B = _log_int(rng, 1, 128)
        T = _log_int(rng, 1, min(4096, 16384 * 4 // (B * hkv)))
        return {"kind": kind, "B": B, "T": T, "hkv": hkv, "bs": bs, "kv_lo": 0,
                "kv_hi": _log_int(rng, 1, 32768)}
    if kind == "attend":
        hkv, grp = rng.choice([(1, 6), (2, 4), (4, 6)])
        if rng.random() < 0.25:  # a prompt's chunk
            B, T = rng.choice([1, 2]), _log_int(rng, 32, 256)
            hi = _log_int(rng, 64, 6144)
        else:
            B, T = _log_int(rng, 1, 64), rng.choice([1, 1, 2, 3, 5, 8])
            hi = _log_int(rng, 64, min(32768, 1100000 // (B * hkv)))
        return {"kind": kind, "B": B, "T": T, "hkv": hkv, "grp": grp, "bs": bs,
                "kv_lo": rng.choice([0, hi // 8, hi]), "kv_hi": hi}
    bf16 = rng.random() < 0.5
    return {"kind": kind, "R": _log_int(rng, 1, 256 if bf16 else 128),
            "V": _log_int(rng, 1000, 248320), "bf16": bf16}


# ---- inputs ---------------------------------------------------------------------------------

def _lens(lo, hi, n):
    """n lengths spread evenly over [lo, hi]; which request has which comes from the seed."""
    return [lo + (hi - lo) * (2 * i + 1) // (2 * n) for i in range(n)]


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen, device=DEV)
    return torch.tensor(values, dtype=I32, device=DEV)[order]


def _tables(positions):
    inv = THETA ** (-torch.arange(0, ROPE, 2, device=DEV, dtype=F64) / ROPE)
    ang = torch.arange(positions, device=DEV, dtype=F64)[:, None] * inv
    ang = torch.cat([ang, ang], -1)
    return ang.cos().float(), ang.sin().float()


def _paged(kv_len, total, bs, gen):
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
        x = x / scale[i:i + 1024, :, None, None]
        cache[i:i + 1024] = x.to(E4M3).view(torch.int8)
    return cache, scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *n: torch.randn(*n, generator=gen, device=DEV)  # noqa: E731
    s = dict(case)
    if case["kind"] == "sample":
        R, V = case["R"], case["V"]
        # a language model's rows: a broad bulk, some rows sharper than others, a few likely tokens
        x = rnd(R, V) * (1.0 + 2.0 * torch.rand(R, 1, generator=gen, device=DEV))
        likely = torch.rand(R, V, generator=gen, device=DEV) < 40.0 / V
        x += 6.0 * likely * torch.rand(R, V, generator=gen, device=DEV)
        pick = lambda v: torch.tensor(v, device=DEV)[torch.randint(  # noqa: E731
            0, len(v), (R,), generator=gen, device=DEV)]
        s["logits"] = x.to(BF) if case["bf16"] else x
        s["temperature"] = pick([0.0, 0.3, 0.6, 0.7, 1.0, 1.0, 1.5])
        s["top_k"] = pick([0, 0, 1, 20, 40, 1000]).int()
        s["top_p"] = pick([1.0, 1.0, 0.5, 0.8, 0.95])
        s["min_p"] = pick([0.0, 0.0, 0.05, 0.1])
        s["u"] = torch.rand(R, generator=gen, device=DEV)
        return s

    B, T, bs = case["B"], case["T"], case["bs"]
    kv = _shuffled(_lens(case["kv_lo"], case["kv_hi"], B), gen)
    s["kv_len"] = kv
    if case["kind"] == "blocks":
        new = _shuffled(_lens(case["new_lo"], T, B), gen)
        cap = (case["kv_hi"] + T + bs - 1) // bs
        have = (kv.long() + bs - 1) // bs
        # a request's new rows reach at most new / bs + 1 further pages
        free = sum(int(case["spare"] * n / bs) + (case["spare"] == 1.0) for n in new.tolist())
        N = max(1, int(have.sum()) + free)
        ids = torch.randperm(N, generator=gen, device=DEV).int()
        s["block_table"] = torch.full((B, cap), -1, dtype=I32, device=DEV)
        held = torch.arange(cap, device=DEV)[None] < have[:, None]
        s["block_table"][held] = ids[:int(have.sum())]
        s["num_blocks"] = have.int()
        s["free_blocks"] = torch.zeros(N, dtype=I32, device=DEV)
        s["free_blocks"][:free] = ids[int(have.sum()):int(have.sum()) + free]
        s["free_count"] = torch.tensor([free], dtype=I32, device=DEV)
        s["new_len"], s["none"] = new, torch.zeros_like(new)
        return s

    hkv = case["hkv"]
    s["cos"], s["sin"] = _tables(case["kv_hi"] + T)
    if case["kind"] == "append":
        # pages of the rows' neighbourhood only; the requests' older pages are not touched
        base = kv // bs * bs
        table, N = _paged(kv, kv - base + T, bs, gen)
        at = (kv - base)[:, None].long() + torch.arange(T, device=DEV)
        s["slots"] = table.long().gather(1, at // bs) * bs + at % bs
        s["key"], s["value"] = rnd(B, T, hkv, DH).to(BF), rnd(B, T, hkv, DH).to(BF)
        s["k_norm"] = rnd(DH) * 0.1
    else:
        s["block_table"], N = _paged(kv, kv + T, bs, gen)
        hq = hkv * case["grp"]
        s["query"], s["gate"] = rnd(B, T, hq, DH).to(BF), rnd(B, T, hq, DH).to(BF)
        s["q_norm"] = rnd(DH) * 0.1
        s["q_len"] = torch.full((B,), T, dtype=I32, device=DEV)
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


def _rows(s):
    """RoPE rows [B, T, 1, 64] of the new tokens, positions clamped to the table."""
    at = s["kv_len"].long()[:, None] + torch.arange(s["T"], device=DEV)
    at = at.clamp(0, s["cos"].shape[0] - 1)
    return s["cos"][at][:, :, None], s["sin"][at][:, :, None]


def _plain_update(s, new_len):
    """One paged::update_blocks_ in place; returns (slots, granted)."""
    table, have, stack, count = s["block_table"], s["num_blocks"], s["free_blocks"], s["free_count"]
    (B, P), N, bs, T = table.shape, stack.numel(), s["bs"], s["T"]
    kv = s["kv_len"].long().clamp(min=0)
    new = new_len.long().clamp(0, T)
    want = (kv + new + bs - 1) // bs
    held = have.long().clamp(0, P)
    at = torch.arange(P, device=DEV)
    # give back: the last request's last block first, so that the first request's is on top
    drop = (at >= want[:, None]) & (at < held[:, None])
    order = drop.flatten().long().flip(0).cumsum(0).flip(0).view(B, P) - 1
    where = torch.where(drop, count.long() + order, N)
    wide = torch.cat([stack, stack.new_zeros(1)])
    wide.scatter_(0, where.flatten(), torch.where(drop, table, 0).flatten())
    free = count.long() + drop.sum()
    # grant, in request order, as far as the pool reaches
    need = torch.where(want <= P, want - held, 0).clamp(min=0)
    upto = need.cumsum(0)
    fits = (want <= P) & ((need == 0) | (upto <= free))
    take = fits[:, None] & (at >= held[:, None]) & (at < want[:, None])
    index = free - 1 - ((upto - need)[:, None] + at - held[:, None])
    got = wide[torch.where(take, index, N)]
    table.copy_(torch.where(take, got, torch.where(drop, -1, table)))
    have.copy_(torch.where(fits, want, held))
    stack.copy_(wide[:N])
    count.copy_(free - torch.where(fits, need, 0).sum())
    granted = torch.where(fits, new, 0)
    pos = kv[:, None] + torch.arange(T, device=DEV)
    slots = table.long().gather(1, (pos // bs).clamp(max=P - 1)) * bs + pos % bs
    slots = torch.where(torch.arange(T, device=DEV) < granted[:, None], slots, -1)
    return slots, granted.int()


def _plain_append(s):
    bs, slots = s["bs"], s["slots"]
    k = _norm_rope(s["key"].float(), s["k_norm"], *_rows(s))
    ok = slots >= 0
    blk, off = slots[ok] // bs, slots[ok] % bs
    N, hkv = s["k_scale"].shape
    first = torch.full((N,), bs, device=DEV).scatter_reduce(0, blk, off, "amin")
    head = slots[:, 0][ok[:, 0]] // bs  # only a request's first page holds older rows
    for_head = torch.arange(bs, device=DEV) < first[head][:, None]
    for x, cache, scale, rows_last in ((k[ok], s["cache_k"], s["k_scale"], False),
                                       (s["value"].float()[ok], s["cache_v"], s["v_scale"], True)):
        size = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
        amax = torch.zeros(N, hkv, device=DEV).scatter_reduce(
            0, blk[:, None].expand(-1, hkv), size, "amax")
        need = _scale_of(amax)
        grown = torch.where((first > 0)[:, None], torch.maximum(scale, need), need)
        grown = torch.where((first < bs)[:, None], grown, scale)
        page = cache[head]
        by = (scale[head] / grown[head])[:, :, None, None]
        again = _e4m3(page.view(E4M3).float() * by)
        mask = for_head[:, None, None, :] if rows_last else for_head[:, None, :, None]
        mask = mask & (by != 1)
        cache[head] = torch.where(mask, again, page)
        scale.copy_(grown)
        q = _e4m3(x / grown[blk][:, :, None])
        if rows_last:
            cache[blk, :, :, off] = q
        else:
            cache[blk, :, off] = q


def _plain_attend(s):
    B, T, hq, _ = s["query"].shape
    table, bs = s["block_table"].long(), s["bs"]
    (N, hkv), P = s["k_scale"].shape, table.shape[1]
    grp, S = hq // hkv, P * bs
    held = (table >= 0) & (table < N)
    page = torch.where(held, table, 0)
    q = _norm_rope(s["query"].float(), s["q_norm"], *_rows(s)) / 16.0
    q = q.view(B, T, hkv, grp, DH).transpose(1, 2).reshape(B, hkv, T * grp, DH)
    k = s["cache_k"][page].view(E4M3).float() * s["k_scale"][page][..., None, None]
    k = k.transpose(1, 2).reshape(B, hkv, S, DH)
    score = q @ k.transpose(-1, -2)
    del k
    score = score.view(B, hkv, T, grp, S)
    at = torch.arange(S, device=DEV)
    t = torch.arange(T, device=DEV)
    last = torch.minimum(s["kv_len"].long()[:, None] + t, (s["kv_len"] + s["q_len"])[:, None] - 1)
    seen = (at <= last[:, :, None]) & held.repeat_interleave(bs, 1)[:, None]
    score = torch.where(seen[:, None, :, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    v = s["cache_v"][page].view(E4M3).float() * s["v_scale"][page][..., None, None]
    v = v.permute(0, 2, 1, 4, 3).reshape(B, hkv, S, DH)
    o = p.view(B, hkv, T * grp, S) @ v
    o = o.view(B, hkv, T, grp, DH).transpose(1, 2).reshape(B, T, hq, DH)
    o = o / (1 + torch.exp(-s["gate"].float()))
    return torch.where((t < s["q_len"][:, None])[:, :, None, None], o, 0.0).to(BF)


def _plain_sample(s):
    x = s["logits"].float()
    R, V = x.shape
    x = torch.where(x.isnan(), -math.inf, x)
    over = x.amax(-1, keepdim=True) == math.inf
    x = torch.where(over, torch.where(x == math.inf, 0.0, -math.inf), x)
    x, order = x.sort(dim=-1, descending=True, stable=True)
    hot = s["temperature"] > 0
    temp = torch.where(hot, s["temperature"], 1.0).double()[:, None]
    w = torch.exp((x.double() - x[:, :1].double()) / temp)
    w = torch.where(x == -math.inf, 0.0, w)
    rank = torch.arange(V, device=DEV)
    k = s["top_k"][:, None]
    w = torch.where((rank < k) | (k <= 0), w, 0.0)
    c = w.cumsum(-1)
    p = s["top_p"].double()[:, None]
    before = torch.cat([torch.zeros_like(c[:, :1]), c[:, :-1]], -1)
    keep = (before < p * c[:, -1:]) | (rank == 0) | ~(p < 1)
    m = s["min_p"].double().clamp(max=1.0)[:, None]
    keep &= (w >= m) | ~(m > 0)
    c = torch.where(keep, w, 0.0).cumsum(-1)
    u = s["u"].double().nan_to_num(0.0).clamp(0.0, U_TOP)[:, None]
    at = (c <= u * c[:, -1:]).sum(-1).clamp(max=V - 1)
    at = torch.where(hot, at, 0)
    ids = order.gather(1, at[:, None])[:, 0]
    return torch.where(x[:, 0] == -math.inf, -1, ids)


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
    ops = _ops()
    if s["kind"] == "blocks":
        plan = lambda new: ops.paged.update_blocks_(  # noqa: E731
            s["kv_len"], new, s["block_table"], s["num_blocks"], s["free_blocks"],
            s["free_count"], s["bs"], s["T"])
        slots, granted = plan(s["new_len"])
        plan(s["none"])
        return slots, granted
    if s["kind"] == "append":
        ops.gqa.kv_append_paged(s["key"], s["value"], s["k_norm"], s["cos"], s["sin"], s["kv_len"],
                                s["slots"], s["cache_k"], s["cache_v"], s["k_scale"], s["v_scale"])
        return None
    if s["kind"] == "attend":
        return ops.gqa.tail_verify_paged(s["query"], s["gate"], s["q_norm"], s["cos"], s["sin"],
                                         s["cache_k"], s["cache_v"], s["k_scale"], s["v_scale"],
                                         s["block_table"], s["kv_len"], s["q_len"])
    return ops.spec.sample(s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"],
                           s["u"])


def _plain(s):
    if s["kind"] == "blocks":
        slots, granted = _plain_update(s, s["new_len"])
        _plain_update(s, s["none"])
        return slots, granted
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[s["kind"]](s)


def run(s):
    """One pass. The block cycle ends with the tables as they were, an append writes the same rows
    again, so that a state can be run any number of times."""
    got = _own(s) if own else _plain(s)
    if s["kind"] == "blocks":
        return {"slots": got[0], "granted": got[1], "block_table": s["block_table"],
                "num_blocks": s["num_blocks"], "free_blocks": s["free_blocks"],
                "free_count": s["free_count"]}
    if s["kind"] == "append":  # the e4m3 values, and the scales that they are multiples of
        return {"k": s["cache_k"].view(E4M3), "v": s["cache_v"].view(E4M3),
                "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return {"attn": got} if s["kind"] == "attend" else {"ids": got}


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    if case["kind"] == "sample":
        n = case["R"] * case["V"]
        return {"bytes": n * (2 if case["bf16"] else 4) + 28 * case["R"], "flops": 4 * n}
    B, T, bs = case["B"], case["T"], case["bs"]
    kv = _lens(case["kv_lo"], case["kv_hi"], B)
    if case["kind"] == "blocks":
        # both calls' slots, the lengths and counts, and each moved block on the stack and in its table
        moved = sum(_lens(case["new_lo"], T, B)) / bs * case["spare"]
        return {"bytes": 2 * 8 * B * T + 2 * 20 * B + 2 * 16 * moved, "flops": 2 * 4 * B * T}
    hkv = case["hkv"]
    if case["kind"] == "append":
        rows = B * T * hkv
        return {"bytes": 2 * rows * DH * 3 + B * T * (8 + 2 * 4 * ROPE), "flops": 12 * rows * DH}
    keys = sum(n + T for n in kv)
    seen = sum(T * n + T * (T + 1) // 2 for n in kv)
    hq = hkv * case["grp"]
    return {"bytes": keys * hkv * (2 * DH + 8 / bs) + 3 * B * T * hq * DH * 2,
            "flops": 4 * DH * hq * seen}


# ---- the same in 64 bits ----------------------------------------------------------------------------

def _turn64(x, w, pos):
    """Normed and rotated rows in 64 bits; the rotation as complex products, its angles from the
    32-bit table that the operators are given."""
    x = x.double()
    x = x / (x.pow(2).sum(-1, keepdim=True) / DH + EPS).sqrt() * (w.double() + 1)
    cos, sin = _tables(int(pos.max()) + 1)
    turn = torch.complex(cos[pos][..., :ROPE // 2].double(), sin[pos][..., :ROPE // 2].double())
    z = torch.complex(x[..., :ROPE // 2], x[..., ROPE // 2:ROPE]) * turn[:, None]
    return torch.cat([z.real, z.imag, x[..., ROPE:]], -1)


def _exact_blocks(s):
    """Two scheduling calls, request by request, on host lists."""
    table, stack = s["block_table"].tolist(), s["free_blocks"].tolist()
    held, free, kv = s["num_blocks"].tolist(), int(s["free_count"]), s["kv_len"].tolist()
    bs, T, P = s["bs"], s["T"], len(table[0])
    first = None
    for new in (s["new_len"].tolist(), s["none"].tolist()):
        want = [-(-(n + m) // bs) for n, m in zip(kv, new)]
        for b in reversed(range(len(kv))):
            while held[b] > want[b]:
                held[b] -= 1
                stack[free], table[b][held[b]] = table[b][held[b]], -1
                free += 1
        short, slots, granted, left = False, [], [], free
        for b, n in enumerate(kv):
            need = max(0, want[b] - held[b]) if want[b] <= P else 0
            left -= need
            short = left < 0
            good = want[b] <= P and (need == 0 or not short)
            if good:
                top = left + need  # where this request's share of the stack begins
                for _ in range(need):
                    top -= 1
                    table[b][held[b]] = stack[top]
                    held[b] += 1
            m = new[b] if good else 0
            granted.append(m)
            slots.append([table[b][(n + t) // bs] * bs + (n + t) % bs for t in range(m)] +
                         [-1] * (T - m))
            free -= need if good else 0
        first = first or (slots, granted)
    as32 = lambda v: torch.tensor(v, dtype=I32, device=DEV)  # noqa: E731
    return {"slots": torch.tensor(first[0], dtype=I64, device=DEV), "granted": as32(first[1]),
            "block_table": as32(table), "num_blocks": as32(held), "free_blocks": as32(stack),
            "free_count": as32([free])}


def _exact_append(s):
    """Request by request and page by page, the pages as 64-bit values with the rows last in K too."""
    bs, T = s["bs"], s["T"]
    values = {"k": s["cache_k"].view(E4M3).double(), "v": s["cache_v"].view(E4M3).double()}
    scales = {"k": s["k_scale"].double(), "v": s["v_scale"].double()}
    for b in range(s["B"]):
        n = int(s["kv_len"][b])
        rows = {"k": _turn64(s["key"][b], s["k_norm"], torch.arange(n, n + T, device=DEV)),
                "v": s["value"][b].double()}
        slots, t = s["slots"][b].tolist(), 0
        while t < T:
            block, off = divmod(slots[t], bs)
            m = min(bs - off, T - t)
            for name, dim in (("k", -2), ("v", -1)):
                x = rows[name][t:t + m].transpose(0, 1)  # [Hkv, m, 256]
                big = x.abs().amax((-2, -1))
                need = torch.exp2(torch.ceil(torch.log2(big / MAX_E4M3)).clamp(min=MIN_EXP))
                old = scales[name][block]
                now = torch.maximum(old, need) if off else need
                page = values[name][block]
                x = (x / now[:, None, None]).float().to(E4M3).double()
                page.narrow(dim, off, m).copy_(x if name == "k" else x.transpose(-1, -2))
                if off:
                    lead = page.narrow(dim, 0, off)
                    lead.copy_((lead * (old / now)[:, None, None]).float().to(E4M3).double())
                scales[name][block] = now
            t += m
    return {**values, "k_scale": scales["k"], "v_scale": scales["v"]}


def _exact_attend(s):
    """Request by request over its own keys, the softmax as a ratio of sums."""
    B, T, hq, _ = s["query"].shape
    out = torch.zeros(B, T, hq, DH, dtype=F64, device=DEV)
    hkv, bs = s["hkv"], s["bs"]
    for b in range(B):
        n, m = int(s["kv_len"][b]), int(s["q_len"][b])
        pages = s["block_table"][b, :-(-(n + m) // bs)].long()
        q = _turn64(s["query"][b, :m], s["q_norm"], torch.arange(n, n + m, device=DEV))
        hide = torch.arange(n + m, device=DEV)[None] > n + torch.arange(m, device=DEV)[:, None]
        for h in range(hkv):
            k = s["cache_k"][pages, h].view(E4M3).double() * s["k_scale"][pages, h].double()[:, None, None]
            v = s["cache_v"][pages, h].view(E4M3).double() * s["v_scale"][pages, h].double()[:, None, None]
            k = k.reshape(-1, DH)[:n + m].t().contiguous()
            v = v.transpose(1, 2).reshape(-1, DH)[:n + m]
            for j in range(h * s["grp"], (h + 1) * s["grp"]):
                e = (q[:, j] @ k / 16.0).masked_fill(hide, -math.inf)
                e = (e - e.amax(-1, keepdim=True)).exp()
                out[b, :m, j] = e @ v / e.sum(-1, keepdim=True)
    return {"attn": out * torch.sigmoid(s["gate"].double())}


def _exact_sample(s):
    """Row by row: the candidates shrink filter by filter."""
    ids = []
    for r in range(s["R"]):
        x = s["logits"][r].double()
        idx = torch.arange(len(x), device=DEV)[~x.isnan() & (x > -math.inf)]
        if not len(idx):
            ids.append(-1)
            continue
        idx = idx[torch.argsort(-x[idx], stable=True)]
        t, k, p, m, u = (float(s[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
        if not t > 0:
            ids.append(int(idx[0]))
            continue
        idx = idx[:int(k)] if k > 0 else idx
        w = torch.exp((x[idx] - x[idx[0]]) / t)
        n = len(w)
        if p < 1:
            run = torch.cumsum(w, 0)
            n = 1 + int(torch.searchsorted(run, torch.tensor([p * float(run[-1])], dtype=F64, device=DEV))[0])
        if m > 0:
            n = min(n, int((w >= min(m, 1.0)).sum()))
        w = w[:max(n, 1)]
        run = torch.cumsum(w, 0)
        goal = torch.tensor([min(max(u, 0.0), U_TOP) * float(run[-1])], dtype=F64, device=DEV)
        ids.append(int(idx[int(torch.searchsorted(run, goal, right=True)[0])]))
    return {"ids": torch.tensor(ids, dtype=I64, device=DEV)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"blocks": _exact_blocks, "append": _exact_append, "attend": _exact_attend,
            "sample": _exact_sample}[case["kind"]](s)
