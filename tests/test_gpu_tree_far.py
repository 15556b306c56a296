"""The tree-verification operators where offsets pass 32 bits, and on views and streams that the other tests do not have: the
same results as for small tensors, bit for bit."""
import numpy as np
import pytest
import torch

from oracle import tree as ot
from _util import BF16_U, assert_rel_close
from test_gpu_tree import _args, _attend_inputs, cuda, trees

pytestmark = pytest.mark.gpu
BF, I32 = torch.bfloat16, torch.int32


@pytest.mark.parametrize("T", [4, 64])
def test_pages_past_32_bits(ops, T):
    """The pages of a small cache as the last ones of one of 4.6 GB: attention (both kernels), append and compaction."""
    bs, N = 128, 140000  # 32 KB a page of one head
    d = _attend_inputs(2, T, 1, 6, bs, [300, 129], [T, T - 1], max(1, T // 4), seed=T)
    small = _args(d)
    n = small[8].shape[0]
    big = list(small)
    for i, shape in ((8, (N, 1, bs, 256)), (9, (N, 1, 256, bs)), (10, (N, 1)), (11, (N, 1))):
        big[i] = torch.zeros(shape, dtype=small[i].dtype, device="cuda")
        big[i][N - n:] = small[i]
    big[12] = torch.where(small[12] >= 0, small[12] + N - n, -1).int()
    big[14] = torch.where(small[14] >= 0, small[14] + (N - n) * bs, -1)
    want, got = (ops.gqa.tree_verify_paged(*a) for a in (small, big))
    assert torch.equal(want, got)
    path = cuda(np.array([[0, 2, 3] + [-1] * (T - 3), [0, 1] + [-1] * (T - 2)], np.int32))
    for a in (small, big):
        ops.gqa.compact_paged_(path, a[14], *[[c] for c in a[8:12]])
    for i in range(8, 12):
        assert torch.equal(small[i], big[i][N - n:]) and not big[i][:2].any()


def test_states_past_32_bits(ops):
    """More than 2^31 state elements: the last requests' outputs, records and states are those of a batch of them alone."""
    B, T, hk, hv, last = 65535, 3, 1, 3, 100
    qkv = (2 * hk + hv) * 128
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    full = dict(state=torch.zeros(B * hv * 128, 128, device="cuda"), parent=cuda(np.tile(trees(1, T, 2, 0), (B, 1))),
                mixed=r(B * T * qkv).to(BF), conv=r(B * qkv, 3).to(BF), a=r(B * T * hv), b=r(B * T * hv),
                z=r(B * T * hv, 128).to(BF))
    full["state"][-last * hv * 128:] = r(last * hv * 128, 128)
    w = (r(qkv, 4), r(qkv), r(hv), r(hv), r(128))
    part = {k: v[-last * (v.shape[0] // B):].clone() for k, v in full.items()}
    path = cuda(np.tile(np.array([0, 2, -1], np.int32), (B, 1)))
    outs = []
    for s, p in ((full, path), (part, path[-last:].contiguous())):
        out, rec = ops.deltanet.verify_tree(s["state"], s["parent"], s["mixed"], s["conv"], w[0], w[1], s["a"], s["b"], s["z"],
                                            w[2], w[3], w[4])
        ops.deltanet.commit_tree_([s["state"]], [s["conv"]], [s["mixed"]], [rec], p, hv)
        outs.append(out)
    assert torch.equal(outs[0][-last * T * hv:], outs[1])
    for k in ("state", "conv"):
        assert torch.equal(full[k][-part[k].shape[0]:], part[k]), k


@pytest.mark.parametrize("missing", [False, True])
def test_many_rows_over_many_steps(ops, missing):
    """384 rows over 400000 keys: more steps to a workgroup than it has pages of in LDS at a time, also where one is missing. A
    chain's, against the chain's kernel: both within the formula's tolerance, so within twice that of each other."""
    d = _attend_inputs(1, 64, 1, 6, 128, [400000], [64], 1, seed=3)
    if missing:
        d["table"][0, [5, 1700]] = -1
    query, gate, key, value, qn, kn, cos, sin, *cache, table, kv, slots, n, _ = args = _args(d)
    out = ops.gqa.tree_verify_paged(*args)
    want = ops.gqa.tail_verify_paged(query, gate, qn, cos, sin, *args[8:12], table, kv, n)
    assert_rel_close(out.float().cpu().numpy(), want.float().cpu().numpy(), tol=4e-3, out_unit=2 * BF16_U)


def test_views_inside_larger_tensors(ops):
    """Integer inputs that begin anywhere in a larger tensor, and a list whose layers are slices of one tensor."""
    T, H, bs = 9, 2, 16
    d = _attend_inputs(2, T, H, 6, bs, [20, 33], [T, T], 3, seed=8)
    whole = _args(d)
    shifted = _args(d)
    for i in (12, 13, 14, 15, 16):
        t = shifted[i]
        room = torch.full((t.numel() + 3,), 7, dtype=t.dtype, device="cuda")
        room[3:] = t.flatten()
        shifted[i] = room[3:].view(t.shape)
    assert torch.equal(ops.gqa.tree_verify_paged(*whole), ops.gqa.tree_verify_paged(*shifted))
    path = shifted[16].clone().fill_(-1)
    path[:, 0], path[0, 1], path[1, 1] = 0, 4, 2
    ids = torch.randint(0, 2, (2, T), device="cuda")
    room = torch.zeros(2 * T + 1, dtype=torch.int64, device="cuda")
    room[1:] = ids.flatten()
    for x, y in zip(ops.spec.accept_tree(ids, ids, whole[16], whole[15]),
                    ops.spec.accept_tree(room[1:].view(2, T), room[1:].view(2, T), shifted[16], shifted[15])):
        assert torch.equal(x, y)
    stack = [torch.stack([c, c]) for c in shifted[8:12]]  # two layers in one tensor
    ops.gqa.compact_paged_(path, shifted[14], *[[c[0], c[1]] for c in stack])
    ops.gqa.compact_paged_(path, whole[14], *[[c] for c in whole[8:12]])
    for c, s in zip(whole[8:12], stack):
        assert torch.equal(c, s[0]) and torch.equal(c, s[1])
    with pytest.raises(RuntimeError):  # the second begins inside the first
        flat = torch.zeros(2 * whole[8].numel(), dtype=torch.int8, device="cuda")
        n = whole[8].numel()
        ops.gqa.compact_paged_(path, whole[14], [flat[:n].view(whole[8].shape), flat[bs * 256:bs * 256 + n].view(whole[8].shape)],
                               *[[c[0], c[1]] for c in stack[1:]])


def test_on_a_stream_of_its_own(ops):
    """A call on another stream than its inputs', with their making in flight before it and a reader behind."""
    d = _attend_inputs(2, 20, 2, 6, 16, [100, 333], [20, 17], 5, seed=4)
    want_args = _args(d)
    want = ops.gqa.tree_verify_paged(*want_args)
    args = _args(d)
    busy = torch.randn(2048, 2048, device="cuda")
    side = torch.cuda.Stream()
    for _ in range(20):
        busy = busy @ busy * 1e-3
    args[0] = args[0] + 0
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops.gqa.tree_verify_paged(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(args[8:12], want_args[8:12]))


@pytest.mark.parametrize("T", [5, 40])
@pytest.mark.parametrize("k_exp,v_exp", [((-9, -5), (-120, 60)), ((-110, -5), (-9, -5)), ((-7, -4), (-100, -96)),
                                         ((-9, -5), (-126, -126))])
def test_scales_far_apart(ops, T, k_exp, v_exp):
    """Pages whose scales are any powers of two between these: the formula's outputs, small or large as they are."""
    d = _attend_inputs(2, T, 2, 6, 16, [300, 45], [T, T], max(1, T // 4), seed=T)
    rng = np.random.default_rng(T)
    for i, (lo, hi) in ((2, k_exp), (3, v_exp)):
        used = d["table"][d["table"] >= 0]
        far = np.exp2(rng.integers(lo, hi + 1, (len(used), 2))).astype(np.float32)
        d["cache"][i][used] = far
    # the tree's own values as large as its pages' scales: the last page of the committed rows holds both
    top = 2.0 ** min(v_exp[1] + 4, 60)
    d["value"] = (d["value"].float() * top).to(BF)
    args = _args(d)
    out = ops.gqa.tree_verify_paged(*args)
    f = lambda k: d[k].double().numpy()  # noqa: E731
    cache = [a.cpu().numpy() for a in args[8:12]]
    cache[0], cache[1] = cache[0].view(np.uint8), cache[1].view(np.uint8)
    with np.errstate(over="ignore", invalid="ignore"):
        ref = ot.tree_verify(f("query"), f("gate"), f("q_norm"), d["cos"], d["sin"], cache, d["table"], d["kv"], d["n"], d["parent"])
    assert np.isfinite(ref).all()
    # A row against its own size, and three absolute terms. Its output is a bf16, half a step of whose subnormals is 2^-134.
    # A weight P s (s: the value's scale) is an f16 of 2^11 to 2^15 times it over the row's largest one, so half a step of
    # the smallest is 2^-25 2^-11 of that, at most 2^-36 smax; it meets a byte of at most 448 at each of the keys, and the
    # sum is over l >= 2^-4 (the running maximum lags by up to 2^4). It counts where the largest scale's rows are all 0: an
    # append's scale is 2^-100 at least, which leaves nothing of the rows of a page of 2^-126.
    got = out.double().cpu().numpy()
    keys = np.array([int(kv) + T for kv in d["kv"]])
    smax = np.stack([cache[3][t[t >= 0]].max(0).astype(np.float64) for t in d["table"]])  # [B, kv head]
    lost = np.repeat(2.0**-36 * 2**4 * 448 * keys[:, None] * smax, 6, axis=1)[:, None]
    err = np.linalg.norm(got - ref, axis=-1)
    assert (err <= (2e-3 + 2**-8) * np.linalg.norm(ref, axis=-1) + 16 * (2.0**-134 + lost)).all()
    if v_exp[0] > -126:  # where no page is below an append's least scale by more than f16 reaches, the first term is enough
        assert (err <= (2e-3 + 2**-8) * np.linalg.norm(ref, axis=-1)).all()
