"""Tree-verification ops without a GPU: shape propagation, refusal of CPU tensors, the C entries' size and pointer checks
(which come before any launch), and `register` with lists of tensors, on stand-ins with a CPU kernel of their own."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

import npn_native
import npn_ops  # noqa: F401

BF, I32, I64, I8 = torch.bfloat16, torch.int32, torch.int64, torch.int8


def _args(B=2, T=5, hk=2, hv=6, H=2, grp=6, N=7, P=3, bs=32):
    qkv, e = (2 * hk + hv) * 128, torch.empty
    parent = e(B, T, dtype=I32)
    dn = (e(B * hv * 128, 128), parent, e(B * T * qkv, dtype=BF), e(B * qkv, 3, dtype=BF), e(qkv, 4), e(qkv), e(B * T * hv),
          e(B * T * hv), e(B * T * hv, 128, dtype=BF), e(hv), e(hv), e(128))
    rows = lambda n: e(B, T, n, 256, dtype=BF)  # noqa: E731
    pages = (e(N, H, bs, 256, dtype=I8), e(N, H, 256, bs, dtype=I8), e(N, H), e(N, H))
    slots, length = e(B, T, dtype=I64), e(B, dtype=I32)
    attn = (rows(H * grp), rows(H * grp), rows(H), rows(H), e(256), e(256), e(100, 64), e(100, 64), *pages,
            e(B, P, dtype=I32), length, slots, length, parent)
    return dn, attn, pages, slots, length, parent


def _calls():
    dn, attn, pages, slots, length, parent = _args()
    ops, ids = torch.ops, torch.empty(2, 5, dtype=I64)
    rec = torch.empty(2 * 5 * (8 * 128 + 6))
    return {"verify": lambda: ops.deltanet.verify_tree(*dn), "attend": lambda: ops.gqa.tree_verify_paged(*attn),
            "accept": lambda: ops.spec.accept_tree(ids, ids, parent, length),
            "commit": lambda: ops.deltanet.commit_tree_([dn[0]], [dn[3]], [dn[2]], [rec], parent, 6),
            "compact": lambda: ops.gqa.compact_paged_(parent, slots, *[[p] for p in pages])}


def test_shapes_propagate():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        calls = _calls()
        out, rec = calls["verify"]()
        assert (out.shape, out.dtype) == ((2 * 5 * 6, 128), BF)
        assert (rec.shape, rec.dtype) == ((2 * 5 * (8 * 128 + 6),), torch.float32)
        assert calls["attend"]().shape == (2, 5, 12, 256)
        accepted, path, ids = calls["accept"]()
        assert [(t.shape, t.dtype) for t in (accepted, path, ids)] == [((2,), I32), ((2, 5), I32), ((2, 5), I64)]
        assert calls["commit"]() is None and calls["compact"]() is None


@pytest.mark.parametrize("name", list(_calls()))
def test_cpu_tensors_are_refused(name):
    with pytest.raises((NotImplementedError, RuntimeError)):
        _calls()[name]()


def test_tree_shape():
    from deltanet_tree_ops import tree_shape
    assert tree_shape(torch.empty(3, 64), "parent") == (3, 64)
    for bad in ((3,), (3, 0), (0, 3), (3, 65), (65536, 1), (1, 2, 3)):
        with pytest.raises(RuntimeError):
            tree_shape(torch.empty(bad), "parent")


def test_size_query():
    q = lambda *s: npn_native.query("npn_gqa_tree_verify_paged_workspace_size", *s)  # noqa: E731
    assert q(1, 1, 6, 1, 5, 16) > 0 and q(4, 64, 24, 4, 300, 128) > 0
    assert q(65535, 1, 6, 1, 5, 16) > 0 and q(65536, 1, 6, 1, 5, 16) == 0
    for bad in ((1, 65, 6, 1, 5, 16), (1, 0, 6, 1, 5, 16), (0, 1, 6, 1, 5, 16), (1, 1, 7, 2, 5, 16), (1, 1, 6, 0, 5, 16),
                (1, 1, 6, 1, 0, 16), (1, 1, 6, 1, 5, 48), (1, 1, 6, 1, -1, 16), (1, 1, 6, 1, 2 ** 32 + 5, 16)):
        assert q(*bad) == 0, bad


def test_entries_check_sizes_and_pointers():
    """Statuses of the C entries for sizes and pointers that they refuse before any launch (which has a status of its own,
    5, where there is no device; the addresses here are made up, so this is no test for where there is one)."""
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    lib, p = npn_native.lib(), 4096  # an aligned address that is never read
    refused = (1, 2, 3, 6)  # null, shape, alignment, value
    assert lib.npn_accept_tree(*[p] * 7, 1, 4, None) == 5
    for B, T in ((0, 4), (1, 0), (1, 65), (2 ** 22 + 1, 4), (-1, 4)):
        assert lib.npn_accept_tree(p, p, p, p, p, p, p, B, T, None) in refused
        assert lib.npn_deltanet_verify_tree(*[p] * 14, B, T, 1, 1, None) in refused
        one = ctypes.cast((ctypes.c_void_p * 1)(p), ctypes.c_void_p)
        assert lib.npn_deltanet_commit_tree(one, one, one, one, 1, p, B, T, 1, 1, None) in refused
        assert lib.npn_gqa_compact_paged(p, p, one, one, one, one, 1, B, T, 1, 4, 16, None) in refused
    for hk, hv in ((0, 0), (2, 3), (1, 0), (-1, -1), (1, 1 << 23)):
        assert lib.npn_deltanet_verify_tree(*[p] * 14, 1, 4, hk, hv, None) in refused
    for i in range(7):
        assert lib.npn_accept_tree(*[None if j == i else p for j in range(7)], 1, 4, None) in refused
    for i in range(14):
        assert lib.npn_deltanet_verify_tree(*[None if j == i else p for j in range(14)], 1, 4, 1, 1, None) in refused
    table = lambda *v: ctypes.cast((ctypes.c_void_p * len(v))(*v), ctypes.c_void_p)  # noqa: E731
    MB = 1 << 20
    commit = lambda *t, layers: lib.npn_deltanet_commit_tree(*[table(*v) for v in t], layers, p, 1, 4, 1, 1,  # noqa: E731
                                                             None)
    compact = lambda *t, layers: lib.npn_gqa_compact_paged(p, p, *[table(*v) for v in t], layers, 1, 4, 1, 4,  # noqa: E731
                                                           16, None)
    good = [(1 * MB, 2 * MB), (3 * MB, 4 * MB), (5 * MB, 6 * MB), (7 * MB, 8 * MB)]
    assert commit(*good, layers=2) == compact(*good, layers=2) == 5
    for i in range(4):  # a null table, a null layer, a layer twice and one that begins inside another
        for bad in ((None, 2 * MB), (1 * MB, None)):
            lists = [bad if j == i else t for j, t in enumerate(good)]
            assert commit(*lists, layers=2) in refused and compact(*lists, layers=2) in refused
        first = good[i][0]
        # 4 blocks of 16 rows of 256 bytes, their 4 scales; 64 KB of state, a window of 3 * 384 bf16
        last = first + ((4 * 16 * 256, 4 * 16 * 256, 16, 16)[i] - (16 if i < 2 else 4))
        for at in (first, last):
            lists = [(first, at) if j == i else t for j, t in enumerate(good)]
            assert compact(*lists, layers=2) == 6
            assert compact(*[t[::-1] for t in lists], layers=2) == 6
        lists = [(first, first + 16 * ((1024, 1024, 1, 1)[i])) if j == i else t for j, t in enumerate(good)]
        assert compact(*lists, layers=2) == 5  # one behind the other
    for i, size in ((0, 65536), (1, 2304)):
        lists = lambda at: [(good[i][0], good[i][0] + at) if j == i else t for j, t in enumerate(good)]  # noqa: E731
        assert commit(*lists(0), layers=2) == commit(*lists(size - 16), layers=2) == 6
        assert commit(*lists(size), layers=2) == 5
    for i in (0, 2):  # K's and V's in one place
        lists = [good[i] if j == i + 1 else t for j, t in enumerate(good)]
        assert compact(*lists, layers=2) == 6 and compact(*lists, layers=1) == 6
    assert lib.npn_deltanet_commit_tree(None, *[table(MB)] * 3, 1, p, 1, 4, 1, 1, None) == 1
    assert lib.npn_gqa_compact_paged(p, p, None, *[table(MB)] * 3, 1, 1, 4, 1, 4, 16, None) == 1
    for bs, n in ((48, 4), (16, 0), (16, -1)):
        assert lib.npn_gqa_compact_paged(p, p, *[table(*t) for t in good], 2, 1, 4, 1, n, bs, None) in refused


def _add_(xs, y):
    for x in xs:
        x.detach().numpy()[:] += float(y.detach().sum())  # as a kernel writes: unseen by torch


npn_native.register("npntest::add_lists_", "(Tensor(a!)[] xs, Tensor y) -> ()", lambda xs, y: None)(_add_)
torch.library.impl("npntest::add_lists_", "cpu", _add_)
add_ = torch.ops.npntest.add_lists_


def test_lists_count_as_written():
    xs, y = [torch.zeros(2), torch.zeros(3)], torch.ones(2)
    before = [x._version for x in xs] + [y._version]
    add_(xs, y)
    assert [x._version for x in xs] == [v + 1 for v in before[:2]] and y._version == before[2]
    assert torch.equal(xs[1], torch.full((3,), 2.0))
    leaf = torch.ones(2, requires_grad=True)
    saved = leaf * xs[0]  # keeps xs[0] for its backward pass
    add_(xs, y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.sum().backward()
    with torch.inference_mode():
        add_([torch.zeros(2), xs[0]], y)
    add_([], y)


def test_lists_refuse_gradients():
    y = torch.ones(2)
    grad = torch.zeros(2, requires_grad=True)
    for call in (lambda: add_([torch.zeros(2), grad], y), lambda: add_([torch.zeros(2)], y.clone().requires_grad_()),
                 lambda: torch.func.grad(lambda v: add_([torch.zeros(2), v], y))(torch.zeros(2))):
        with pytest.raises(RuntimeError, match="requires grad"):
            call()
    with torch.no_grad():
        add_([grad], y)
    with fwd.dual_level(), pytest.raises(RuntimeError, match="tangent"):
        add_([torch.zeros(2), fwd.make_dual(torch.zeros(2), torch.ones(2))], y)


def test_lists_through_compile():
    import torch._dynamo
    torch._dynamo.reset()

    def step(xs, y):
        add_(xs, y)
        return xs[0] + xs[1]

    xs = [torch.zeros(2), torch.ones(2)]
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(xs, torch.ones(2))
    assert torch.equal(got, torch.full((2,), 5.0)) and torch.equal(xs[0], torch.full((2,), 2.0))
