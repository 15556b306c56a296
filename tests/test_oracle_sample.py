"""The sampler's oracle (oracle/sample.py) against known answers and frequencies, and the entry
point's refusals, which reach no GPU."""
import numpy as np
import pytest
import torch

from oracle import sample as os_

NAN, INF = float("nan"), float("inf")


def pick(x, T=1.0, k=0, p=1.0, m=0.0, u=0.0):
    return os_.sample_row(np.array(x, np.float32), np.float32(T), k, np.float32(p), np.float32(m), np.float32(u))


@pytest.mark.parametrize("want,x,kw", [
    (1, [0, 2, 1], dict(T=0)), (1, [0, 2, 2], dict(T=-1)), (1, [0, 2, 2], dict(T=NAN)),
    (-1, [-INF, NAN], {}), (0, [5, NAN], dict(u=0.9)),
    (1, [3, INF, 3, INF], dict(u=0.4)), (3, [3, INF, 3, INF], dict(u=0.6)),
    (2, [-0.0, -1, 0.0, -1], dict(u=0.5, k=2)),          # -0 and 0 are equal: ranks 0 and 2
    (3, [0, 0, 0, 0], dict(u=0.75)), (2, [0, 0, 0, 0], dict(u=0.74)),
    (1, [0, 0, 0, 0], dict(u=0.99, p=0.5)),              # two of four equal ones reach half
    (2, [0, 0, 0, 0], dict(u=0.99, p=np.float32(0.5) + np.float32(1e-7))),
    (0, [0, 0, 0, 0], dict(u=0.99, p=0.0)), (0, [0, 0], dict(u=0.99, p=-1)), (1, [0, 0], dict(u=0.99, p=NAN)),
    (1, [0, 0, -1], dict(u=0.99, m=1.0)), (1, [0, 0, -1], dict(u=0.99, m=7.0)), (2, [0, 0, -1], dict(u=0.99, m=NAN)),
    (2, [0, 0, -1], dict(u=INF)), (0, [0, 0], dict(u=NAN)), (0, [0, 0], dict(u=-1)),
    (1, [0, 1e30, 5], dict(u=0.999)), (0, [1, 2, 3], dict(T=INF, u=0.99)),
])
def test_known_answers(want, x, kw):
    assert pick(x, **kw) == want


def test_frequencies():
    """Uniform u on a fine grid reproduces the kept tokens' probabilities to a grid step each."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal(20).astype(np.float32)
    n = 4000
    got = np.bincount([pick(x, T=0.7, k=12, p=0.9, m=0.05, u=(i + 0.5) / n) for i in range(n)], minlength=20) / n
    w = np.exp((x.astype(np.float64) - x.max()) / np.float32(0.7))
    order = np.argsort(-w)
    keep = order[:12]
    cum = np.cumsum(w[keep]) / w[keep].sum()
    keep = keep[:int((cum < np.float32(0.9)).sum()) + 1]
    keep = keep[w[keep] >= np.float32(0.05)]
    want = np.zeros(20)
    want[keep] = w[keep] / w[keep].sum()
    assert np.abs(got - want).max() <= 1.0 / n + 1e-12


def test_refusals_on_the_host():
    import npn_native
    A = 1 << 20

    def st(ptrs=[A] * 7, bf16=0, R=2, V=10, ws=A, n=1 << 40):
        return npn_native.lib().npn_sample(ptrs[0], bf16, *ptrs[1:], R, V, ws, n, None)
    for i in range(7):
        assert st([0 if j == i else A for j in range(7)]) == 1
    for bad in (dict(R=0), dict(V=0), dict(V=(1 << 20) + 1), dict(bf16=2), dict(bf16=-1)):
        assert st(**bad) == 2, bad
    assert st([A + 4] + [A] * 6) == 3 and st(ws=A + 8) == 3
    n = npn_native.query("npn_sample_workspace_size", 2, 10)
    assert n > 0 and st(n=n - 1) == 4 and st(ws=None) == 4
    assert npn_native.query("npn_sample_workspace_size", 65536, 10) == 0


def test_op_refuses_cpu_tensors_and_propagates_shapes():
    import npn_ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    r = torch.ones(2)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.ops.spec.sample(torch.zeros(2, 5), r, r.int(), r, r, r)
    with FakeTensorMode():
        r = torch.empty(3)
        ids = torch.ops.spec.sample(torch.empty(3, 7, dtype=torch.bfloat16), r, r.int(), r, r, r)
        assert ids.shape == (3,) and ids.dtype == torch.int64
