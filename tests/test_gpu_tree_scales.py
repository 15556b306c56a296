"""What a node's row does to the nodes that do not see it but share a page's scale with it (gqa::tree_verify_paged).
Tolerances as in test_gpu_tree.py."""
import numpy as np
import pytest
import torch

from oracle import tree as ot
from _util import BF16_U, assert_rel_close
from test_gpu_tree import _args, _attend_inputs

pytestmark = pytest.mark.gpu


def _others(d, node):
    """The nodes that do not see `node` of request 0."""
    return [t for t in range(d["query"].shape[1]) if node not in ot.line(d["parent"][0], t)]


@pytest.mark.parametrize("T", [6, 10, 40])
@pytest.mark.parametrize("what", ["sign", "half"])
def test_a_node_s_row_within_its_page_s_scale_reaches_its_line_alone(ops, T, what):
    """Another key and value of a node, of no larger magnitude: no bit of the others' outputs changes."""
    d = _attend_inputs(1, T, 2, 6, 16, [61], [T], 3, seed=21)
    node = T // 3
    calm = ops.gqa.tree_verify_paged(*_args(d))
    if what == "sign":
        d["key"][0, node].neg_()
        d["value"][0, node].neg_()
    else:  # (a key's own length does not count)
        d["value"][0, node].mul_(0.5)
    got = ops.gqa.tree_verify_paged(*_args(d))
    other = _others(d, node)
    assert 0 < len(other) < T and torch.equal(got[0, other], calm[0, other])
    assert not torch.equal(got[0, node], calm[0, node])


@pytest.mark.parametrize("T", [6, 10, 40])
@pytest.mark.parametrize("exp", [7, 12])
def test_a_node_s_large_row_takes_its_page_s_other_rows_to_its_scale(ops, T, exp):
    """A value far above the others' makes its page's scale grow: the page's other rows, committed ones among them, are
    rounded to it, and nodes that do not see the value are the formula's on those."""
    d = _attend_inputs(1, T, 2, 6, 16, [61], [T], 3, seed=21)
    node = T // 3
    calm = ops.gqa.tree_verify_paged(*_args(d))
    d["value"][0, node].mul_(2.0 ** exp)
    args = _args(d)
    got = ops.gqa.tree_verify_paged(*args)
    torch.cuda.synchronize()
    f = lambda k: d[k].double().numpy()  # noqa: E731
    want = [c.copy() for c in d["cache"]]
    ot.kv_append(f("key"), f("value"), f("k_norm"), d["cos"], d["sin"], d["kv"], d["slots"], d["parent"], want)
    cache = [a.cpu().numpy() for a in args[8:12]]
    cache[0], cache[1] = cache[0].view(np.uint8), cache[1].view(np.uint8)
    for i in (1, 2, 3):
        assert np.array_equal(cache[i], want[i]), i
    ref = ot.tree_verify(f("query"), f("gate"), f("q_norm"), d["cos"], d["sin"], cache, d["table"], d["kv"], d["n"], d["parent"])
    other = _others(d, node)
    mine = [t for t in range(T) if t not in other]
    for rows in (other, mine):
        assert_rel_close(got[0, rows].float().cpu().numpy(), ref[0, rows], tol=2e-3, out_unit=BF16_U)
    assert not torch.equal(got[0, other], calm[0, other])
