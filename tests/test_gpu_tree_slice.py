"""The verify slice's steps over trees at the end of its pages and after steps of the other kind."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, I32 = torch.bfloat16, torch.int32


def _slice(kv, s_max=64, K=3):
    from spec_verify_step import VerifySlice
    return VerifySlice(len(kv), K, kv, s_max, pattern="DG", seed=1, paged_block=16)


def _step_args(B, T, n, seed=0):
    from spec_verify_step import HIDDEN
    g = torch.Generator(device="cuda").manual_seed(seed)
    parent = torch.arange(-1, T - 1, dtype=I32, device="cuda").expand(B, -1).contiguous()
    ids = torch.randint(0, 9, (B, T), generator=g, device="cuda")
    target = ids.roll(-1, 1).contiguous()  # every draft is accepted
    return (torch.randn(B * T, HIDDEN, generator=g, device="cuda").to(BF), parent, ids, target,
            torch.tensor(n, dtype=I32, device="cuda"))


@pytest.mark.parametrize("kv,n,ok", [([64, 10], [0, 4], True), ([63, 10], [1, 4], True), ([63, 10], [-1, 9], True),
                                     ([62, 10], [3, 1], False), ([64, 10], [1, 1], False), ([10, 61], [4, 9], False)])
def test_slice_at_the_end_of_its_pages(kv, n, ok):
    """A step over trees needs room for the nodes that a sequence has in it, not for all T: one at s_max sits out
    while the others go on. Eager and replayed."""
    B, T = 2, 4
    eager, args = _slice(kv), _step_args(B, T, n)
    if not ok:
        with pytest.raises(RuntimeError, match="no room"):
            eager.step_tree(*args)
    with pytest.raises(RuntimeError, match="no room"):
        eager.step_tree(*args[:4])
    replayed = _slice(kv)
    args[4].zero_()
    replayed.step_tree(*args)
    replayed.capture_tree(*args)
    args[4].copy_(torch.tensor(n, dtype=I32))
    if not ok:
        with pytest.raises(RuntimeError, match="no room"):
            replayed.replay_tree()
        return
    nodes = np.clip(n, 0, T)
    _, accepted, _, _ = eager.step_tree(*args)
    got = replayed.replay_tree()
    torch.cuda.synchronize()
    for v in (eager, replayed):
        assert v.kv_len.tolist() == [k + int(m) for k, m in zip(kv, nodes)]
    assert accepted.tolist() == got[1].tolist() == [int(m) - 1 for m in nodes]


def test_replay_tree_after_a_chain_s_step():
    """The captured step reads states and lengths that a chain's step has left behind: refused, as step_tree is."""
    B, T = 2, 4
    v, args = _slice([5, 10]), _step_args(B, T, [4, 4])
    with pytest.raises(RuntimeError, match="capture_tree"):
        v.replay_tree()
    v.step_tree(*args)
    v.capture_tree(*args)
    v.replay_tree()
    v.forward(args[0])
    v.accept_and_rollback(torch.tensor([1, 2], dtype=I32, device="cuda"))
    kv = v.kv_len.tolist()
    for call in (v.replay_tree, lambda: v.step_tree(*args)):
        with pytest.raises(RuntimeError, match="checkpoints"):
            call()
    assert v.kv_len.tolist() == kv
