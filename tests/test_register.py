"""Ops registered by npn_native.register, on stand-ins with a CPU kernel of their own: what the
dispatcher does above the kernel, which needs no GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import npn_native

X = torch.arange(4.0)


def _double(x, n):
    assert not isinstance(x, torch._subclasses.FakeTensor)
    return x.detach() * 2 + n


npn_native.register("npntest::double", "(Tensor x, int n) -> Tensor", lambda x, n: torch.empty_like(x))(_double)
torch.library.impl("npntest::double", "cpu", _double)


def _fill(x, y):
    x.detach().numpy()[:] = float(y.detach().sum())  # as a kernel writes: unseen by torch


npn_native.register("npntest::fill_", "(Tensor(a!) x, Tensor y) -> ()", lambda x, y: None)(_fill)
torch.library.impl("npntest::fill_", "cpu", _fill)
double, fill_ = torch.ops.npntest.double, torch.ops.npntest.fill_


def test_runs_where_no_gradient_is_expected():
    want = X * 2 + 1
    assert torch.equal(double(X, 1), want) and torch.equal(double(x=X, n=1), want)
    leaf = X.clone().requires_grad_()
    with torch.no_grad():
        out = double(leaf, 1)
    assert torch.equal(out, want) and not out.requires_grad
    with torch.inference_mode():
        assert torch.equal(double(X, 1), want) and torch.equal(double(X.clone(), 1), want)
    assert torch.equal(torch.func.vmap(lambda x: double(x, 1))(X.reshape(2, 2)), want.reshape(2, 2))
    assert torch.equal(torch.func.grad(lambda y, x: (y * double(x, 1)).sum())(X, X), want)
    assert torch.equal(torch.func.jvp(lambda y: y * double(X, 1), (X,), (torch.ones(4),))[1], want)
    with fwd.dual_level():
        assert torch.equal(fwd.unpack_dual(fwd.make_dual(X, X) * double(X, 1)).tangent, X * want)


@pytest.mark.parametrize("op", [lambda x: double(x, 1).sum(), lambda x: fill_(torch.zeros(2), x)],
                         ids=["returns", "in_place"])
def test_refuses_gradients_wherever_they_come_from(op):
    with pytest.raises(RuntimeError, match="requires grad"):
        op(X.clone().requires_grad_())
    for transform in (torch.func.grad, torch.func.vjp, torch.func.jacrev):
        with pytest.raises(RuntimeError, match="requires grad"):
            transform(op, X) if transform is torch.func.vjp else transform(op)(X)
    with pytest.raises(RuntimeError, match="requires grad"):
        torch.func.vmap(torch.func.grad(lambda x: double(x, 1).sum()))(X.reshape(2, 2))
    with pytest.raises(RuntimeError, match="tangent"):
        torch.func.jvp(op, (X,), (torch.ones(4),))
    with pytest.raises(RuntimeError, match="tangent"):
        torch.func.jacfwd(op)(X)
    with fwd.dual_level():
        dual = fwd.make_dual(X, torch.ones(4))
        with pytest.raises(RuntimeError, match="tangent"):
            op(dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
            op(dual)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_refuses_gradients_in_compiled_code(backend):
    import torch._dynamo
    torch._dynamo.reset()
    fn = torch.compile(lambda x: double(x, 1) * 3, backend=backend, fullgraph=True)
    assert torch.equal(fn(X), (X * 2 + 1) * 3)
    with pytest.raises(Exception, match="requires grad"):
        fn(X.clone().requires_grad_())
    with torch.no_grad():
        assert torch.equal(fn(X.clone().requires_grad_()), (X * 2 + 1) * 3)


def test_in_place_arguments_count_as_written():
    """A tensor that autograd has kept for another op's backward pass and the op then writes is noticed."""
    kept, w = torch.ones(4), torch.ones(4).requires_grad_()
    loss = (w * kept).sum()
    version = kept._version
    fill_(kept, X)
    assert kept._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.no_grad():
        version = kept._version
        fill_(kept, X)
        assert kept._version > version
    with torch.inference_mode():
        fill_(torch.ones(4), X)  # a tensor without a version
        version = kept._version
        fill_(kept, X)
    assert kept._version > version
