"""Second derivatives of the row-wise training operators: refused, never dropped.  The wrapper of their backward passes is
looked at on the CPU, the operators themselves on the GPU."""
import pytest
import torch


def node(linear):
    """x^3 (or 3 x) with a backward pass that is marked as the operators' are."""
    from cagnet_amd import gcn

    class Node(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, unused):
            ctx.save_for_backward(x)
            return 3 * x if linear else x**3

        @staticmethod
        @gcn._first_order(linear=linear)
        def backward(ctx, g):
            (x,) = ctx.saved_tensors
            return (3 * g if linear else 3 * x**2 * g), None

    return lambda x: Node.apply(x, None)


def test_gradient_penalty_on_a_sum_raises():
    """The incoming gradient of a sum needs none; the operator's depends on x all the same."""
    x = torch.tensor([2.0, -1.0], requires_grad=True)
    (g,) = torch.autograd.grad(node(False)(x).sum(), x, create_graph=True)
    assert g.tolist() == [12.0, 3.0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        torch.autograd.grad(x.sum() + g.square().sum(), x)


def test_linear_operators_have_a_zero_second_derivative_under_a_constant():
    x = torch.tensor([2.0, -1.0], requires_grad=True)
    (g,) = torch.autograd.grad(node(True)(x).sum(), x, create_graph=True)
    assert g.tolist() == [3.0, 3.0] and not g.requires_grad
    up = torch.ones(2, requires_grad=True)
    (g,) = torch.autograd.grad(node(True)(x), x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_first_derivatives_without_and_with_create_graph():
    for linear in (False, True):
        x = torch.tensor([2.0, -1.0], requires_grad=True)
        node(linear)(x).sum().backward()
        (g,) = torch.autograd.grad(node(linear)(x).sum(), x, create_graph=True)
        assert torch.equal(x.grad, g.detach())


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["rms_norm", "norm_residual r", "norm_residual h"])
def test_gradient_penalty_through_the_norms_raises(cuda, op):
    from cagnet_amd import gcn

    gen = torch.Generator().manual_seed(3)
    z, x = (torch.randn(12, 20, generator=gen).to(cuda).requires_grad_() for _ in range(2))
    w = torch.ones(20, device=cuda, requires_grad=True)
    call = {"rms_norm": lambda: gcn.rms_norm(z, w), "norm_residual r": lambda: gcn.norm_residual(z, x, w, None)[0],
            "norm_residual h": lambda: gcn.norm_residual(z, x, w, None)[1]}[op]
    (want,) = torch.autograd.grad(call().sum(), z)
    (g,) = torch.autograd.grad(call().sum(), z, create_graph=True)
    assert torch.equal(g, want)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (z.sum() + g.square().sum()).backward()


@pytest.mark.gpu
def test_linear_operators_under_a_sum(cuda):
    """Their gradients are constants there: a penalty on them adds nothing, and nothing raises."""
    from cagnet_amd import gcn

    x = torch.ones(6, 9, device=cuda, requires_grad=True)
    idx = torch.tensor([1, 1, 5], device=cuda)
    for y in (gcn.dropout(x, 0.4, gcn.rng_state(2, cuda)), gcn.embedding(x, idx, 2.0)):
        (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
        (second,) = torch.autograd.grad((x * x).sum() + g.square().sum(), x)
        assert torch.equal(second, 2 * x.detach())
