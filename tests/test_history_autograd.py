"""What the operators over histories do under automatic differentiation beside
a plain backward pass, on the CPU kernels (the autograd nodes are the same on
every device)."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from mdl_amd.block_norm import gated_residual_norm
from mdl_amd.history import RelativeBuckets, history_attention, relative_position_bias

RULE = RelativeBuckets(6, 8)


def rand(*shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(sum(shape)))


# Every differentiable input of the three operators, and a call with that input replaced.
def _attention(q=None, k=None, v=None, table=None):
    return history_attention(rand(2, 5, 4, 3) if q is None else q, rand(2, 6, 2, 3) if k is None else k,
                             rand(2, 6, 2, 3) if v is None else v, window=3, sinks=1,
                             bias_table=rand(6, 4) if table is None else table, buckets=RULE)


def _norm(x=None, o=None, post=None, following=None, gate=None, scale=None):
    rows, weight = rand(4, 7), rand(7)
    pick = lambda t, other: other if t is None else t  # noqa: E731
    return gated_residual_norm(pick(x, rows), pick(o, rows), pick(post, weight), pick(following, weight),
                               gate=pick(gate, rows), residual_scale=pick(scale, weight))[1]


INPUTS = {
    "attention q": (lambda t: _attention(q=t), (2, 5, 4, 3)),
    "attention k": (lambda t: _attention(k=t), (2, 6, 2, 3)),
    "attention v": (lambda t: _attention(v=t), (2, 6, 2, 3)),
    "attention table": (lambda t: _attention(table=t), (6, 4)),
    "bias table": (lambda t: relative_position_bias(t, 4, 5, RULE), (6, 4)),
    "norm x": (lambda t: _norm(x=t), (4, 7)),
    "norm block_out": (lambda t: _norm(o=t), (4, 7)),
    "norm post_weight": (lambda t: _norm(post=t), (7,)),
    "norm next_weight": (lambda t: _norm(following=t), (7,)),
    "norm gate": (lambda t: _norm(gate=t), (4, 7)),
    "norm residual_scale": (lambda t: _norm(scale=t), (7,)),
    "first norm x": (lambda t: gated_residual_norm(t, None, None, rand(7))[1], (4, 7)),
}


@pytest.mark.parametrize("name", INPUTS)
@pytest.mark.parametrize("requires_grad", [False, True])
def test_a_tangent_is_refused(name, requires_grad):
    """No operator here has a forward-mode formula: a dual input raises, and
    does not come back without its tangent."""

    call, shape = INPUTS[name]
    t = rand(*shape).requires_grad_(requires_grad)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError):
            call(forward_ad.make_dual(t, torch.ones(shape)))
        call(t)  # a plain tensor inside the level is as good as outside
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, (rand(*shape),), (torch.ones(shape),))


@pytest.mark.parametrize("name", INPUTS)
def test_a_second_derivative_raises(name):
    """First gradients are right under create_graph too; what would go through
    them again raises, instead of leaving its part out."""

    call, shape = INPUTS[name]
    t = rand(*shape).requires_grad_()
    plain = torch.autograd.grad(call(t).square().sum(), t)[0]
    (grad,) = torch.autograd.grad(call(t).square().sum(), t, create_graph=True)
    assert torch.equal(grad.detach(), plain)
    with pytest.raises(RuntimeError, match="once"):
        (grad.square().sum() + t.sum()).backward()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(grad.square().sum() + t.sum(), t)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.functional.hvp(lambda x: call(x).square().sum(), rand(*shape), torch.ones(shape))


def test_a_second_derivative_raises_for_what_only_the_gradients_share():
    # k requires nothing of its own: the upstream gradient alone leads back to w
    w = rand(2, 5, 4, 3).requires_grad_()
    q = rand(2, 5, 4, 3).requires_grad_()
    (grad,) = torch.autograd.grad((_attention(q=q) * w).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(grad.sum(), w)


def test_a_gradient_that_depends_on_nothing_differentiable_is_a_constant():
    # the bias is linear in its table, and this upstream gradient is given
    table = rand(6, 4).requires_grad_()
    (grad,) = torch.autograd.grad(relative_position_bias(table, 4, 5, RULE), table, rand(4, 4, 5), create_graph=True)
    assert not grad.requires_grad


def test_what_does_not_pass_the_operators_twice_is_left_alone():
    # a penalty on another branch of the same graph
    q, a = rand(2, 5, 4, 3).requires_grad_(), rand(3).requires_grad_()
    loss = _attention(q=q).sum() + a.pow(3).sum()
    dq, da = torch.autograd.grad(loss, [q, a], create_graph=True)
    da.square().sum().backward()
    torch.testing.assert_close(a.grad, 36 * a.detach() ** 3)
    assert dq.requires_grad and q.grad is None
