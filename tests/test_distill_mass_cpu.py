"""CPU: the gradient that vocab_oracle.distill states is the derivative of the loss that it states, for lists whose probabilities and rest
bucket do not add up to one too.  The derivative is taken by autograd of the loss written out in 64 bits."""
import pytest
import torch

import vocab_oracle as oracle
from distill_lists import KINDS, lists, loss64


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_oracle_gradient_is_the_derivative(kind, tail):
    x, values, index, lse, temp = lists(kind, torch.float32, 203)
    g = torch.linspace(0.5, 1.5, x.shape[0]).double()
    loss, grad, _ = oracle.distill(x, values, index, lse, temp, tail, g)
    z = x.double().requires_grad_()
    want, mass = loss64(z, values, index, lse, temp, tail)
    (want_grad,) = torch.autograd.grad((want * g).sum(), z)
    assert (loss - want).abs().max() < 1e-11 and (grad - want_grad).abs().max() < 1e-11
    assert grad.sum(1).abs().max() < 1e-11                        # softmax does not see a constant added to a row
    if tail and kind != "fits":
        assert (mass - 1).abs().max() > 1e-3                      # what these lists are for
