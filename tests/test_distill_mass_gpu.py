"""GPU: the gradient of ops.top_distill is that of the loss it returns, for lists whose probabilities and rest bucket do not add up to one
too: against autograd of the loss in 64 bits, against differences of the loss, and by its sum over a row.

Tolerances.  A sum of exponentials, fp32 within a thread and double across threads, is within 1e-5 (EPS).  A gradient element is a sum of
terms of sizes w q_v, p_r q_v / q_r and p_v, each within 3 EPS (sum, quotient, exponential), then rounded to its type by half a step,
finfo.eps / 2, and by half the smallest step where it leaves the normal range."""
import pytest
import torch

from distill_lists import KINDS, lists, loss64

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs a GPU"
    from nast_amd import ops as o
    return o


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [203, 40001])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("kind", KINDS)
def test_gradient_is_that_of_the_loss(ops, kind, tail, V, dtype):
    x, values, index, lse, temp = lists(kind, dtype, V)
    g = torch.linspace(0.25, 1.5, x.shape[0])
    leaf = x.cuda().requires_grad_()
    loss = ops.top_distill(leaf, ops.TopLogits(values.cuda(), index.cuda(), lse.cuda(), temp), temp, tail)
    (grad,) = torch.autograd.grad(loss, leaf, g.cuda())
    z = x.double().requires_grad_()
    want_loss, mass = loss64(z, values, index, lse, temp, tail)
    (want,) = torch.autograd.grad((want_loss * g.double()).sum(), z)
    want_loss = want_loss.detach()
    # the sum's error enters a loss with the mass of its terms
    assert ((loss.detach().cpu().double() - want_loss).abs() <= EPS * mass.clamp(min=1.0) + want_loss.abs() * 2.0 ** -24).all()
    p = torch.zeros_like(want).scatter_add_(1, index, (values.double() / temp - (lse.double().unsqueeze(1) if tail else torch.logsumexp(
        values.double() / temp, 1, keepdim=True))).exp())
    q = torch.softmax(z.detach() / temp, 1)
    named = torch.zeros_like(p, dtype=torch.bool).scatter_(1, index, True)
    bucket = (mass - p.sum(1)).clamp(min=0).unsqueeze(1) * torch.where(named, 0.0, q) / torch.where(named, 0.0, q).sum(1, keepdim=True).clamp(min=1e-300)
    scale = (mass.unsqueeze(1) * q + p + bucket) * g.double().unsqueeze(1) / temp
    fin = torch.finfo(dtype)
    tol = 3 * EPS * scale + want.abs() * fin.eps / 2 + fin.smallest_normal * fin.eps
    assert ((grad.cpu().double() - want).abs() <= tol).all()
    assert (grad.cpu().double().sum(1).abs() <= tol.sum(1)).all()


@pytest.mark.parametrize("kind", KINDS)
def test_gradient_against_differences(ops, kind):
    """h = 0.025.  A loss below 8 is rounded by 2.4e-7 at most; the sum of the few tokens outside the list has 3 roundings, an instruction's
    1.2e-7 and 2.6 * 1.24e-7 of arguments, 6.2e-7, and 2.4e-7 of two merges, and enters with a mass below 2.5: 2.2e-6.  Two such losses
    over 2 h: 1e-4.  The third derivative is below 2.5 / T^3 * 0.2: h^2 / 6 of it 2.4e-5."""
    x, values, index, lse, temp = (t.cuda() if torch.is_tensor(t) else t for t in lists(kind, torch.float32, 23, R=1))
    top = ops.TopLogits(values, index, lse, temp)
    leaf = x.clone().requires_grad_()
    ops.top_distill(leaf, top, temp, True).sum().backward()
    for e in range(x.shape[1]):
        if x[0, e].isinf():
            assert leaf.grad[0, e] == 0
            continue
        a, b = x.clone(), x.clone()
        a[0, e] += 0.025
        b[0, e] -= 0.025
        d = (ops.top_distill(a, top, temp, True) - ops.top_distill(b, top, temp, True)).item() / (a[0, e] - b[0, e]).item()
        assert abs(d - leaf.grad[0, e].item()) < 1.3e-4


def test_generator_distill_of_a_rounded_list(ops):
    """the same through the node that holds the product: gradients to x, W and b; fp32 products over 64, relative 1e-4"""
    gen = torch.Generator().manual_seed(3)
    _, values, index, lse, temp = lists("rounded", torch.float32, 203)
    x, W, b = (torch.randn(*s, generator=gen) for s in ((4, 64), (203, 64), (203,)))
    leaves = [t.cuda().requires_grad_() for t in (x, W, b)]
    top = ops.TopLogits(values.cuda(), index.cuda(), lse.cuda(), temp)
    ops.generator_distill(*leaves, temp, top, True).sum().backward()
    want = [t.double().requires_grad_() for t in (x, W, b)]
    loss, mass = loss64(torch.nn.functional.linear(*want), values, index, lse, temp, True)
    assert (mass - 1).abs().max() > 1e-3
    loss.sum().backward()
    for got, ref in zip(leaves, want):
        assert (got.grad.cpu().double() - ref.grad).abs().max() <= 1e-4 * ref.grad.abs().max()
