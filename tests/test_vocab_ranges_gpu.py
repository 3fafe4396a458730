"""GPU: the ends of the ranges that ops.top_logits, ops.top_distill and ops.verify_draft state, against plain statements in 64 bits.

A sum of exponentials is within 1e-5 (EPS, relative) up to V = 2^24; a loss within that and its own rounding, a gradient element within 3 EPS
of the magnitudes it is a difference of, half a step of its type and half the smallest step."""
import pytest
import torch

import vocab_oracle as oracle

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs a GPU"
    from nast_amd import ops as o
    return o


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype,R,V,K", [(torch.float32, 2, (1 << 24) - 1, 256), (torch.bfloat16, 1, (1 << 24) - 1, 3), (torch.float16, 3, (1 << 22) + 5, 65)])
def test_distill_longest_rows(ops, dtype, R, V, K, tail):
    gen = torch.Generator(device="cuda").manual_seed(K)
    x = (torch.randn(R, V, generator=gen, device="cuda") * 2.5).to(dtype)
    t = (x.float() + torch.randn(R, V, generator=gen, device="cuda"))
    values, index = t.topk(K, 1)
    index[0, 0], index[0, 1], index[0, 2] = 0, V - 1, V // 2 + 1           # first, last and one between the chunks
    lse = torch.logsumexp(t.double(), 1).float()
    values = values + 8.0                                                   # (most of the mass in the list, less than all of it)
    lse = torch.maximum(lse, torch.logsumexp(values.double(), 1).float() + 0.1)
    g = torch.linspace(0.5, 2.0, R, device="cuda")
    leaf = x.requires_grad_()
    loss = ops.top_distill(leaf, ops.TopLogits(values, index, lse, 1.0), 1.0, tail)
    (grad,) = torch.autograd.grad(loss, leaf, g)
    want, want_grad, scale = oracle.distill(x, values, index, lse, 1.0, tail, g)
    assert ((loss.detach().cpu().double() - want).abs() <= EPS + want.abs() * 2.0 ** -24).all()
    fin = torch.finfo(dtype)
    tol = 3 * EPS * scale + want_grad.abs() * fin.eps / 2 + fin.smallest_normal * fin.eps
    assert ((grad.cpu().double() - want_grad).abs() <= tol).all()


@pytest.mark.parametrize("op", ["top", "distill"])
def test_many_short_rows(ops, op):
    R, V, k = (1 << 22) + 3, 9, 4
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(R, V, generator=gen, device="cuda") * 2
    at = torch.tensor([0, 1, 1 << 20, (1 << 22) - 1, 1 << 22, R - 1], device="cuda")
    top = ops.top_logits(x, k)
    if op == "top":
        order = torch.sort(x, dim=1, descending=True, stable=True)
        assert torch.equal(top.index, order.indices[:, :k]) and torch.equal(top.values, order.values[:, :k])
        want = torch.logsumexp(x.double(), 1)
        assert ((top.lse.double() - want).abs() <= EPS + want.abs() * 2.0 ** -24).all()
        return
    z = (x * 0.9).requires_grad_()
    loss = ops.top_distill(z, top, 1.0, tail=True)
    (grad,) = torch.autograd.grad(loss, z, torch.ones(R, device="cuda"))
    want, want_grad, scale = oracle.distill(z[at], top.values[at], top.index[at], top.lse[at], 1.0, True, torch.ones(6))
    assert ((loss[at].detach().cpu().double() - want).abs() <= EPS + want.abs() * 2.0 ** -24).all()
    assert ((grad[at].cpu().double() - want_grad).abs() <= 3 * EPS * scale + want_grad.abs() * 2.0 ** -24 + 1e-44).all()
    assert grad.double().sum(1).abs().max() <= 3 * EPS * 4                  # (a row's magnitudes add up to 2 + 2 p_r at most)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,N,V", [(2, 1024, 40), (1, 1024, 1201), (1, 3, 1 << 20), (2, 1, (1 << 20) - 3)])
def test_verify_longest(ops, dtype, B, N, V):
    gen = torch.Generator().manual_seed(N + V)
    target = torch.randn(B, N + 1, V, generator=gen) * 2.5
    draft = (target[:, :N] + torch.randn(B, N, V, generator=gen) * 0.02).to(dtype)
    target = target.to(dtype)
    q = torch.softmax(draft.double(), -1)
    tokens = (q / torch.empty(B, N, V, dtype=torch.float64).exponential_(generator=gen)).argmax(-1)
    u, E = torch.rand(B, N, generator=gen) * 0.98, torch.empty(B, V).exponential_(generator=gen)
    u[0, -1] = 1.5                                                           # the last draft of the first sequence falls, if not one before
    for q_, u_ in ((draft, u), (draft, u * 0.5), (None, u * 0)):
        out, accepted = ops.verify_draft(*(None if t is None else t.cuda() for t in (target, tokens, u_, E, q_)))
        want_out, want = oracle.verify(target, tokens, u_, E, q_, None, 1.0)
        assert torch.equal(accepted.cpu(), want) and torch.equal(out.cpu(), want_out)
