"""GPU: ops.top_logits, ops.top_distill and ops.verify_draft against plain 64-bit statements (vocab_oracle).

Tolerances.  EPS bounds the relative error of a sum of exponentials: each exponential is within 1.2e-6 (its argument, down to -30 in
units of log 2 before it stops to matter, is rounded once: 30 * 2^-24 * ln 2, plus one unit of the instruction), a thread adds at
most 128 vectors of 8 in fp32 (136 * 2^-24 = 8.1e-6), everything across threads is in double: below 1e-5 in all.  A log-sum-exp then is
within EPS plus its own rounding; a loss, whose derivative by the log of the rest's sum is q_r - p_r and below 1, the same; a gradient
element is a sum of terms of sizes q_v, p_r q_v / q_r, p_v, each within 3 EPS (sum, quotient and exponential), then rounded to its
type: half a step, torch.finfo(t).eps / 2, and half the smallest step where it leaves the normal range."""
import math

import pytest
import torch

import vocab_oracle as oracle

pytestmark = pytest.mark.gpu
EPS = 1e-5
INF = math.inf
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs a GPU"
    from nast_amd import ops as o
    return o


def rows(R, V, dtype, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(R, V, generator=g) * scale).to(dtype).cuda()


def check_top(ops, x, k, temp=1.0):
    got = ops.top_logits(x, k, temp)
    index, lse = oracle.top(x, k, temp)
    assert got.values.dtype == x.dtype and got.index.dtype == torch.int64 and got.lse.dtype == torch.float32
    assert got.values.shape == x.shape[:-1] + (k,) and got.index.shape == got.values.shape and got.lse.shape == x.shape[:-1]
    assert torch.equal(got.index.cpu().reshape(-1, k), index)
    flat = x.detach().reshape(-1, x.shape[-1])
    want = flat.gather(1, index.cuda()).float()
    assert torch.equal(got.values.float().reshape(-1, k).nan_to_num(9e9), want.nan_to_num(9e9))
    lse_got = got.lse.cpu().double().reshape(-1)
    over = lse.isfinite() & lse.float().isinf()           # beyond fp32's largest number, 3.4e38: its rounding is an infinity
    assert torch.equal(lse_got[over], lse[over].float().double())
    lse, lse_got = lse[~over], lse_got[~over]
    fine = lse.isfinite()
    assert torch.equal(lse_got[~fine].isnan(), lse[~fine].isnan() | (lse[~fine] == INF))
    assert ((lse_got - lse).abs()[fine] <= EPS + lse.abs()[fine] * 2.0 ** -24).all()
    return got


# ------------------------------------------------------------------------------------------------
# top logits
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (2, 8, 8), (4, 9, 1), (3, 255, 255), (2, 256, 256), (2, 300, 256), (7, 1001, 17),
                                   (3, 4096, 64), (2, 9600, 32), (2, 9601, 200), (1, 32767, 256), (1, 32769, 5), (1, 70001, 64)])
def test_top_logits(ops, dtype, R, V, k):
    check_top(ops, rows(R, V, dtype, R * V + k), k, 1.0 if V % 2 else 0.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [1, 40, 256])
@pytest.mark.parametrize("kind", ["equal", "two values", "-inf", "few", "lowest", "nan", "inf", "zeros", "sorted", "block", "reversed"])
def test_top_logits_unusual_rows(ops, dtype, k, kind):
    V = 5003
    x = rows(3, V, dtype, k)
    low = torch.finfo(dtype).min
    if kind == "equal":
        x[:] = 0.37
    elif kind == "two values":
        x[:] = torch.where(torch.arange(V, device="cuda") % 3 == 0, 1.0, -1.0).to(dtype)
    elif kind == "-inf":
        x[1] = -INF
    elif kind == "few":                                   # fewer tokens than k: the -inf ones with the lowest ids fill up
        x[:, 5:-7] = -INF
    elif kind == "lowest":
        x[0, 100:] = low
        x[1] = low
    elif kind == "nan":
        x[0, 17] = float("nan")
        x[1] = float("nan")
        x[2, ::7] = -float("nan")
    elif kind == "inf":
        x[0, 4000] = INF
        x[1, ::2] = INF
    elif kind == "zeros":                                 # -0 equals +0
        x[:] = torch.where(torch.arange(V, device="cuda") % 2 == 0, -0.0, 0.0).to(dtype)
    elif kind == "sorted":
        x = x.sort(1, descending=True).values
    elif kind == "reversed":
        x = x.sort(1).values
    else:                                                 # the large ones side by side
        x[:, 2000:2400] += 30
    check_top(ops, x, k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_top_logits_strides_and_alignment(ops, dtype):
    base = rows(24, 1003, dtype, 3)
    check_top(ops, base[:, 1:], 9)
    check_top(ops, base[:, 3:500], 9)
    check_top(ops, base[::3, 5:], 9)
    check_top(ops, base.view(4, 6, 1003)[:, 1:], 9)
    check_top(ops, base.view(4, 6, 1003)[1:, 2:4, 7:], 9, 2.0)
    check_top(ops, base.view(2, 3, 4, 1003)[:, :, 1:], 9)
    check_top(ops, base[0], 9)
    check_top(ops, base[:1].expand(5, 1003), 9)
    assert ops.top_logits(base[:0], 4).values.shape == (0, 4)
    assert ops.top_logits(base.view(4, 6, 1003)[:, :0], 4).lse.shape == (4, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_top_logits_largest(ops, dtype):
    """the longest rows and lists: as many entries to join as there can be; ties, a NaN and -inf across the chunks"""
    V, k = 1 << 20, 256
    x = rows(5, V, dtype, 1)
    x[1] = 0.5
    x[2] = x[2].sort(descending=True).values
    x[3, ::4097] = float("nan")
    x[4, 100:-100] = -INF
    check_top(ops, x, k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_top_logits_nans_in_one_chunk(ops, dtype):
    """chunks that go different ways: NaNs in one (more of them than the join keeps), equal values in another, signalling NaNs alone"""
    V = 70001
    for k in (1, 64, 256):
        x = rows(4, V, dtype, k)
        x[0, :5000] = float("nan")
        x[1, 40000:] = 1.25
        x[2, 30000:30003] = float("nan")
        kind = torch.int32 if dtype == torch.float32 else torch.int16
        x[3] = torch.full((V,), {torch.float32: 0x7fa00000, torch.bfloat16: 0x7fa0, torch.float16: 0x7d00}[dtype], dtype=kind, device="cuda").view(dtype)
        check_top(ops, x, k)
        check_top(ops, x[:, :1500], k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V", [(257, 9001), (12, 9001), (12, 40001), (12, 65536), (12, 65537)])
def test_top_logits_unusual_long_rows(ops, dtype, R, V):
    """a row of each kind, in chunks and whole, at every alignment"""
    for k in (1, 64, 256):
        x = rows(R, V + 3, dtype, k)
        x[0] = 0.37
        x[1, ::3] = 9.0
        x[2] = -INF
        x[3, 5:-7] = -INF
        x[4, 100:] = torch.finfo(dtype).min
        x[5, ::7] = -float("nan")
        x[6, ::2] = INF
        x[7] = torch.where(torch.arange(V + 3, device="cuda") % 2 == 0, -0.0, 0.0).to(dtype)
        x[8] = x[8].sort(descending=True).values
        x[9] = x[9].sort().values
        x[10, 2000:2400] += 30
        for lead in (0, 1, 3):
            check_top(ops, x[:, lead:lead + V], k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temp", [1.0, 1e-3, 1e-6, 1e20])
def test_top_logits_magnitudes(ops, dtype, temp):
    """rows whose largest logit over the temperature is tiny, around 2^24 and far beyond, of both signs"""
    x = rows(12, 9001, dtype, 8)
    for r, (scale, shift) in enumerate([(1e-6, 0), (1, 0), (1, 300), (1, -300), (1e3, 0), (100, 6e4), (100, -6e4), (1, 11629), (4, 23256)]):
        x[r] = (x[r].float() * scale + shift).to(dtype)
    if dtype != torch.float16:
        x[9] = x[9] * 1e8
        x[10] = x[10] * 1e37
        x[11] = -x[11].abs() * 1e37
    for n in (9001, 700):
        check_top(ops, x[:, :n], 16, temp)


def test_top_logits_far_offsets(ops):
    """rows that lie beyond 2^31 elements of their tensor"""
    R, V = 20000, 120000
    x = torch.empty(R, V, dtype=torch.bfloat16, device="cuda").zero_()
    at = torch.tensor([0, 9999, 17900, 19999], device="cuda")
    x[at] = rows(4, V, torch.bfloat16, 5)
    got = ops.top_logits(x, 8)
    index, lse = oracle.top(x[at[1:]], 8, 1.0)
    assert torch.equal(got.index[at[1:]].cpu(), index)
    assert ((got.lse[at[1:]].cpu().double() - lse).abs() <= EPS + lse.abs() * 2.0 ** -24).all()
    assert torch.equal(got.index[5], torch.arange(8, device="cuda"))
    logits = x.requires_grad_()
    top = ops.TopLogits(got.values, got.index, got.lse, 1.0)
    loss = ops.top_distill(logits, top, 1.0, tail=True)
    (grad,) = torch.autograd.grad(loss[-1] * 3.0, logits)
    want = oracle.distill(x[-1:], got.values[-1:], got.index[-1:], got.lse[-1:], 1.0, True, torch.tensor([3.0]))
    check_grad(grad[-1:], want[1], want[2])
    assert int(torch.count_nonzero(grad[:-1:1999])) == 0


# ------------------------------------------------------------------------------------------------
# distillation
# ------------------------------------------------------------------------------------------------
def check_grad(got, want, scale):
    fin = torch.finfo(got.dtype)
    got = got.detach().cpu().double().reshape(want.shape)
    assert torch.equal(got.isnan(), want.isnan())
    tol = 3 * EPS * scale + want.abs() * fin.eps / 2 + fin.smallest_normal * fin.eps
    worst = ((got - want).abs() / tol.clamp(min=1e-300)).nan_to_num(0.0).max()
    assert worst <= 1, f"gradient off by {worst:.3g} of its tolerance"


def check_distill(ops, x, values, index, lse, temp, tail, g=None):
    lead = x.shape[:-1]
    if g is None:
        g = torch.linspace(0.25, 1.5, max(1, lead.numel()), device="cuda")[:lead.numel()].view(lead)
    leaf = x.detach().requires_grad_()
    loss = ops.top_distill(leaf, ops.TopLogits(values, index, lse, temp), temp, tail=tail)
    assert loss.dtype == torch.float32 and loss.shape == lead
    (grad,) = torch.autograd.grad(loss, leaf, g)
    assert grad.dtype == x.dtype and grad.shape == x.shape
    wl, wg, ws = oracle.distill(x, values, index, lse, temp, tail, g)
    got = loss.detach().cpu().double().reshape(-1)
    assert torch.equal(got.isnan(), wl.isnan()) and torch.equal(got == INF, wl == INF)
    fine = wl.isfinite()
    assert ((got - wl).abs()[fine] <= EPS + wl.abs()[fine] * 2.0 ** -24).all(), (got, wl)
    check_grad(grad, wg, ws)
    return loss.detach(), grad


def teacher_of(x, k, temp, seed, dtype=None):
    t = (x.float() + torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)).cuda()).to(dtype or x.dtype)
    v, i = t.float().topk(k, -1)
    return v.to(t.dtype), i, torch.logsumexp(t.double() / temp, -1).float()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (3, 2, 1), (5, 7, 3), (2, 8, 7), (4, 9, 1), (2, 300, 256), (7, 1001, 17), (2, 9600, 32), (2, 9601, 200),
                                   (1, 32759, 20), (1, 32760, 20), (2, 32761, 20), (1, 70001, 64)])
def test_top_distill(ops, dtype, tail, R, V, k):
    temp = (1.0, 2.0, 0.6)[(R + V) % 3]
    x = rows(R, V, dtype, R * V + k)
    check_distill(ops, x, *teacher_of(x, k, temp, 1, DTYPES[(V + k) % 3]), temp, tail)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_top_distill_slots(ops, dtype, tail):
    """lists that end early, empty lists, ids outside the vocabulary, an id twice, teacher logits of -inf, all tokens listed"""
    V, K, temp = 203, 12, 1.5
    x = rows(9, V, dtype, 5)
    values, index, lse = teacher_of(x, K, temp, 2)
    index[0, 4:] = -1
    index[1] = -1
    index[2, 0], index[2, 5] = V, -7
    index[3, 7] = index[3, 2]
    index[4, 3] = index[4, 4] = index[4, 11] = index[4, 9]
    values[5, 2:] = -INF
    values[6] = -INF
    index[7] = torch.arange(K, device="cuda") % 3                        # three tokens, four times each
    index[8, :] = torch.iinfo(torch.int64).max
    loss, grad = check_distill(ops, x, values, index, lse, temp, tail)
    for r in (1, 6, 8):
        assert loss[r] == 0 and not grad[r].any()
    x = rows(2, K, dtype, 6)
    v, i, _ = teacher_of(x, K, temp, 3)
    check_distill(ops, x, v, i, torch.logsumexp(v.double() / temp, 1).float() + 0.25, temp, tail)     # nothing left for the bucket
    check_distill(ops, rows(3, 40, dtype, 8), v[:1].expand(3, K), i[:1].expand(3, K), lse[:3], temp, tail)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("K", [40, 65, 256])
@pytest.mark.parametrize("V", [9600, 16383, 16384, 40001])
def test_top_distill_ids_in_many_slots(ops, V, K, tail):
    """the same id in slots of one wavefront and of several, once, twice and everywhere, in rows beside others without"""
    dtype = DTYPES[(V + K) % 3]
    x = rows(5, V, dtype, K)
    values, index, lse = teacher_of(x, K, 1.0, 2)
    values = values - 2.0                                                # (some of them twice stay below a sum of one)
    index[0, K // 2:2 * (K // 2)] = index[0, :K // 2]
    index[1, 1::13] = index[1, 0]
    index[2, -1] = index[2, 0]
    index[3] = index[3, 0]
    check_distill(ops, x, values, index, lse, 1.0, tail)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_top_distill_unusual_rows(ops, dtype, tail):
    V, K, temp = 1003, 6, 1.0
    x = rows(9, V, dtype, 7)
    values, index, lse = teacher_of(x, K, temp, 2)
    x[0, 500:] = -INF
    x[0, index[0]] = 1.0
    x[1] = -INF
    x[1, index[1]] = 2.0                                                 # only listed tokens
    x[2, index[2, 3]] = -INF                                             # the student rules a teacher's token out: infinite loss
    x[3, 9] = float("nan")
    x[4] = torch.finfo(dtype).min
    x[5, index[5]] += 60                                                 # next to nothing outside the list
    x[6] = -INF
    x[7, 3] = INF
    x[8, index[8]] -= 60                                                 # next to nothing inside it
    check_distill(ops, x, values, index, lse, temp, tail)
    # rows of no weight, and rows without a list, are zeros whatever they hold
    index[3] = index[6] = -1
    g = torch.ones(9, device="cuda")
    g[7] = g[2] = 0
    loss, grad = check_distill(ops, x, values, index, lse, temp, tail, g)
    assert loss[3] == 0 and loss[6] == 0
    for r in (2, 3, 6, 7):
        assert not grad[r].any()


@pytest.mark.parametrize("tail", [False, True])
def test_top_distill_small_loss(ops, tail):
    """one slot of p ~ 0.01: a loss of ~1e-4 made of terms near 1 keeps its digits.  The rest's sum is known to EPS and enters with
    q_r - p_r ~ 2e-3, the slot's terms are in double: an error of 2e-3 * EPS = 2e-8."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(6, 20000, generator=g).cuda()
    x[:, 77] = 5.5
    t = x.clone()
    t[:, 77] += 0.2
    lse = torch.logsumexp(t.double(), 1).float()
    index = torch.full((6, 1), 77, device="cuda")
    got = ops.top_distill(x, ops.TopLogits(t[:, 77:78].contiguous(), index, lse, 1.0), 1.0, tail=True).cpu().double()
    want = oracle.distill(x, t[:, 77:78], index, lse, 1.0, True, torch.ones(6))[0]
    assert want.max() < 1e-3
    assert ((got - want).abs() <= 2e-8 + want * 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_top_distill_strides(ops, dtype):
    base = rows(24, 1003, dtype, 3)
    for x in (base[:, 1:], base[::3, 5:], base.view(4, 6, 1003)[:, 1:], base.view(4, 6, 1003)[1:, 2:4, 7:], base.view(2, 3, 4, 1003)[:, :, 1:],
              base[0], base[:1].expand(5, 1003)):
        v, i, lse = teacher_of(x.contiguous(), 9, 1.0, 4)
        check_distill(ops, x, v, i, lse, 1.0, True)
    x = base.view(4, 6, 1003)
    v, i, lse = teacher_of(x, 10, 1.0, 4)
    check_distill(ops, x, v[..., ::2], i[..., ::2], lse, 1.0, True)
    empty = ops.top_distill(base[:0].requires_grad_(), ops.TopLogits(v[0, :0], i[0, :0], lse[0, :0], 1.0))
    assert empty.shape == (0,)
    empty.sum().backward()


def test_top_distill_large_gradient(ops):
    """a gradient larger than the last-level cache, rows picked from it"""
    R, V, K = 600, 131075, 9
    x = rows(R, V, torch.float32, 5).requires_grad_()
    index = torch.randint(0, V, (R, K), generator=torch.Generator().manual_seed(1)).cuda()
    index[:, 3] = index[:, 4]
    values = x.detach().gather(1, index) + 3.0
    lse = torch.logsumexp(x.detach(), 1) + 2.5
    g = torch.rand(R, device="cuda")
    for tail in (False, True):
        loss = ops.top_distill(x, ops.TopLogits(values, index, lse, 1.0), 1.0, tail=tail)
        (grad,) = torch.autograd.grad(loss, x, g)
        pick = torch.tensor([0, 1, 299, R - 1], device="cuda")
        wl, wg, ws = oracle.distill(x.detach()[pick], values[pick], index[pick], lse[pick], 1.0, tail, g[pick])
        assert ((loss[pick].detach().cpu().double() - wl).abs() <= EPS + wl.abs() * 2.0 ** -24).all()
        check_grad(grad[pick], wg, ws)


def test_top_distill_autograd(ops):
    """the graph kept and walked twice, a broadcast leaf, a leaf changed in between, a second derivative refused"""
    x = rows(1, 77, torch.float32, 4).requires_grad_()
    v, i, lse = teacher_of(x.detach().expand(6, 77).contiguous(), 5, 1.0, 2)
    top = ops.TopLogits(v, i, lse, 1.0)
    loss = ops.top_distill(x.expand(6, 77), top, 1.0, tail=True).sum()
    (a,) = torch.autograd.grad(loss, x, retain_graph=True)
    (b,) = torch.autograd.grad(loss, x)
    want = oracle.distill(x.detach().expand(6, 77), v, i, lse, 1.0, True, torch.ones(6))
    assert torch.equal(a, b)
    check_grad(a, want[1].sum(0, keepdim=True), want[2].sum(0, keepdim=True) + 6 * want[1].abs().sum(0, keepdim=True) * 2.0 ** -24 / EPS)
    leaf = rows(6, 77, torch.float32, 4).requires_grad_()
    loss = ops.top_distill(leaf, top).sum()
    with torch.no_grad():
        leaf.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    w = torch.ones(6, device="cuda", requires_grad=True)
    (first,) = torch.autograd.grad((ops.top_distill(leaf, top) * w).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first.sum().backward()


def test_refusals(ops):
    from nast_amd._lib import NastHipError
    x = rows(4, 50, torch.float32, 1)
    for bad, match in ((x.double(), "fp32, bf16 or fp16"), (x.long(), "fp32, bf16 or fp16"), (x.t(), "contiguous"), (x[:, :0], "vocabulary axis"),
                       (torch.tensor(1.0, device="cuda"), "vocabulary axis")):
        with pytest.raises(NastHipError, match=match):
            ops.top_logits(bad, 1)
        with pytest.raises(NastHipError, match=match):
            lead = bad.shape[:-1] if bad.dim() else ()
            ops.top_distill(bad, ops.TopLogits(torch.zeros(*lead, 1, device="cuda"), torch.zeros(*lead, 1, dtype=torch.int64, device="cuda"), None, 1.0))
    for k in (0, -1, 51, 257):
        with pytest.raises(NastHipError, match="k="):
            ops.top_logits(x, k)
    with pytest.raises(NastHipError, match="temperature"):
        ops.top_logits(x, 1, 0.0)
    with pytest.raises(NastHipError, match="bad sizes"):
        ops.top_logits(torch.zeros(1, (1 << 20) + 1, device="cuda"), 1)
    top = ops.top_logits(x, 3)
    with pytest.raises(NastHipError, match="two devices"):
        ops.top_distill(x, top._replace(index=top.index.cpu()))
    with pytest.raises(NastHipError, match="temperature"):
        ops.top_distill(x, top, 2.0, tail=True)
    target, tokens, u, E, draft = drafts(2, 3, 50, torch.float32, 1)
    good = dict(target=target, tokens=tokens, u=u, E=E, draft=draft, lengths=None, temperature=1.0)
    for name, bad, match in (("target", target[0], "B, N"), ("target", target.double(), "fp32, bf16"), ("tokens", tokens.int(), "tokens"),
                             ("tokens", tokens[:, :2], "tokens"), ("u", u.double(), "u:"), ("u", u[:1], "u:"), ("E", E[:, :49], "E:"),
                             ("E", E.half(), "E:"), ("draft", draft.half(), "draft"), ("draft", target, "draft"), ("lengths", torch.ones(2, device="cuda"), "lengths"),
                             ("lengths", torch.ones(3, dtype=torch.int64, device="cuda"), "lengths"), ("temperature", 0.0, "temperature"),
                             ("E", E.cpu(), "two devices"), ("draft", draft.cpu(), "two devices")):
        with pytest.raises(NastHipError, match=match):
            ops.verify_draft(**{**good, name: bad})


def test_top_distill_differences(ops):
    """the gradient against central differences of the loss: a loss within 2e-7 divided by 2h = 0.05, plus h^2 / 6 of a third
    derivative below 0.2"""
    x = rows(1, 11, torch.float32, 1)
    v, i, lse = teacher_of(x, 4, 1.3, 2)
    i[0, 3] = i[0, 1]
    for tail in (False, True):
        top = ops.TopLogits(v, i, lse, 1.3)
        leaf = x.clone().requires_grad_()
        ops.top_distill(leaf, top, 1.3, tail=tail).backward(torch.ones(1, device="cuda"))
        for e in range(11):
            a, b = x.clone(), x.clone()
            a[0, e] += 0.025
            b[0, e] -= 0.025
            h = (a[0, e] - b[0, e]).item()
            d = (ops.top_distill(a, top, 1.3, tail=tail) - ops.top_distill(b, top, 1.3, tail=tail)).item() / h
            assert abs(d - leaf.grad[0, e].item()) < 1e-4


def test_generator_distill_refusals_and_no_rows(ops):
    top = ops.TopLogits(torch.zeros(2, 3, device="cuda"), torch.zeros(2, 3, device="cuda", dtype=torch.int64), None, 1.0)
    x, W, b = torch.randn(2, 16, device="cuda"), torch.randn(40, 16, device="cuda"), torch.zeros(40, device="cuda")
    for bad in ((x, W[:, :8].contiguous(), b), (x, W, b[:39]), (x, W[:, ::2], b), (x, W.t().contiguous().t(), b), (x[:1], W, b), (x.half(), W, b)):
        with pytest.raises(ops._lib.NastHipError):
            ops.generator_distill(*bad, 1.0, top)
    none = ops.TopLogits(top.values[:0], top.index[:0], None, 1.0)
    leaves = [t.clone().requires_grad_() for t in (x[:0], W, b)]
    loss = ops.generator_distill(*leaves, 1.0, none)
    assert loss.shape == (0,)
    loss.sum().backward()
    assert all(t.grad is None or not t.grad.any() for t in leaves)


def test_generator_top_and_distill(ops):
    """Generator.distill against autograd of a plain statement in 64 bits; fp32 products over K = 64: relative 1e-4 as elsewhere"""
    from nast_amd import transformer as tf
    torch.manual_seed(2)
    d, V, K, temp = 64, 1001, 20, 1.7
    teacher, student = tf.Generator(d, V).cuda(), tf.Generator(d, V).cuda()
    x = torch.randn(3, 5, d, device="cuda")
    top = teacher.top(x, temp, K)
    tl = torch.nn.functional.linear(x.double(), teacher.proj.weight.double(), teacher.proj.bias.double())
    assert not top.values.requires_grad and top.temperature == temp
    assert (top.values.double() - tl.gather(-1, top.index)).abs().max() < 1e-4
    for tail in (False, True):
        student.zero_grad()
        xs = x.clone().requires_grad_()
        w = torch.rand(3, 5, device="cuda")
        loss = student.distill(xs, temp, top, tail)
        (loss * w).sum().backward()
        xr, W, b = (t.detach().double().requires_grad_() for t in (x, student.proj.weight, student.proj.bias))
        z = torch.nn.functional.linear(xr, W, b) / temp
        logq, t = torch.log_softmax(z, -1), top.values.double() / temp
        logp = t - (top.lse.double() if tail else torch.logsumexp(t, -1)).unsqueeze(-1)
        ref = (logp.exp() * (logp - logq.gather(-1, top.index))).sum(-1)
        if tail:
            pr = 1 - logp.exp().sum(-1)
            outside = torch.ones_like(logq).scatter(-1, top.index, 0.0)
            ref = ref + pr * (pr.log() - (logq.exp() * outside).sum(-1).log())
        (ref * w).sum().backward()
        assert (loss.double() - ref).abs().max() < 1e-4 * ref.abs().max()
        for got, want in ((xs.grad, xr.grad), (student.proj.weight.grad, W.grad), (student.proj.bias.grad, b.grad)):
            assert (got.double() - want).abs().max() < 1e-4 * want.abs().max()


# ------------------------------------------------------------------------------------------------
# verification
# ------------------------------------------------------------------------------------------------
def drafts(B, N, V, dtype, seed, noise=0.5, temp=1.0, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    target = (torch.randn(B, N + 1, V, generator=g) * scale)
    draft = target[:, :N] + torch.randn(B, N, V, generator=g) * noise
    target, draft = target.to(dtype), draft.to(dtype)
    q = torch.softmax(draft.double() / temp, -1)
    tokens = (q / torch.empty(B, N, V, dtype=torch.float64).exponential_(generator=g)).argmax(-1) if N else torch.zeros(B, 0, dtype=torch.int64)
    u, E = torch.rand(B, N, generator=g), torch.empty(B, V).exponential_(generator=g)
    return [t.cuda() for t in (target, tokens, u, E, draft)]


def check_verify(ops, target, tokens, u, E, draft=None, lengths=None, temp=1.0):
    out, accepted = ops.verify_draft(target, tokens, u, E, draft, lengths, temp)
    wo, wa = oracle.verify(target, tokens, u, E, draft, lengths, temp)
    assert torch.equal(accepted.cpu(), wa), (accepted.cpu(), wa)
    assert torch.equal(out.cpu(), wo), (out.cpu(), wo)
    return out, accepted


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,N,V", [(1, 0, 5), (1, 1, 1), (3, 2, 2), (5, 3, 7), (4, 8, 1001), (2, 65, 33), (2, 130, 9), (3, 4, 9600), (1, 3, 32769), (2, 2, 70001),
                                   (300, 3, 129)])
def test_verify_draft(ops, dtype, B, N, V):
    temp = (1.0, 0.7, 1.9)[(B + N) % 3]
    target, tokens, u, E, draft = drafts(B, N, V, dtype, B * V + N, temp=temp)
    lengths = torch.randint(0, N + 1, (B,), generator=torch.Generator().manual_seed(N)).cuda()
    check_verify(ops, target, tokens, u, E, draft, None, temp)
    check_verify(ops, target, tokens, u, E, draft, lengths, temp)
    check_verify(ops, target, tokens, u, E, None, lengths, temp)
    check_verify(ops, target, target[:, :N].argmax(-1), u, E, None, None, temp)
    check_verify(ops, target, tokens, u * 0, E, draft, lengths - 1, temp)          # a length below 0 counts as 0
    check_verify(ops, target, tokens, u, E, target[:, :N], lengths + N, temp)      # the target as its own drafter: everything stands


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 5003, 40001])
def test_verify_draft_filtered_rows(ops, dtype, V):
    """improbable words cut off (-inf) on both sides, most of what is drawn from has no probability in the draft"""
    for seed in range(6):
        target, tokens, u, E, draft = drafts(16, 3, V, dtype, seed + V, noise=0.8)
        target = target.masked_fill(target < target.amax(-1, keepdim=True) - 7, -INF)
        draft = draft.masked_fill(draft < draft.amax(-1, keepdim=True) - 6, -INF)
        lengths = (torch.arange(16) % 4).cuda()
        check_verify(ops, target, draft.argmax(-1), u, E, draft, lengths, 0.8)
        check_verify(ops, target, tokens, u, E, None, lengths, 0.8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_verify_draft_unusual_rows(ops, dtype):
    B, N, V = 12, 3, 501
    target, tokens, u, E, draft = drafts(B, N, V, dtype, 11, noise=0.3)
    u[:] = 0.2
    low = torch.finfo(dtype).min
    target[0, 1, 5] = float("nan")
    target[1, 0] = -INF
    target[2, 0, 7] = INF
    draft[3, 0] = -INF
    draft[4, 0, 3] = float("nan")
    tokens[5, 0], tokens[6, 1], tokens[7, 0] = -1, V, torch.iinfo(torch.int64).min
    draft[8, 0, tokens[8, 0]] = -INF
    target[9, 0, tokens[9, 0]] = -INF
    target[10, :, 2:] = low
    draft[10, :, 2:] = low
    target[11] = low
    check_verify(ops, target, tokens, u, E, draft)
    check_verify(ops, target, tokens, u, E, None)
    target[:, 3] = -INF                                       # nothing to draw from behind the last draft
    check_verify(ops, target, target[:, :N].argmax(-1), u * 0, E, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [64, 40000])
def test_verify_draft_borders(ops, dtype, V):
    """comparisons that fp32 cannot decide: a ratio next to u, equal scores, p and q nearly the same, a residual of nothing"""
    target = torch.zeros(4, 2, V, dtype=dtype, device="cuda")            # p = 1/V everywhere
    draft = torch.zeros(4, 1, V, dtype=dtype, device="cuda")
    draft[:, :, V // 2:] = -INF                                          # q = 2/V on the lower half: ratio 1/2
    tokens = torch.zeros(4, 1, dtype=torch.int64, device="cuda")
    half = torch.tensor(0.5)
    u = torch.stack([torch.nextafter(half, half * 0), torch.nextafter(half, half * 2), half * 0, half * 2]).view(4, 1).cuda()
    E = torch.ones(4, V, device="cuda")                                  # all scores equal: the lowest id of the upper half
    out, accepted = check_verify(ops, target, tokens, u, E, draft)
    assert accepted.tolist() == [1, 0, 1, 0]
    assert out[1].tolist() == [V // 2, -1] and out[0].tolist() == [0, 0]
    # u of 1 or more, or NaN, refuses a token that p and q agree on: nothing is left of p - q, the draw is made from p
    same = rows(4, 2 * V, dtype, 2).view(4, 2, V)
    check_verify(ops, same, tokens, torch.full((4, 1), 1.5, device="cuda"), E, same[:, :1].contiguous())
    check_verify(ops, same, tokens, torch.full((4, 1), float("nan"), device="cuda"), E, same[:, :1].contiguous())
    # two tokens whose scores differ in the last bit of fp32 or not at all
    E = torch.ones(4, V, device="cuda")
    E[:, 9] = torch.nextafter(torch.tensor(1.0), torch.tensor(0.0))
    out, _ = check_verify(ops, target, tokens, u * 0, E, draft)
    assert (out[:, 1] == 9).all()
    E[:, 3] = 0.0                                                        # an Exp(1) draw of 0 wins
    out, _ = check_verify(ops, target, tokens, u * 0, E, draft)
    assert (out[:, 1] == 3).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [64, 40000])
def test_verify_draft_borders_many_places(ops, dtype, V):
    """a ratio of 1/2 at every place: u next to it decides, place after place, clear decisions between"""
    N = 70
    target = torch.zeros(5, N + 1, V, dtype=dtype, device="cuda")
    draft = torch.zeros(5, N, V, dtype=dtype, device="cuda")
    draft[:, :, V // 2:] = -INF
    tokens = torch.arange(N, device="cuda").remainder(V // 2).expand(5, N)
    below = float(torch.nextafter(torch.tensor(0.5), torch.tensor(0.0)))
    u = torch.full((5, N), below, device="cuda")
    u[1, 68], u[2, 3], u[2, 2], u[3, :66], u[4, 66] = 0.5, 0.5, 0.9, 0.1, 0.5
    E = torch.rand(5, V, generator=torch.Generator().manual_seed(3)).add(0.5).cuda()
    _, accepted = check_verify(ops, target, tokens, u, E, draft)
    assert accepted.tolist() == [70, 68, 2, 70, 66]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [600, 40000])
def test_verify_draft_smallest_draws(ops, dtype, V):
    """Exp(1) draws below the smallest normal number (their reciprocal has no fp32), zeros, infinities, the largest number"""
    target, tokens, u, E, draft = drafts(6, 2, V, dtype, 21, noise=0.5)
    at = torch.tensor([V - 1, 7, 311], device="cuda")
    E[0, at] = torch.tensor([1e-40, 2e-40, 3e-45], device="cuda")
    E[1, at] = torch.tensor([1e-40, 1.3e-38, 1e-37], device="cuda")
    E[2, at] = torch.tensor([0.0, 0.0, 1e-44], device="cuda")
    E[3] = 1e-42
    E[4, at] = INF
    E[5] = torch.finfo(torch.float32).max
    for t in (1.0, 0.05):
        check_verify(ops, target, tokens, u, E, draft, None, t)
        check_verify(ops, target, tokens, u * 0 + 2, E, draft, None, t)
        check_verify(ops, target, tokens, u, E, None, None, t)


@pytest.mark.parametrize("dtype", DTYPES)
def test_verify_draft_strides(ops, dtype):
    target, tokens, u, E, draft = drafts(6, 5, 301, dtype, 4)
    check_verify(ops, target[::2, 1:, 3:], tokens[::2, 1:].clamp(max=297), u[::2, 1:], E[::2, 3:], draft[::2, 1:, 3:])
    check_verify(ops, target[:, :, ::2], tokens // 2, u, E[:, ::2], draft[:, :, ::2])
    check_verify(ops, target[:1].expand(6, 6, 301), tokens, u, E, draft[:1].expand(6, 5, 301))
    out, accepted = ops.verify_draft(target[:0], tokens[:0], u[:0], E[:0], draft[:0])
    assert out.shape == (0, 6) and accepted.shape == (0,)


def test_verify_draft_far_offsets(ops):
    """rows that lie beyond 2^31 elements of their tensor"""
    V = 120000
    base = torch.zeros(4500, 4, V, dtype=torch.bfloat16, device="cuda")
    target, tokens, u, E, draft = drafts(4, 3, V, torch.bfloat16, 9)
    base[::1499], base[1::1499, :3] = target, draft
    far_target, far_draft = base[::1499], base[1::1499, :3]
    assert far_target.stride(0) * 3 > 1 << 31
    check_verify(ops, far_target, tokens, u, E, far_draft)
    check_verify(ops, far_target, tokens, u * 0, E, far_draft)


def test_verify_draft_distribution(ops):
    """the tokens that come out follow the target, wherever the drafts came from: frequencies within 5 standard deviations"""
    import nast_amd.utils as U
    torch.manual_seed(5)
    B, V = 40000, 6
    for temp in (1.0, 1.6):
        target = torch.tensor([[0.3, -1.0, 2.0, 0.0, -2.0, 1.0], [1.0, 1.5, -1.0, 0.2, 0.0, -3.0]]).cuda()
        draft = torch.tensor([[1.0, 0.0, 1.0, -1.0, 0.0, -1.0]]).cuda()
        q = torch.softmax(draft[0] / temp, 0)
        tokens = torch.multinomial(q, B, replacement=True).view(B, 1)
        out, accepted = U.verify_draft(target.expand(B, 2, V), tokens, draft.expand(B, 1, V), None, temp)
        p = torch.softmax(target.double() / temp, 1)
        for place, rows_ in ((0, out[:, 0]), (1, out[accepted == 1, 1])):
            n = rows_.numel()
            freq = torch.bincount(rows_, minlength=V).double() / n
            assert ((freq - p[place]).abs() <= 5 * (p[place] * (1 - p[place]) / n).sqrt()).all()
        with U.inject_noise([torch.zeros(4, 1, device="cuda"), torch.ones(4, V, device="cuda")]):
            again, _ = U.verify_draft(target.expand(4, 2, V), tokens[:4], draft.expand(4, 1, V))
        assert torch.equal(again[:, :1], tokens[:4]) and (again[:, 1] == p[1].argmax()).all()


@pytest.mark.parametrize("with_q", [True, False])
def test_verify_draft_in_rounds(ops, with_q):
    """a batch whose rows (320 MB) are read in more than one round, sequences that end in each of them"""
    B, N, V = 64, 24, 50021
    g = torch.Generator(device="cuda").manual_seed(3)
    target = torch.randn(B, N + 1, V, generator=g, device="cuda") * 3
    draft = target[:, :N] + torch.randn(B, N, V, generator=g, device="cuda") * 0.1
    tokens = (draft - torch.empty_like(draft).exponential_(generator=g).log()).argmax(-1)       # drawn from softmax(draft)
    u, E = torch.rand(B, N, generator=g, device="cuda"), torch.empty(B, V, device="cuda").exponential_(generator=g)
    lengths = (torch.arange(B) % (N + 1)).cuda()
    lengths[::2] = N
    if with_q:
        _, accepted = check_verify(ops, target, tokens, u, E, draft, lengths)
    else:                                                                # the likeliest tokens, p around 0.1, against u below 0.05
        _, accepted = check_verify(ops, target, target[:, :N].argmax(-1), u * 0.05, E, None, lengths)
    assert (accepted < 5).any() and (accepted > 11).any() and len(set(accepted.tolist())) > 6


# ------------------------------------------------------------------------------------------------
# together, on other streams, in graphs
# ------------------------------------------------------------------------------------------------
def _chain(ops, teacher, student, E, u, draft_tokens):
    top = ops.top_logits(teacher, 12, 1.0)
    loss = ops.top_distill(student, top, 1.0, tail=True)
    (grad,) = torch.autograd.grad(loss.sum(), student)
    n = teacher.shape[1] - 1
    out, accepted = ops.verify_draft(teacher, draft_tokens, u, E, student.detach()[:, :n])
    return [top.values, top.index, top.lse, loss.detach(), grad, out, accepted]


def _chain_inputs(seed, V=5001):
    teacher, tokens, u, E, draft = drafts(4, 3, V, torch.bfloat16, seed)
    student = torch.cat((draft, draft[:, :1]), 1).requires_grad_()
    return teacher, student, E, u, tokens


def test_chain_on_streams(ops):
    """the operators after one another, on two streams at once, equal the same on the default stream"""
    inputs = [_chain_inputs(s) for s in (1, 2)]
    want = [_chain(ops, *i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    for _ in range(3):
        got = []
        for s, i in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append(_chain(ops, *i))
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            assert all(torch.equal(a, b) for a, b in zip(w, g))


@pytest.mark.parametrize("V", [501, 40001])
def test_chain_in_graphs(ops, V):
    """captured twice, replayed in turn with new inputs, beside eager work"""
    batches = [_chain_inputs(s, V) for s in range(4)]
    static = [[t.detach().clone().requires_grad_(t.requires_grad) for t in b] for b in batches[:2]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in static:
            _chain(ops, *s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_chain(ops, *s))
        graphs.append(g)
    for turn in range(4):
        now = [batches[turn], batches[(turn + 1) % 4]]
        for s, b in zip(static, now):
            for t, v in zip(s, b):
                t.detach().copy_(v.detach())
        want = [_chain(ops, *b) for b in now]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert all(torch.equal(a, b) for a, b in zip(w, o))
        ops.top_logits(batches[turn][0], 5)


@pytest.mark.parametrize("packed", [False, True])
def test_style_transformer_distills(ops, packed):
    """StyleTransformer.forward(teacher_top=): the loss of its own log-probabilities against the teacher's list, its gradients those of
    the plain statement on the log-probabilities; padded and packed execution"""
    from helpers import make_param, synth_batch
    from nast_amd import transformer as tf
    import numpy as np
    torch.manual_seed(3)
    V, L, B, K = 60, 10, 6, 7
    F = tf.StyleTransformer(make_param(V=V, d=64, h=4, N=2, L=L, learnable=True)).cuda()
    with torch.no_grad():
        for p in F.parameters():
            if p.dim() == 1:
                p.add_(torch.randn_like(p) * 0.1)
    sent, lens = (t.cuda() for t in synth_batch(np.random.default_rng(1), B, L, V))
    style = (torch.arange(B) % 2).cuda()
    mask = (torch.arange(L, device="cuda") < lens.unsqueeze(1)).float()
    teacher = torch.randn(B, L, V, device="cuda") * 3
    top = ops.top_logits(teacher, K, 1.0)
    args = dict(generate=False, temperature=1.0, use_inference_z=True)
    for tail in (False, True):
        F.zero_grad()
        lp = F(sent, lens, sent, lens, style, **args)[0]
        logq = lp.double()
        logp = top.values.double() - (top.lse.double() if tail else torch.logsumexp(top.values.double(), -1)).unsqueeze(-1)
        ref = (logp.exp() * (logp - logq.gather(-1, top.index))).sum(-1)
        if tail:
            pr = (1 - logp.exp().sum(-1)).clamp(min=1e-30)
            ref = ref + pr * (pr.log() - (logq.exp() * torch.ones_like(logq).scatter(-1, top.index, 0.0)).sum(-1).log())
        (ref * mask).sum().backward()
        want = {n: p.grad.clone() for n, p in F.named_parameters() if p.grad is not None}
        F.zero_grad()
        with ops.packed_rows(packed):
            loss = F(sent, lens, sent, lens, style, teacher_top=top, teacher_tail=tail, **args)[0]
        assert ((loss.double() - ref) * mask).abs().max() < 1e-4 * (ref * mask).abs().max()
        (loss * mask).sum().backward()
        largest = max(g.abs().max() for g in want.values())      # the scale: gradients of key biases are rounding noise
        for n, p in F.named_parameters():
            if n in want:
                assert (p.grad - want[n]).abs().max() <= 1e-4 * largest, n
    from nast_amd import _lib
    with pytest.raises(_lib.NastHipError, match="teacher_top"):
        F(sent, lens, sent, lens, style, teacher_top=top, nll_targets=sent, **args)
    with pytest.raises(_lib.NastHipError):
        with ops.packed_rows(packed):
            F(sent, lens, sent, lens, style, teacher_top=ops.top_logits(teacher[:, :-1], K, 1.0), **args)
