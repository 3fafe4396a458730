"""GPU: the bounds of error behind ops.verify_draft's decisions, on the rows that strain them: maxima that rise a little from chunk to
chunk and from batch to batch, so that a sum is brought to a larger maximum as often as it can be."""
import math

import pytest
import torch

import vocab_oracle as oracle

pytestmark = pytest.mark.gpu
INF = math.inf


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs a GPU"
    from nast_amd import ops as o
    return o


def ramp(V, chunk, plateau, step, dtype=torch.float32):
    """Nothing but `plateau` zeros in the first chunk, which hold most of the row's sum, and one element in each chunk behind it, each larger
    than the one before by `step`, a multiple of 2^-14 (exact in fp32 up to 128 * step)."""
    x = torch.full((V,), -INF)
    x[:plateau] = 0.0
    at = torch.arange(chunk, V, chunk)
    x[at + 5] = (at // chunk) * step
    return x.to(dtype)


@pytest.mark.parametrize("steps", [(69, 192), (199, 261), (320, 64), (255, 233)])
@pytest.mark.parametrize("V,chunk", [(1 << 20, 8192), (1 << 17, 8192), (1 << 17, 1 << 15)])
def test_ratio_on_rising_rows(ops, V, chunk, steps):
    """u next to p(d) / q(d), inside and outside of what fp32 can tell apart"""
    target = torch.stack((ramp(V, chunk, 8000, steps[0] * 2.0 ** -14), torch.zeros(V)))[None]
    draft = ramp(V, chunk, 4000, steps[1] * 2.0 ** -14)[None, None]
    E = torch.ones(1, V)
    tokens = torch.tensor([[17]])
    ratio = (torch.softmax(target[0, 0].double(), 0)[17] / torch.softmax(draft[0, 0].double(), 0)[17]).item()
    assert 0.2 < ratio < 0.9
    args = [t.cuda() for t in (target, tokens, E, draft)]
    seen = set()
    for off in (1e-7, 1e-6, 3e-6, 6e-6, 9e-6, 1.05e-5, 1.2e-5, 2e-5):
        for sign in (1, -1):
            u = torch.tensor([[ratio * (1 + sign * off)]])
            stands = u.double().item() < ratio
            out, accepted = ops.verify_draft(args[0], args[1], u.cuda(), args[2], args[3])
            assert accepted.item() == int(stands), (off, sign)
            seen.add(stands)
            want, _ = oracle.verify(target, tokens, u, E, draft, None, 1.0) if off in (1e-6, 2e-5) else (out.cpu(), None)
            assert torch.equal(out.cpu(), want)
    assert seen == {True, False}


def rows_for_sums(kind, R, V, dtype):
    g = torch.Generator(device="cuda").manual_seed(V + R)
    rise = torch.linspace(0.05, 24.0, R, device="cuda").unsqueeze(1)
    ids = torch.arange(V, device="cuda")
    if kind == "random":
        return (torch.randn(R, V, generator=g, device="cuda") * torch.linspace(0.1, 6.0, R, device="cuda").unsqueeze(1)).to(dtype)
    if kind == "rising":
        return (rise * ids / V).to(dtype)
    if kind == "falling":
        return (rise * (V - ids) / V).to(dtype)
    if kind == "one and the others":                              # a maximum with a tenth of the sum, the others alike
        x = torch.full((R, V), -math.log(V / 10.0), device="cuda") + rise * 0.01
        x[torch.arange(R), torch.randint(0, V, (R,), generator=g, device="cuda")] = rise.squeeze(1) * 0.01
        return x.to(dtype)
    # most of the sum in the first batch of a workgroup, one larger element in each batch behind it
    x = torch.full((R, V), -INF, device="cuda")
    batch = 1024 * (4 if dtype == torch.float32 else 8)
    x[:, :batch] = 0.0
    at = torch.arange(batch, V, batch, device="cuda")
    x[:, at + 8] = (at // batch) * (rise * 2.0 ** -8)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["random", "rising", "falling", "one and the others", "step a batch"])
@pytest.mark.parametrize("R,V", [(520, 9600), (520, 32768), (520, 32761), (4, 131072), (520, 131072), (512, 262144)])
def test_row_sums(ops, kind, R, V, dtype):
    """-log q(d) of a list of the one token d shows the sum: within 5e-6 where a chunk has no more than 2^15 elements, as the decisions
    of verify_draft take it, within 8e-6 for the longer chunks of distillation, plus the loss's own rounding, half a step"""
    x = rows_for_sums(kind, R, V, dtype)
    d = x.argmax(1, keepdim=True)
    loss = ops.top_distill(x, ops.TopLogits(torch.zeros(R, 1, device="cuda"), d, None, 1.0)).double()
    want = torch.cat([(torch.logsumexp(r.double(), 1) - r.double().amax(1)) for r in x.split(64)])
    bound = 5e-6 if V <= 1 << 15 or R < 16 else 8e-6
    assert ((loss - want).abs() <= bound + want.abs() * 2.0 ** -24).all(), ((loss - want).abs().max(), bound)
