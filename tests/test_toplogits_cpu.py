"""CPU: what ops.top_logits / top_distill / verify_draft and their C entries refuse, before anything is launched; the 64-bit statements
the GPU tests compare with, against known answers."""
import ctypes as C
import math

import pytest
import torch

import vocab_oracle as oracle
from nast_amd import _lib, ops


def refused(name, *args, match=None):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == -1
    assert match in lib.nast_last_error().decode()


P = 256                      # an aligned address that is never read: every call here ends at a check
R = _lib.Rows(8, 0, 0)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 8)
    top = ops.TopLogits(torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2), 1.0)
    with pytest.raises(_lib.NastHipError, match="GPU only"):
        ops.top_logits(x, 3)
    with pytest.raises(_lib.NastHipError, match="GPU only"):
        ops.top_distill(x, top)
    with pytest.raises(_lib.NastHipError, match="fp32|GPU only"):
        ops.generator_distill(torch.zeros(2, 4), torch.zeros(8, 4), torch.zeros(8), 1.0, top)
    with pytest.raises(_lib.NastHipError, match="GPU only"):
        ops.verify_draft(torch.zeros(2, 2, 8), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1), torch.ones(2, 8))


@pytest.mark.parametrize("t", [0.0, -1.0, 1e-40, math.inf, math.nan])
def test_temperature_is_refused(t):
    with pytest.raises(_lib.NastHipError, match="temperature"):
        ops.top_distill(torch.zeros(2, 8), None, t)
    refused("nast_top_logits", P, 0, R, P, P, P, 1, 8, 1, t, P, None, match="temperature")
    refused("nast_top_distill_fwd", P, 0, R, P, 0, P, 1, None, P, P, 1, 8, t, P, None, match="temperature")
    refused("nast_top_distill_bwd", P, P, 0, R, P, 0, P, 1, P, 2 * P, R, 1, 8, t, None, match="temperature")
    refused("nast_verify_draft", P, 0, 8, None, 0, 0, 0, P, P, P, None, P, P, 1, 1, 8, t, P, None, match="temperature")


@pytest.mark.parametrize("top,tail,match", [
    (lambda v, i, s: (v[:, 0], i, s, 1.0), False, "teacher's list"),
    (lambda v, i, s: (v, i[:1], s, 1.0), False, "teacher's list"),
    (lambda v, i, s: (v[:1], i[:1], s, 1.0), False, "teacher's list"),
    (lambda v, i, s: (v, i.int(), s, 1.0), False, "int64"),
    (lambda v, i, s: (v.double(), i, s, 1.0), False, "fp32, bf16 or fp16"),
    (lambda v, i, s: (v[:, :0], i[:, :0], s, 1.0), False, "1 to 256"),
    (lambda v, i, s: (v.expand(3, 2, 3).reshape(2, 9).repeat(1, 30), i.repeat(1, 90), s, 1.0), False, "1 to 256"),
    (lambda v, i, s: (v, i, None, 1.0), True, "log-sum-exp"),
    (lambda v, i, s: (v, i, s.double(), 1.0), True, "log-sum-exp"),
    (lambda v, i, s: (v, i, s[:1], 1.0), True, "log-sum-exp"),
    (lambda v, i, s: (v, i, s, 2.0), True, "temperature"),
])
def test_teacher_lists_are_refused(top, tail, match):
    v, i, s = torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2)
    with pytest.raises(_lib.NastHipError, match=match):
        ops.top_distill(torch.zeros(2, 8), ops.TopLogits(*top(v, i, s)), 1.0, tail)


def test_c_entries_refuse():
    big = 1 << 24
    top = lambda x=P, dtype=0, v=P, i=P, s=P, rows=2, V=8, k=3: ("nast_top_logits", x, dtype, R, v, i, s, rows, V, k, 1.0, P, None)
    refused(*top(dtype=3), match="dtype")
    refused(*top(V=0), match="bad sizes")
    refused(*top(V=big), match="bad sizes")
    refused(*top(rows=-1), match="bad sizes")
    refused(*top(rows=big), match="too many rows")
    for k in (0, 9, 257):
        refused(*top(k=k), match="k=")
    refused(*top(x=None), match="NULL")
    refused(*top(s=None), match="NULL")
    refused(*top(x=P + 2), match="misaligned")
    fwd = lambda x=P, dtype=0, td=0, K=3, loss=P, rows=2, V=8, ws=P: ("nast_top_distill_fwd", x, dtype, R, P, td, P, K, None, loss, P, rows, V, 1.0,
                                                                  ws, None)
    refused(*fwd(dtype=-1), match="dtype")
    refused(*fwd(td=7), match="dtype")
    refused(*fwd(K=0), match="slots")
    refused(*fwd(K=257), match="slots")
    refused(*fwd(V=big), match="bad sizes")
    refused(*fwd(loss=None), match="NULL")
    refused(*fwd(x=P + 1, dtype=1), match="misaligned")
    refused(*fwd(rows=1, V=200000, ws=None), match="workspace")
    refused(*fwd(rows=big - 1, V=600000), match="too many rows")
    bwd = lambda g=P, x=P, gx=2 * P, rows=2, V=8: ("nast_top_distill_bwd", g, x, 0, R, P, 0, P, 3, P, gx, R, rows, V, 1.0, None)
    refused(*bwd(gx=P), match="in-place")
    refused(*bwd(g=None), match="NULL")
    refused(*bwd(rows=big - 1, V=200000), match="too many rows")
    refused(*bwd(gx=2 * P + 1), match="misaligned")
    ver = lambda t=P, q=None, dtype=0, tok=P, E=P, B=2, N=3, V=8, ws=P: ("nast_verify_draft", t, 32, 8, q, 24, 8, dtype, tok, P, E, None, P, P, B, N, V, 1.0,
                                                                         ws, None)
    refused(*ver(dtype=3), match="dtype")
    refused(*ver(N=-1), match="bad sizes")
    refused(*ver(N=1025), match="bad sizes")
    refused(*ver(V=0), match="bad sizes")
    refused(*ver(t=None), match="NULL")
    refused(*ver(tok=None), match="NULL")
    refused(*ver(ws=None), match="NULL")
    refused(*ver(q=P + 2), match="misaligned")
    refused(*ver(B=1 << 20, N=15), match="bad sizes")
    refused(*ver(V=(1 << 20) + 1), match="bad sizes")
    for name, args in (("nast_top_logits_workspace_bytes", (2, 8, 3, 0)), ("nast_top_distill_workspace_bytes", (2, 8, 0)),
                       ("nast_verify_draft_workspace_bytes", (2, 3, 8, 0))):
        assert getattr(_lib.load(), name)(*args) >= 0


def test_oracle_known_answers():
    x = torch.tensor([[0.0, math.log(3.0), -math.inf, 0.0]])
    index, lse = oracle.top(x, 3, 1.0)
    assert index.tolist() == [[1, 0, 3]] and abs(lse.item() - math.log(5.0)) < 1e-6
    # teacher 1/2, 1/2 on ids 0 and 3, student 1/5, 1/5: KL = log(1/2) - log(1/5); dz = q - p
    loss, grad, _ = oracle.distill(x, torch.zeros(1, 3), torch.tensor([[0, 3, -1]]), None, 1.0, False, torch.ones(1))
    assert abs(loss.item() - math.log(2.5)) < 1e-6
    assert torch.allclose(grad, torch.tensor([[0.2 - 0.5, 0.6, 0.0, 0.2 - 0.5]]).double(), atol=1e-6)
    # with the teacher's own normaliser 4: 1/4, 1/4 and 1/2 for the rest, where the student has 3/5
    loss, grad, _ = oracle.distill(x, torch.zeros(1, 2), torch.tensor([[0, 3]]), torch.tensor([math.log(4.0)]), 1.0, True, torch.ones(1))
    assert abs(loss.item() - (0.5 * math.log(1.25) + 0.5 * math.log(0.5 / 0.6))) < 1e-6
    assert torch.allclose(grad, torch.tensor([[-0.05, 0.1, 0.0, -0.05]]).double(), atol=1e-6)
    target = torch.tensor([0.5, 0.3, 0.2]).log().expand(1, 2, 3)
    draft = torch.tensor([[[0.25, 0.5, 0.25]]]).log()
    args = lambda u: (target, torch.tensor([[1]]), torch.tensor([[u]]), torch.ones(1, 3), draft, None, 1.0)
    assert [t.tolist() for t in oracle.verify(*args(0.59))] == [[[1, 0]], [1]]
    assert [t.tolist() for t in oracle.verify(*args(0.61))] == [[[0, -1]], [0]]
