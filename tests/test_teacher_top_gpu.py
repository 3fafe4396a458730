"""GPU: StyleTransformer.forward(teacher_top=) refuses lists of another layout, whether rows are packed or not, and does not look at what
it does not need."""
import numpy as np
import pytest
import torch

from helpers import make_param, synth_batch

pytestmark = pytest.mark.gpu
V, L, B, K = 60, 10, 6, 7


@pytest.fixture(scope="module")
def setup():
    assert torch.cuda.is_available(), "needs a GPU"
    from nast_amd import ops, transformer as tf
    torch.manual_seed(3)
    F = tf.StyleTransformer(make_param(V=V, d=64, h=4, N=2, L=L, learnable=True)).cuda()
    sent, lens = (t.cuda() for t in synth_batch(np.random.default_rng(1), B, L, V))
    style = (torch.arange(B) % 2).cuda()
    top = ops.top_logits(torch.randn(B, L + 1, V, device="cuda") * 3, K, 1.0)     # one position more than the sentences have
    right = ops.TopLogits(*(t[:, :L] for t in top[:3]), 1.0)
    run = lambda t, tail: F(sent, lens, sent, lens, style, generate=False, temperature=1.0, use_inference_z=True, teacher_top=t, teacher_tail=tail)[0]
    return ops, right, top, run


@pytest.mark.parametrize("packed", [False, True])
def test_lists_of_another_layout(setup, packed):
    ops, right, long, run = setup
    with ops.packed_rows(packed):
        loss = run(right, True)
        for bad, tail in ((right._replace(values=long.values), False), (right._replace(index=long.index), False), (long, False),
                          (right._replace(lse=long.lse), True), (right._replace(lse=None), True),
                          (ops.TopLogits(*(t.transpose(0, 1) for t in right[:3]), 1.0), False),
                          (right._replace(values=right.values.cpu()), False), (right._replace(index=right.index.cpu()), False)):
            with pytest.raises(ops._lib.NastHipError):
                run(bad, tail)
        # without a tail the log-sum-exp is not needed, whatever it is
        list_alone = run(right, False)
        for other in (None, long.lse, right.lse.double(), right.lse.cpu()):
            assert torch.equal(run(right._replace(lse=other), False), list_alone)
        assert torch.equal(run(right, True), loss) and not torch.equal(loss, list_alone)


def test_pick_top(setup):
    ops, right, _, _ = setup
    at = torch.tensor([0, 5, 5, B * L - 1], device="cuda")
    got = ops.pick_top(right, (B, L), at, 1.0, True)
    for a, b in zip(got[:3], right[:3]):
        assert torch.equal(a, b.reshape(B * L, *b.shape[2:])[at])
    assert ops.pick_top(right, (B, L), at).lse is None and got.temperature == 1.0
