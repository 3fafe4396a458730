"""CPU: a teacher's lists are checked against the layout they are said to have before rows of them are picked."""
import pytest
import torch

from nast_amd import _lib, ops

B, T, K = 2, 5, 3


def lists(values=(B, T, K), index=(B, T, K), lse=(B, T)):
    return ops.TopLogits(torch.zeros(values), torch.zeros(index, dtype=torch.int64), None if lse is None else torch.zeros(lse), 1.0)


@pytest.mark.parametrize("top,tail,match", [
    (lists(values=(B, T + 1, K)), False, "teacher's list"),
    (lists(index=(B, T + 1, K)), False, "teacher's list"),
    (lists((B, T + 1, K), (B, T + 1, K)), False, "teacher's list"),
    (lists((B, T - 1, K), (B, T - 1, K)), False, "teacher's list"),
    (lists((T, B, K), (T, B, K)), False, "teacher's list"),
    (lists((B * T, K), (B * T, K)), False, "teacher's list"),
    (lists(lse=(B, T + 1)), True, "log-sum-exp"),
    (lists(lse=(T, B)), True, "log-sum-exp"),
    (lists(lse=(B, T, 1)), True, "log-sum-exp"),
    (lists(lse=None), True, "log-sum-exp"),
    (lists()._replace(temperature=2.0), True, "temperature"),
    (lists(), False, "GPU only"),
])
def test_pick_top_refuses(top, tail, match):
    with pytest.raises(_lib.NastHipError, match=match):
        ops.pick_top(top, (B, T), torch.zeros(4, dtype=torch.int64), 1.0, tail)
