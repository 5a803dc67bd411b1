"""The loss of rows that are nearly sure: a logarithm of a sum just above one."""
import pytest
import torch

from eagersgd_b200.ops import functional as ops

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("hard", [True, False])
def test_the_loss_of_a_sure_row(hard):
    for d in torch.linspace(3, 15, 97).tolist():
        logits = torch.tensor([[0.0, -d]], device="cuda")
        values, named = torch.zeros(1, 1, device="cuda"), torch.zeros(1, 1, dtype=torch.int64, device="cuda")
        if hard:
            got = ops.distillation_loss(logits, values[:, :0], named[:, :0], 1.0, named[:, 0], 1.0)
        else:
            got = ops.distillation_loss(logits, values, named)
        want = torch.log1p(torch.exp(logits[0, 1].double()))
        # the sum, at most 1.05, is rounded once; its exponential is off by 2^-21 of 0.05 at most, the logarithm and the loss by a step
        assert abs(got.double() - want) < 1.05 * 2.0 ** -24 + (2.0 ** -21 + 2.0 ** -22) * 0.05, d
