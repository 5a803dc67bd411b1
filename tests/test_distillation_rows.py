"""Rows without a teacher or a label: what their logits are is nobody's business, in the kernel and in the plain form."""
import pytest
import torch

from eagersgd_b200.ops import functional as ops
from test_distillation import _case

INF = float("inf")
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _both(logits, values, named, t, labels, w):
    leaf = logits.detach().requires_grad_()
    loss = ops.distillation_loss(leaf, values, named, t, labels, w)
    return loss.detach(), torch.autograd.grad(loss, leaf)[0]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("w", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("what", [float("nan"), INF, -INF])
def test_rows_that_have_no_term(what, w, dtype, device):
    logits, values, named, labels = _case(6, 40, 5, dtype, device=device)
    named[0], values[2], labels[0], labels[2] = -1, -INF, -1, 40               # rows 0 and 2: neither
    labels[1] = -1
    clean = _both(logits, values, named, 2.0, labels, w)
    logits[[0, 2]] = what
    if w == 1:
        logits[1] = what                                                       # a teacher who has no weight
    if w == 0:
        labels = None
    loss, grad = _both(logits, values, named, 2.0, labels, w)
    assert torch.equal(loss, clean[0]) and torch.equal(grad, clean[1])
    assert not grad[[0, 2]].any() and torch.isfinite(grad).all()


@pytest.mark.parametrize("device", DEVICES)
def test_a_row_with_one_of_the_two_terms(device):
    """The other term's row of NaN is NaN."""
    logits, values, named, labels = _case(3, 10, 4, torch.float32, device=device)
    logits[1] = float("nan")
    labels[1] = -1
    loss, grad = _both(logits, values, named, 2.0, labels, 0.5)
    assert torch.isnan(loss) and torch.isnan(grad[1]).all() and torch.isfinite(grad[[0, 2]]).all()
    named[1], labels[1] = -1, 3
    loss, grad = _both(logits, values, named, 2.0, labels, 0.5)
    assert torch.isnan(loss) and torch.isnan(grad[1]).all() and torch.isfinite(grad[[0, 2]]).all()
