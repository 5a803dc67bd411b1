"""Temperatures that the arithmetic does not have are refused, and those at its ends are right."""
import pytest
import torch

from eagersgd_b200 import _build
from eagersgd_b200.ops import functional as ops
from test_distillation import _case, _formula

INF = float("inf")


@pytest.mark.parametrize("t,fits", [(1e-46, False), (1e-39, False), (1e-20, False), (1.2e-19, True), (1e18, True), (1.8e19, True), (2e19, False), (1e39, False),
                                    (1e300, False), (INF, False), (0.0, False), (-0.0, False), (float("nan"), False)])
def test_temperatures(t, fits):
    with pytest.raises(RuntimeError, match="not on a GPU" if fits else "temperature"):
        _build.load_torch().distillation_loss(torch.zeros(2, 10), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int64), t, None, 0.0)


@pytest.mark.parametrize("t,w", [(0.0, 0.5), (-1.0, 0.5), (INF, 0.5), (float("nan"), 0.5), (1.0, 1.5), (1.0, -0.5), (1.0, float("nan"))])
def test_the_plain_form_refuses_too(t, w):
    logits, values, named, labels = _case(3, 10, 4, torch.float32, device="cpu")
    with pytest.raises(ValueError, match="temperature"):
        ops.distillation_loss(logits, values, named, t, labels, w)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1.2e-19, 1e-10, 1e6, 1e18])
def test_far_temperatures(t):
    """Next to none: the largest logits alone count; next to infinite: all alike."""
    logits, values, named, _ = _case(4, 30, 5, torch.float32)
    leaf = logits.requires_grad_()
    loss = ops.distillation_loss(leaf, values, named, t)
    grad, = torch.autograd.grad(loss, leaf)
    wide = logits.detach().double().cpu().requires_grad_()
    want, _ = _formula(wide, values.double().cpu(), named.cpu(), t, None, 0.0)
    want_grad, = torch.autograd.grad(want, wide)
    # a row's terms are differences of logits, up to 20 / T, and of logarithms of 30 and 5, some 16 roundings of them each
    terms = 16 * 2.0 ** -24 * (20 / t + 4)
    assert abs(loss.item() - want.item()) < t * t * terms
    # T (q - p) a row: the exponentials' arguments are off by two roundings, they themselves by 2^-21
    assert ((grad.double().cpu() - want_grad).abs() <= t / 4 * (2.0 ** -19 + 2.0 ** -22 * 20 / t if t > 1 else 2.0 ** -19)).all()
