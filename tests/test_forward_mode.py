"""Group norm, scans and distillation make no forward-mode derivative: an operand with a tangent is refused, and not taken for a constant."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from eagersgd_b200 import _build
from eagersgd_b200.ops import functional as ops
from test_distillation import _case
from test_group_norm import _fits
from test_scan import CONV_FITS, CONV_STEP_FITS, SCAN_FITS, STEP_FITS

DISTILL_FITS = dict(logits=torch.zeros(2, 10), values=torch.zeros(2, 3), classes=torch.zeros(2, 3, dtype=torch.int64), t=1.0,
                    labels=torch.zeros(2, dtype=torch.int64), w=0.5)
CASES = [(op, fits, name) for op, fits in (("group_norm_act", _fits()), ("distillation_loss", DISTILL_FITS), ("causal_conv", CONV_FITS),
                                           ("causal_conv_step", CONV_STEP_FITS), ("selective_scan", SCAN_FITS), ("selective_scan_step", STEP_FITS))
         for name, v in fits.items() if isinstance(v, torch.Tensor) and v.is_floating_point()]


@pytest.mark.parametrize("grads", [True, False])
@pytest.mark.parametrize("op,fits,name", CASES)
def test_a_tangent_is_refused(op, fits, name, grads):
    f = getattr(_build.load_torch(), op)
    with fwd.dual_level(), torch.set_grad_enabled(grads):
        v = fits[name]
        a = dict(fits, **{name: fwd.make_dual(v, torch.ones_like(v))})
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(*a.values())
        with fwd._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="not on a GPU"):
            f(*a.values())
        with pytest.raises(RuntimeError, match="not on a GPU"):
            f(*fits.values())


def test_the_restatements_have_one():
    logits, values, named, labels = _case(3, 10, 4, torch.float64, device="cpu")
    d = torch.randn(3, 10, dtype=torch.float64)
    with fwd.dual_level():
        got = fwd.unpack_dual(ops.distillation_loss(fwd.make_dual(logits, d), values, named, 2.0, labels, 0.5)).tangent
    leaf = logits.requires_grad_()
    grad, = torch.autograd.grad(ops.distillation_loss(leaf, values, named, 2.0, labels, 0.5), leaf)
    assert abs(got - (grad * d).sum()) < 1e-12


@pytest.mark.gpu
def test_a_tangent_is_refused_on_the_gpu():
    x = torch.randn(2, 16, 4, 4, device="cuda")
    gamma, beta = torch.ones(16, device="cuda"), torch.zeros(16, device="cuda")
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.group_norm_act(fwd.make_dual(x, x), 4, gamma, beta)
    assert torch.isfinite(ops.group_norm_act(x, 4, gamma, beta)).all()
