"""The plain forms refuse a derivative that they do not make, as the kernels do, and do not leave it out."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from eagersgd_b200 import _build
from eagersgd_b200.ops import functional as ops
from eagersgd_b200.ops import scan
from test_distillation import _case
from test_scan import CONV_STEP_FITS, STEP_FITS, _conv_case, _scan_case

F64 = torch.float64


def _calls():
    c, _, state = _scan_case(2, 5, 6, 4, F64, "cpu")
    state = state.double()
    x, w, bias, _ = _conv_case(2, 5, 6, 3, F64, "cpu")
    last = torch.randn(2, 2, 6, dtype=F64)
    now = {k: v if k in ("A", "D", "delta_bias") else v[:, 0] for k, v in c.items()}
    logits, values, named, _ = _case(3, 10, 4, F64, device="cpu")
    return {"causal_conv": (last, lambda s: scan.causal_conv(x, w, bias, state=s)),
            "causal_conv_step": (last, lambda s: scan.causal_conv_step(x[:, 0], s, w, bias)[0]),
            "causal_conv of no step": (last, lambda s: scan.causal_conv(x[:, :0], w, bias, state=s)),
            "selective_scan": (state, lambda s: scan.selective_scan(**c, state=s)),
            "selective_scan_step": (state, lambda s: scan.selective_scan_step(**now, state=s)[0]),
            "distillation_loss": (values, lambda v: ops.distillation_loss(logits, v, named))}


@pytest.mark.parametrize("name", list(_calls()))
def test_refused(name):
    t, f = _calls()[name]
    want = f(t)
    with pytest.raises(RuntimeError, match="detach it"):
        f(t.clone().requires_grad_())
    with torch.no_grad():
        assert torch.equal(f(t.clone().requires_grad_()), want)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="detach it"):
            f(fwd.make_dual(t, torch.ones_like(t)))
    assert torch.equal(f(t.clone().requires_grad_().detach()), want)


@pytest.mark.parametrize("op,fits", [("causal_conv_step", CONV_STEP_FITS), ("selective_scan_step", STEP_FITS)])
def test_room_for_a_state_that_wants_a_gradient(op, fits):
    f, room = getattr(_build.load_torch(), op), torch.zeros_like(fits["state"])
    with pytest.raises(RuntimeError, match="detach it"):
        f(*dict(fits, out=room.requires_grad_()).values())
    with torch.no_grad(), pytest.raises(RuntimeError, match="not on a GPU"):
        f(*dict(fits, out=room).values())
