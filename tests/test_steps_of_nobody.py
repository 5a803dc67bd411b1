"""A step of no sequence: nothing in, nothing out."""
import pytest
import torch

from eagersgd_b200.ops import scan
from test_scan import BF16, F32, _conv_case, _scan_case


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("own", [True, False])
def test_steps(own, device, dtype):
    c, _, state = _scan_case(0, 1, 24, 16, dtype, device)
    now = {k: v if k in ("A", "D", "delta_bias") else v[:, 0] for k, v in c.items()}
    y, new = scan.selective_scan_step(**now, state=state, out=state if own else None)
    assert y.shape == (0, 24) and y.dtype == dtype and new.shape == (0, 24, 16)
    x, w, bias, _ = _conv_case(0, 1, 24, 4, dtype, device)
    last = torch.zeros(0, 3, 24, dtype=dtype, device=device)
    y, new = scan.causal_conv_step(x[:, 0], last, w, bias, out=last if own else None)
    assert y.shape == (0, 24) and y.dtype == dtype and new.shape == (0, 3, 24)
