"""An accumulator's memory lasts as long as its sink, whoever else holds the tensor."""
import pytest
import torch

from eagersgd_b200 import _build

pytestmark = pytest.mark.gpu


def test_an_accumulator_that_nobody_else_holds():
    params = [torch.nn.Parameter(torch.randn(1 << 18, device="cuda")) for _ in range(3)]
    sinks = _build.load_torch().GradSinks([len(params)], lambda bucket: None)
    before = torch.cuda.memory_allocated()
    for p in params:
        sinks.add(p, torch.zeros_like(p), 0)
    assert torch.cuda.memory_allocated() - before == len(params) << 20
    sinks.close()
    del sinks
    assert torch.cuda.memory_allocated() == before


def test_gradients_arrive_in_it():
    from eagersgd_b200.ops import functional as ops
    gamma, beta = (torch.nn.Parameter(torch.ones(32, device="cuda")) for _ in range(2))
    sinks = _build.load_torch().GradSinks([2], lambda bucket: None)
    for p in (gamma, beta):
        sinks.add(p, torch.zeros_like(p), 0)
    sinks.begin_step()
    sinks.set_active(True)
    x = torch.randn(4, 32, 6, 6, device="cuda").contiguous(memory_format=torch.channels_last).requires_grad_()
    others = [torch.zeros(32, device="cuda") for _ in range(64)]               # would be where a freed accumulator was
    ops.group_norm_act(x, 4, gamma, beta, "silu").sum().backward()
    sinks.set_active(False)
    sinks.close()
    assert gamma.grad is None and beta.grad is None and not any(o.any() for o in others)
