"""The distillation loss and its backward pass in graphs of their own, each replayed as often as its user likes."""
import pytest
import torch

from eagersgd_b200.ops import functional as ops
from test_distillation import _case

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_backward_pass_in_a_second_graph(dtype):
    logits, values, named, labels = _case(5, 77, 6, dtype)
    static, factor = logits.clone().requires_grad_(), torch.tensor(0.5, device="cuda")
    pool = torch.cuda.graph_pool_handle()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ahead, back = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(ahead, pool=pool, stream=stream):
            loss = ops.distillation_loss(static, values, named, 2.0, labels, 0.5)
        with torch.cuda.graph(back, pool=pool, stream=stream):
            grad, = torch.autograd.grad(loss, static, factor)
    torch.cuda.current_stream().wait_stream(stream)
    for seed in (0, 1):
        new = _case(5, 77, 6, dtype, seed=seed)[0].requires_grad_()
        with torch.no_grad():
            static.copy_(new)
        ahead.replay()
        for f in (0.5, 3.0, 0.25):
            factor.fill_(f)
            back.replay()
            want_loss = ops.distillation_loss(new, values, named, 2.0, labels, 0.5)
            want, = torch.autograd.grad(want_loss, new, torch.tensor(f, device="cuda"))
            assert torch.equal(loss, want_loss) and torch.equal(grad, want), (seed, f)
