"""The loss against a teacher's top logits: against the formula in 64 bits, and what it refuses."""
import pytest
import torch

from near import near
from eagersgd_b200 import _build
from eagersgd_b200.ops import functional as ops

BF16, F32 = torch.bfloat16, torch.float32
INF = float("inf")
gpu = pytest.mark.gpu


def _formula(logits, values, classes, t, labels, w):
    """Row by row in 64 bits: (loss, its rows)."""
    rows = []
    for r in range(logits.shape[0]):
        row = logits.new_zeros(())
        named = [(int(c), v) for c, v in zip(classes[r], values[r]) if 0 <= c < logits.shape[1] and v != -INF]
        if named and w < 1:
            p = torch.softmax(torch.stack([v for _, v in named]) / t, 0)
            log_q = torch.log_softmax(logits[r] / t, 0)
            for (c, _), pk in zip(named, p):
                if pk > 0:
                    row = row + (1 - w) * t * t * pk * (pk.log() - log_q[c])
        if w > 0 and 0 <= labels[r] < logits.shape[1]:
            row = row - w * torch.log_softmax(logits[r], 0)[labels[r]]
        rows.append(row)
    rows = torch.stack(rows)
    return rows.mean(), rows


def _case(rows, classes, top, dtype, seed=0, values_dtype=None, device="cuda"):
    g = torch.Generator().manual_seed(seed + rows * classes)
    logits = (torch.randn(rows, classes, generator=g) * 3).to(dtype).to(device)
    named = torch.stack([torch.randperm(classes, generator=g)[:top] for _ in range(rows)]).to(device)
    values = (torch.randn(rows, top, generator=g) * 3).to(values_dtype or dtype).to(device)
    return logits, values, named, torch.randint(0, classes, (rows,), generator=g).to(device)


def _check(logits, values, named, labels, t, w, factor=1.0):
    wide = logits.detach().double().cpu().requires_grad_()
    want, by_row = _formula(wide, values.double().cpu(), named.cpu(), t, labels.cpu() if labels is not None else None, w)
    want_grad, = torch.autograd.grad(want * factor, wide) if want.requires_grad else (torch.zeros_like(wide),)
    leaf = logits.detach().requires_grad_()
    loss = ops.distillation_loss(leaf, values, named, t, labels, w)
    got, = torch.autograd.grad(loss * factor, leaf)
    # a row's terms are differences of logits (up to m / T, times T^2) and logarithms of sums, a dozen roundings each and those of
    # the sums of exponentials, whose own error is that of their argument
    m = wide.detach()[torch.isfinite(wide.detach())].abs().max().item() + values[torch.isfinite(values)].abs().max().item() if values.numel() else 20.0
    steps = 64 + 8 * m / min(t, 1.0)
    near(loss, want.detach(), (1 + t * t) * (2 * m / t + 12), steps, "loss")
    # the gradient: fractions of the rows' weight
    near(got, want_grad, want_grad.abs() + factor * (1 + t) / logits.shape[0] * 1e-2, steps, "gradient", roundings=1 if factor == 1.0 else 2)
    with torch.no_grad():
        assert torch.equal(ops.distillation_loss(logits, values, named, t, labels, w), loss.detach())


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,w", [(1.0, 0.0), (2.0, 0.3), (0.5, 1.0), (4.0, 0.5)])
@pytest.mark.parametrize("rows,classes,top", [(1, 1, 1), (3, 2, 2), (5, 10, 3), (4, 101, 50), (2, 1000, 64), (3, 1027, 129), (2, 4097, 33), (2, 32003, 64)])
def test_sizes(rows, classes, top, t, w, dtype):
    logits, values, named, labels = _case(rows, classes, top, dtype)
    _check(logits, values, named, labels if w > 0 else None, t, w)


@gpu
@pytest.mark.parametrize("factor", [0.5, 3.0])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_factor_on_the_loss(dtype, factor):
    logits, values, named, labels = _case(7, 333, 20, dtype)
    _check(logits, values, named, labels, 2.0, 0.25, factor)


@gpu
def test_a_teacher_of_another_type():
    for a, b in ((BF16, F32), (F32, BF16)):
        logits, values, named, _ = _case(4, 55, 7, a, values_dtype=b)
        _check(logits, values, named, None, 1.5, 0.0)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_without_a_teacher_or_label(dtype):
    logits, values, named, labels = _case(6, 40, 5, dtype)
    named[0] = -1                                   # nobody
    named[1, 2:] = 40                               # two only
    values[2] = -INF                                # nobody, said in the other way
    labels[0], labels[3] = -1, 40
    _check(logits, values, named, labels, 2.0, 0.5)
    _check(logits, values, named, None, 2.0, 0.0)
    logits[0] = float("nan")                        # what such a row holds does not matter
    loss = ops.distillation_loss(logits.requires_grad_(), values, named, 2.0, labels, 0.5)
    grad, = torch.autograd.grad(loss, logits)
    assert torch.isfinite(loss) and torch.isfinite(grad).all() and not grad[0].any()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_masked_classes(dtype):
    """Classes masked with -inf or with the type's lowest value get no probability, whole vectors of them neither."""
    logits, values, named, labels = _case(4, 200, 8, dtype)
    logits[0, 16:160] = -INF
    logits[1, :150] = torch.finfo(dtype).min
    logits[2, 1:] = -INF
    named[0] = torch.arange(8)
    named[1] = torch.arange(160, 168)
    named[2], labels[2], named[2, 1:] = 0, 0, -1
    labels[0], labels[1] = 3, 170
    _check(logits, values, named, labels, 2.0, 0.3)


@gpu
def test_classes_named_more_than_once_count_as_often():
    logits, values, named, labels = _case(3, 30, 9, F32)
    named[0, 3:6] = named[0, 0]
    named[1] = 7
    labels[1] = 7
    _check(logits, values, named, labels, 1.0, 0.4)


@gpu
def test_a_teacher_of_nothing():
    logits, _, _, labels = _case(3, 30, 2, F32)
    values, named = torch.empty(3, 0, device="cuda"), torch.empty(3, 0, dtype=torch.int64, device="cuda")
    _check(logits, values, named, labels, 1.0, 0.4)
    assert ops.distillation_loss(logits, values, named).item() == 0


@gpu
def test_padded_sliced_and_odd_rows():
    """Rows as the dense layer pads them, a slice of wider ones, and rows that begin anywhere."""
    logits, values, named, labels = _case(5, 101, 9, F32)
    want = ops.distillation_loss(logits, values, named, 2.0, labels, 0.5)
    padded = torch.full((5, 104), float("nan"), device="cuda")[:, :101].copy_(logits)
    wide = torch.full((5, 300), float("nan"), device="cuda")[:, 100:201].copy_(logits)
    odd = torch.empty(5 * 101 + 1, device="cuda")[1:].view(5, 101).copy_(logits)
    for v in (padded, wide, odd, logits.t().contiguous().t()):
        leaf = v.detach().requires_grad_()
        loss = ops.distillation_loss(leaf, values, named, 2.0, labels, 0.5)
        assert torch.equal(loss, want)
        grad, = torch.autograd.grad(loss, leaf)
        assert torch.isfinite(grad).all()
        _check(v, values, named, labels, 2.0, 0.5)


@gpu
def test_behind_the_dense_layer():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(16, 64, generator=g).to(BF16).cuda().requires_grad_()
    w = torch.randn(101, 64, generator=g).to(BF16).cuda().requires_grad_()
    _, values, named, labels = _case(16, 101, 9, F32)
    logits = ops.linear(x, w)
    assert logits.stride(0) == 104
    dx, = torch.autograd.grad(ops.distillation_loss(logits, values, named, 2.0, labels, 0.5), x)
    wide = x.detach().double().cpu().requires_grad_()
    loss, _ = _formula(wide @ w.detach().double().cpu().t(), values.double().cpu(), named.cpu(), 2.0, labels.cpu(), 0.5)
    want, = torch.autograd.grad(loss, wide)
    # the dense layer rounds its gradient to bf16 first: 101 products off by half a step each, and the result
    assert (dx.double().cpu() - want).abs().max() < 2.0 ** -8 * (want.abs().max() + w.double().abs().max().item() * 3 / 16 * 2)


@gpu
def test_a_kept_graph_and_a_second_backward():
    logits, values, named, _ = _case(4, 50, 5, F32)
    leaf = logits.requires_grad_()
    loss = ops.distillation_loss(leaf, values, named)
    one, = torch.autograd.grad(loss, leaf, retain_graph=True)
    three, = torch.autograd.grad(loss, leaf, torch.tensor(3.0, device="cuda"), retain_graph=True)
    last, = torch.autograd.grad(loss, leaf, torch.tensor(2.0, device="cuda"))
    assert torch.equal(three, one * 3) and torch.equal(last, one * 2)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, leaf)


@gpu
def test_captured_with_its_backward_pass():
    logits, values, named, labels = _case(4, 50, 5, F32)
    static = logits.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = ops.distillation_loss(static, values, named, 2.0, labels, 0.5)
        grad, = torch.autograd.grad(loss * 2, static)
    for seed in (1, 2):
        new = _case(4, 50, 5, F32, seed=seed)[0]
        with torch.no_grad():
            static.copy_(new)
        graph.replay()
        leaf = new.requires_grad_()
        want_loss = ops.distillation_loss(leaf, values, named, 2.0, labels, 0.5)
        want, = torch.autograd.grad(want_loss * 2, leaf)
        assert torch.equal(loss, want_loss) and torch.equal(grad, want)


@gpu
def test_a_teacher_of_nan():
    """No row without a teacher: the loss and the row's gradient are NaN, on the GPU as in the formula, and the other rows' are not."""
    for top in (1, 5):
        logits, values, named, _ = _case(3, 40, top, F32)
        values[1] = float("nan")
        for leaf, v, n in ((logits, values, named), (logits.cpu(), values.cpu(), named.cpu())):
            leaf = leaf.detach().requires_grad_()
            loss = ops.distillation_loss(leaf, v, n)
            grad, = torch.autograd.grad(loss, leaf)
            assert torch.isnan(loss) and torch.isnan(grad[1, n[1]]).all() and torch.isfinite(grad[[0, 2]]).all()


@gpu
def test_a_captured_backward_pass_alone():
    """A forward pass made once, its backward pass captured: every replay gives the same gradient."""
    logits, values, named, _ = _case(5, 77, 6, BF16)
    factor = torch.tensor(0.5, device="cuda")
    leaf = logits.requires_grad_()
    want, = torch.autograd.grad(ops.distillation_loss(leaf, values, named), leaf, factor)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        loss = ops.distillation_loss(leaf, values, named)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got, = torch.autograd.grad(loss, leaf, factor)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@gpu
def test_logits_past_32_bits():
    """More than 2^31 of them: the last rows' loss and gradient are those of the rows alone."""
    rows, classes = 70003, 32008
    logits = torch.empty(rows, classes, dtype=BF16, device="cuda")
    logits[:-2] = 0
    small, values, named, _ = _case(2, classes, 5, BF16)
    logits[-2:] = small
    all_values, all_named = torch.zeros(rows, 5, device="cuda"), torch.full((rows, 5), -1, dtype=torch.int64, device="cuda")
    all_values[-2:], all_named[-2:] = values.float(), named
    leaf = logits.requires_grad_()
    loss = ops.distillation_loss(leaf, all_values, all_named)
    grad, = torch.autograd.grad(loss, leaf, torch.tensor(float(rows), device="cuda"))
    ref = small.requires_grad_()
    want = ops.distillation_loss(ref, values.float(), named)
    want_grad, = torch.autograd.grad(want, ref, torch.tensor(2.0, device="cuda"))
    assert abs(loss.item() * rows - want.item() * 2) < 1e-4 * want.item()
    # both are rounded to bf16, times their row's weight, and again, times the factor; a named class is a difference of fp32 fractions
    assert ((grad[-2:].float() - want_grad.float()).abs() <= 4.1 * 2.0 ** -8 * want_grad.float().abs() + 1e-6).all() and not grad[:-2].any()


@gpu
def test_gradient_against_differences():
    logits, values, named, labels = _case(2, 20, 4, F32)
    leaf = logits.detach().requires_grad_()
    grad, = torch.autograd.grad(ops.distillation_loss(leaf, values, named, 2.0, labels, 0.5), leaf)
    d, e = torch.randn(2, 20, generator=torch.Generator().manual_seed(1)).cuda(), 2.0 ** -6
    ends = [ops.distillation_loss(logits + s * e * d, values, named, 2.0, labels, 0.5).double().item() for s in (1, -1)]
    # e^2 times a third derivative of order one, and roundings of a loss of some 10 over 2 e
    assert abs((ends[0] - ends[1]) / (2 * e) - (grad * d).double().sum().item()) < 5e-3


# ------------------------------------------------------------------------------------------------ without a GPU
@pytest.mark.parametrize("dtype", [F32, torch.float64])
def test_the_restatement_is_the_formula(dtype):
    logits, values, named, labels = _case(6, 40, 5, dtype, device="cpu")
    named[0], named[1, 2:], values[2], labels[3], named[4, 1] = -1, 40, -INF, 40, int(named[4, 0])
    leaf = logits.requires_grad_()
    loss = ops.distillation_loss(leaf, values, named, 2.0, labels, 0.5)
    grad, = torch.autograd.grad(loss, leaf)
    wide = logits.detach().double().requires_grad_()
    want, _ = _formula(wide, values.double(), named, 2.0, labels, 0.5)
    want_grad, = torch.autograd.grad(want, wide)
    assert abs(loss.item() - want.item()) < 1e-5 and (grad.double() - want_grad).abs().max() < 1e-6


@pytest.mark.parametrize("change,message", [
    (dict(logits=torch.zeros(2, 3, 4)), "2-D"), (dict(logits=torch.zeros(2, 10, dtype=torch.float16)), "neither"),
    (dict(values=torch.zeros(2, 3, dtype=torch.float16)), "neither"), (dict(values=torch.zeros(3, 3)), "teacher"),
    (dict(classes=torch.zeros(2, 3, dtype=torch.int32)), "teacher_classes"), (dict(classes=torch.zeros(2, 4, dtype=torch.int64)), "teacher"),
    (dict(values=torch.zeros(2, 1025), classes=torch.zeros(2, 1025, dtype=torch.int64)), "1024"),
    (dict(t=0.0), "temperature"), (dict(t=-1.0), "temperature"), (dict(t=float("nan")), "temperature"), (dict(w=1.5), "hard weight"),
    (dict(w=-0.1), "hard weight"), (dict(w=0.5, labels=None), "without labels"), (dict(labels=torch.zeros(3, dtype=torch.int64)), "labels"),
    (dict(labels=torch.zeros(2)), "labels"), (dict(logits=torch.zeros(0, 10)), "no mean"), (dict(values=torch.zeros(2, 3, requires_grad=True)), "detach"),
    (dict(), "not on a GPU"),
])
def test_refusals(change, message):
    a = dict(logits=torch.zeros(2, 10), values=torch.zeros(2, 3), classes=torch.zeros(2, 3, dtype=torch.int64), t=1.0,
             labels=torch.zeros(2, dtype=torch.int64), w=0.5)
    a.update(change)
    with pytest.raises(RuntimeError, match=message):
        _build.load_torch().distillation_loss(*a.values())
