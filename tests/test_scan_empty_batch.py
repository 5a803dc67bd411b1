"""A scan classifier without a sequence, as the LSTM classifier takes it."""
import pytest
import torch

from eagersgd_b200.models import LSTMClassifier, ScanClassifier
from eagersgd_b200.train.step import prepare_model


def _run(model, x):
    y = model(x)
    assert y.shape == (0, 5)
    y.sum().backward()
    for k, p in model.named_parameters():
        assert p.grad is not None and p.grad.shape == p.shape and not p.grad.any(), k
    if isinstance(model, ScanClassifier):
        lengths = torch.zeros(0, dtype=torch.int64, device=x.device)
        assert model(x, lengths).shape == (0, 5)
        logits, state = model.prompt(x, lengths)
        assert logits.shape == (0, 5) and model.step(x[:, 0].contiguous(), state).shape == (0, 5)
        assert model.hidden_states(x).shape == (6, 0, 16)


@pytest.mark.parametrize("kind", [LSTMClassifier, ScanClassifier])
def test_no_sequence(kind):
    _run(kind(8, 16, 2, 5), torch.randn(0, 6, 8))


@pytest.mark.gpu
def test_no_sequence_on_the_gpu():
    _run(prepare_model(ScanClassifier(8, 16, 2, 5), torch.device("cuda")), torch.randn(0, 6, 8, device="cuda").to(torch.bfloat16))


def test_no_step_has_no_last_one():
    with pytest.raises(IndexError):
        ScanClassifier(8, 16, 2, 5)(torch.randn(2, 0, 8))


def test_frames_of_more_dimensions_are_laid_flat():
    net = ScanClassifier(24, 16, 1, 5)
    x = torch.randn(2, 6, 2, 3, 4)
    assert torch.equal(net(x), net(x.reshape(2, 6, 24)))
