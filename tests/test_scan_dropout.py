"""Dropout between a scan classifier's layers, as between the LSTM's."""
import pytest
import torch

from eagersgd_b200.models import ScanClassifier, create_model
from eagersgd_b200.models.video import ResNetLSTM


def _twins(dropout, layers=2):
    a, b = (ScanClassifier(8, 16, layers, 5, dropout=p) for p in (0.0, dropout))
    b.load_state_dict(a.state_dict())
    return a, b, torch.randn(3, 6, 8)


def test_in_training_alone():
    plain, net, x = _twins(0.5)
    want = plain(x)
    assert not torch.equal(net(x), net(x)) and not torch.equal(net(x), want)
    net.eval()
    assert torch.equal(net(x), want) and torch.equal(net.prompt(x)[0], want)
    logits, state = net.prompt(x[:, :3])
    for t in range(3, 6):
        logits = net.step(x[:, t], state)
    assert torch.allclose(logits, want, rtol=1e-4, atol=1e-5)


def test_between_layers_alone():
    plain, net, x = _twins(0.5, layers=1)
    assert torch.equal(net(x), plain(x)) and torch.equal(net(x), net(x))
    plain, net, x = _twins(0.5, layers=3)
    seen = []
    for layer in net.layers:
        layer.register_forward_pre_hook(lambda m, a: seen.append(a[0]))
    net(x)
    assert [bool((h == 0).any()) for h in seen] == [False, True, True]
    kept = (seen[1] != 0).float().mean()
    assert 0.25 < kept < 0.75                   # 288 values, of which half are kept


def test_the_rate_arrives():
    frames = torch.nn.Module()
    frames.features = lambda x: x.mean((2, 3)).repeat(1, 4)
    for sequence in ("scan", "lstm"):
        assert ResNetLSTM(num_classes=7, hidden=16, frame_net=frames, feature_dim=12, sequence=sequence, dropout=0.3).rnn.dropout == 0.3
        assert ResNetLSTM(num_classes=7, hidden=16, frame_net=frames, feature_dim=12, sequence=sequence).rnn.dropout == 0.5
    assert create_model("scan", classes=5, input_dim=8, hidden=16, dropout=0.2).dropout == 0.2


def test_a_network_saved_without_it_has_none():
    net = ScanClassifier(8, 16, 2, 5)
    del net.__dict__["dropout"]
    x = torch.randn(3, 6, 8)
    assert torch.equal(net(x), net(x))


@pytest.mark.gpu
def test_in_a_captured_training_step():
    """Every replay drops others: the losses of one batch at a rate of zero differ."""
    from eagersgd_b200.ops import functional as ops
    from eagersgd_b200.parallel.group import Group
    from eagersgd_b200.train.step import TrainStep
    torch.manual_seed(0)
    x, y = torch.randn(8, 17, 64, device="cuda").to(torch.bfloat16), torch.arange(8, device="cuda")
    for dropout in (0.0, 0.5):
        step = TrainStep(ScanClassifier(64, 96, 2, 40, width=160, dropout=dropout), Group(), mode="solo", limiter=4, lr=0.0, momentum=0.0,
                         weight_decay=0.0, loss_fn=ops.softmax_cross_entropy)
        step.capture(x, y)
        losses = [float(step.run_device(x, y)) for _ in range(4)]
        assert all(v == v for v in losses) and len(set(losses)) == (4 if dropout else 1)
        step.close()
