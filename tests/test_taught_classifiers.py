"""Group norm, causal convolution, selective scan and distillation as models use them together."""
import copy

import pytest
import torch

from eagersgd_b200.models import ScanClassifier, create_model
from eagersgd_b200.models.resnet import BatchNormAct, GroupNormAct, cifar_resnet, imagenet_resnet
from eagersgd_b200.models.video import ResNetLSTM
from eagersgd_b200.ops import functional as ops
from eagersgd_b200.train.step import TrainStep, prepare_model

gpu = pytest.mark.gpu


def _teacher(rows, classes, top, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    named = torch.stack([torch.randperm(classes, generator=g)[:top] for _ in range(rows)])
    return (3 * torch.randn(rows, top, generator=g)).to(device), named.to(device), named[:, 0].contiguous().to(device)


def _taught(values, named):
    return lambda logits, y: ops.distillation_loss(logits, values, named, temperature=2.0, labels=y, hard_weight=0.5)


# ------------------------------------------------------------------------------------------------ without a GPU
def test_a_stream_of_steps_gives_what_the_sequence_gives():
    torch.manual_seed(0)
    m = ScanClassifier(24, 32, 2, 10)
    x, lengths = torch.randn(4, 9, 24), torch.tensor([9, 3, 5, 1])
    whole = m(x, lengths)
    for i, n in enumerate(lengths):
        logits, state = m.prompt(x[i:i + 1, :n])
        assert torch.allclose(logits, whole[i:i + 1], rtol=1e-4, atol=1e-5)
    logits, state = m.prompt(x[:, :4])
    for t in range(4, 9):
        logits = m.step(x[:, t], state)
    assert torch.allclose(logits, m(x), rtol=1e-4, atol=1e-5)


def test_every_parameter_of_a_scan_classifier_learns():
    m = create_model("scan", classes=5, input_dim=8, hidden=16, layers=2)
    values, named, labels = _teacher(3, 5, 2, "cpu")
    _taught(values, named)(m(torch.randn(3, 6, 8)), labels).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any() for p in m.parameters())


def test_networks_with_group_norm():
    for version in (1, 2):
        net = cifar_resnet(8, version, 10, norm="group")
        kinds = {type(m) for m in net.modules()}
        assert GroupNormAct in kinds and BatchNormAct not in kinds and not list(net.buffers())
        x = torch.randn(3, 3, 32, 32)
        one = torch.cat([net(x[i:i + 1]) for i in range(3)])
        assert torch.allclose(net(x), one, rtol=1e-4, atol=1e-5)             # nothing of the batch
        net.eval()
        assert torch.allclose(net(x), one, rtol=1e-4, atol=1e-5)
    norms = [m for m in imagenet_resnet(18, 1, 10, norm="group").modules() if isinstance(m, GroupNormAct)]
    assert {(m.num_groups, m.num_channels) for m in norms} == {(8, 64), (16, 128), (32, 256), (32, 512)}
    with pytest.raises(ValueError, match="layer"):
        cifar_resnet(8, 1, 10, norm="layer")


def test_batch_norm_networks_are_what_they_were():
    torch.manual_seed(1)
    a = cifar_resnet(8, 1, 10)
    torch.manual_seed(1)
    b = cifar_resnet(8, 1, 10, norm="batch")
    assert list(a.state_dict()) == list(b.state_dict())
    assert all(torch.equal(u, v) for u, v in zip(a.state_dict().values(), b.state_dict().values()))


def test_decay_checkpoints_and_flags_know_group_norm():
    from eagersgd_b200.ckpt.tf_layout import tf_variables
    from eagersgd_b200.train import flags
    from eagersgd_b200.train.resnet_main import DATASETS, build_model
    net = cifar_resnet(8, 1, 10, norm="group")
    decayed, plain = TrainStep._param_groups(net, 1e-4, False)
    assert {id(p) for p in plain["params"]} == {id(p) for m in net.modules() if isinstance(m, GroupNormAct) for p in m.parameters()}
    with pytest.raises(NotImplementedError, match="group norm"):
        tf_variables(net)
    args = flags.resolve(flags.build_parser("x").parse_args(["--norm", "group", "-rs", "8"]))
    args.dataset = "cifar10"
    assert build_model(args, DATASETS["cifar10"]).norm == "group"


@pytest.mark.parametrize("flag", ["--export_dir", "--pretrained_model_checkpoint_path", "--virtual_batch_size"])
def test_what_is_about_batch_norm_is_refused_before_training(flag, capsys):
    from eagersgd_b200.train import resnet_main
    with pytest.raises(SystemExit):
        resnet_main.main(["--norm", "group", "--dataset", "cifar10", flag, "4"])
    assert "not with --norm group" in capsys.readouterr().err


def test_lengths_beyond_the_sequence_end_with_it():
    net = ScanClassifier(8, 16, 1, 5)
    x = torch.randn(3, 6, 8)
    want = net(x, torch.tensor([6, 6, 1]))
    assert torch.equal(net(x, torch.tensor([9, 1 << 40, -2]))[:2], want[:2])
    assert torch.isfinite(net(x, torch.tensor([9, 6, -2]))).all()


def test_a_users_own_group_norm_decays_as_it_did():
    from eagersgd_b200.train.step import TrainStep
    own = torch.nn.Sequential(torch.nn.Conv2d(3, 8, 1), torch.nn.GroupNorm(2, 8), torch.nn.BatchNorm2d(8))
    decayed, plain = TrainStep._param_groups(own, 1e-4, False)
    assert {id(p) for p in plain["params"]} == {id(p) for p in own[2].parameters()}
    assert any(p is own[1].weight for p in decayed["params"])


def test_clips_through_a_scan():
    frames = torch.nn.Module()
    frames.features = lambda x: x.mean((2, 3)).repeat(1, 4)
    net = ResNetLSTM(num_classes=7, hidden=16, layers=1, frame_net=frames, feature_dim=12, sequence="scan")
    assert net(torch.randn(2, 5, 3, 8, 8)).shape == (2, 7)
    with pytest.raises(ValueError, match="sequence"):
        ResNetLSTM(frame_net=frames, feature_dim=12, sequence="gru")


# ------------------------------------------------------------------------------------------------ on a GPU
def _gradients(model, x, lengths, loss, labels):
    model.zero_grad(set_to_none=True)
    out = loss(model(x, lengths) if lengths is not None else model(x), labels)
    out.backward()
    return out.detach().float(), {k: p.grad.float().clone() for k, p in model.named_parameters()}


@gpu
@pytest.mark.parametrize("ragged", [False, True])
def test_a_taught_scan_classifier_against_the_restatements(ragged):
    torch.manual_seed(0)
    m = prepare_model(ScanClassifier(64, 96, 2, 40, width=160), torch.device("cuda"))
    x = torch.randn(5, 33, 64, device="cuda").to(torch.bfloat16)
    lengths = torch.tensor([33, 1, 8, 20, 32], device="cuda") if ragged else None
    values, named, labels = _teacher(5, 40, 6, "cuda")
    loss, grads = _gradients(m, x, lengths, _taught(values, named), labels)
    with ops.reference_ops():
        want, wants = _gradients(m, x, lengths, _taught(values, named), labels)
    # each of some fifteen operators a layer rounds to bf16, forward and backward: 60 roundings of half a step (2^-8), which add up as
    # their root mean square (a quarter of a step each)
    bound = 60 ** 0.5 * 2.0 ** -9 * 4
    assert abs(loss - want) < bound * want.abs()
    for k in grads:
        assert (grads[k] - wants[k]).norm() < bound * wants[k].norm(), k


@gpu
def test_steps_of_a_stream_on_the_gpu():
    torch.manual_seed(0)
    m = prepare_model(ScanClassifier(64, 96, 2, 40, width=160), torch.device("cuda"))
    x = torch.randn(6, 20, 64, device="cuda").to(torch.bfloat16)
    logits, state = m.prompt(x[:, :12])
    for t in range(12, 20):
        logits = m.step(x[:, t], state)
    with torch.no_grad():
        want = m(x)
    assert (logits.float() - want.float()).norm() < 30 ** 0.5 * 2.0 ** -9 * 4 * want.float().norm()


@gpu
@pytest.mark.parametrize("kind", ["scan", "resnet"])
def test_a_taught_step_updates_by_its_gradient(kind):
    """The training step's accumulators get the gradients that autograd gives."""
    from eagersgd_b200.parallel.group import Group
    torch.manual_seed(0)
    if kind == "scan":
        model, x = ScanClassifier(64, 96, 1, 40, width=160), torch.randn(8, 17, 64, device="cuda").to(torch.bfloat16)
    else:
        model = cifar_resnet(8, 1, 40, norm="group")
        x = torch.randn(8, 3, 32, 32, device="cuda").to(torch.bfloat16).contiguous(memory_format=torch.channels_last)
        for m in model.modules():
            if isinstance(m, GroupNormAct):
                torch.nn.init.ones_(m.weight)
    values, named, labels = _teacher(8, 40, 6, "cuda")
    twin = prepare_model(copy.deepcopy(model), torch.device("cuda"))
    want_loss, wants = _gradients(twin, x, None, _taught(values, named), labels)
    step = TrainStep(model, Group(), mode="solo", limiter=4, lr=1.0, momentum=0.0, weight_decay=0.0, loss_fn=_taught(values, named))
    before = {k: p.detach().clone() for k, p in step.model.named_parameters()}
    loss = step.run_device(x, labels)
    torch.cuda.synchronize()
    assert torch.equal(loss.float(), want_loss)
    compared = 0
    for k, p in step.model.named_parameters():
        if p.dtype != torch.float32:
            continue
        moved = (before[k] - p.detach()).reshape(-1)
        # one product of bf16 gradients may come in another order, and a bucket's slots are rounded to bf16 before the update
        assert (moved - wants[k].reshape(-1)).norm() < 2.0 ** -6 * wants[k].norm() + 1e-6 * before[k].norm(), k
        compared += 1
    assert compared >= 5
    step.close()


@gpu
@pytest.mark.parametrize("kind", ["scan", "resnet"])
def test_a_taught_step_in_a_graph(kind):
    from eagersgd_b200.parallel.group import Group
    torch.manual_seed(0)
    if kind == "scan":
        model, x = ScanClassifier(64, 96, 2, 40, width=160), torch.randn(8, 17, 64, device="cuda").to(torch.bfloat16)
    else:
        model = cifar_resnet(8, 1, 40, norm="group")
        x = torch.randn(8, 3, 32, 32, device="cuda").to(torch.bfloat16).contiguous(memory_format=torch.channels_last)
    values, named, labels = _teacher(8, 40, 6, "cuda")
    step = TrainStep(model, Group(), mode="solo", limiter=4, lr=0.02, loss_fn=_taught(values, named))
    step.capture(x, labels)
    losses = [float(step.run_device(x, labels)) for _ in range(4)]
    assert all(v == v and v < 1e4 for v in losses) and step.stats()["status"] == 0
    assert len(set(losses)) > 1                                               # replays go on learning
    step.close()
