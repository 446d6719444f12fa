"""Encoder variants of the network: host behaviour, and the GPU path against the host's formulas."""

from __future__ import annotations

import pytest
import torch

from alphatriangle_amd.config import EnvConfig, ModelConfig
from alphatriangle_amd.models.encoder import BoardEncoder
from alphatriangle_amd.models.model import AlphaTriangleNet

VARIANTS = [("relative", "pre"), ("differential", "pre"), ("softmax", "sandwich"), ("relative", "sandwich"), ("differential", "sandwich")]


def _small(attention: str, norm: str, **more) -> tuple[EnvConfig, ModelConfig]:  # noqa: ANN003
    env = EnvConfig(ROWS=3, COLS=4, PLAYABLE_RANGE_PER_ROW=[(0, 4)] * 3, NUM_SHAPE_SLOTS=1)
    return env, ModelConfig(
        CONV_FILTERS=[8], CONV_KERNEL_SIZES=[3], CONV_STRIDES=[1], CONV_PADDING=[1], NUM_RESIDUAL_BLOCKS=0, RESIDUAL_BLOCK_FILTERS=8, TRANSFORMER_DIM=32,
        TRANSFORMER_HEADS=4, TRANSFORMER_LAYERS=2, TRANSFORMER_FC_DIM=48, FC_DIMS_SHARED=[16], POLICY_HEAD_DIMS=[16], VALUE_HEAD_DIMS=[16],
        OTHER_NN_INPUT_FEATURES_DIM=14, TRANSFORMER_ATTENTION=attention, TRANSFORMER_NORM=norm, **more)


def _randomise(m: torch.nn.Module) -> None:
    """Every parameter off its starting value (zero biases and gates would hide their terms)."""
    g = torch.Generator().manual_seed(7)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(torch.randn(p.shape, generator=g).to(p) * 0.1)


@pytest.mark.parametrize("attention,norm", VARIANTS)
def test_network_trains_a_step_on_the_host(attention: str, norm: str):
    env, mc = _small(attention, norm)
    torch.manual_seed(0)
    net = AlphaTriangleNet(mc, env)
    assert isinstance(net.transformer_body, BoardEncoder)
    x, other = torch.rand(5, 1, 3, 4), torch.rand(5, 14)
    policy, value = net(x, other)
    (policy.square().mean() + value.square().mean()).backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in net.parameters())
    twin = AlphaTriangleNet(mc, env)
    twin.load_state_dict(net.state_dict())
    net.eval(), twin.eval()
    assert torch.equal(net(x, other)[0], twin(x, other)[0])


def test_default_network_is_untouched():
    env, mc = _small("softmax", "pre")
    net = AlphaTriangleNet(mc, env)
    assert isinstance(net.transformer_body, torch.nn.TransformerEncoder)
    stock = torch.nn.TransformerEncoderLayer(d_model=32, nhead=4, dim_feedforward=48, norm_first=True)
    assert list(net.transformer_body.layers[0].state_dict()) == list(stock.state_dict())


def test_relative_bias_breaks_the_symmetry_of_positions():
    """Without a bias the encoder commutes with permutations of its tokens; the learned board bias sees them."""
    env, mc = _small("relative", "pre")
    torch.manual_seed(1)
    body = AlphaTriangleNet(mc, env).transformer_body.double().eval()
    tokens, perm = torch.randn(12, 2, 32, dtype=torch.double), torch.randperm(12, generator=torch.Generator().manual_seed(0))
    assert torch.allclose(body(tokens)[perm], body(tokens[perm]), atol=1e-12)
    with torch.no_grad():
        for layer in body.layers:
            layer.position_bias.normal_()
    assert not torch.allclose(body(tokens)[perm], body(tokens[perm]), atol=1e-3)


@pytest.mark.parametrize("attention,norm", VARIANTS)
def test_body_gradients_by_differences(attention: str, norm: str):
    env, mc = _small(attention, norm)
    torch.manual_seed(2)
    body = AlphaTriangleNet(mc, env).transformer_body.double().eval()
    _randomise(body)
    tokens = torch.randn(12, 2, 32, dtype=torch.double)
    weight = torch.randn(12, 2, 32, dtype=torch.double)
    params = dict(body.named_parameters())
    grads = dict(zip(params, torch.autograd.grad((body(tokens) * weight).sum(), list(params.values()))))
    eps = 1e-6
    for name, p in params.items():
        direction = torch.randn_like(p)
        vals = []
        for s in (eps, -eps):
            with torch.no_grad():
                p.add_(s * direction)
                vals.append(float((body(tokens) * weight).sum()))
                p.sub_(s * direction)
        want = float((grads[name] * direction).sum())
        # fp64: rounding 1e-16 |f| / eps ~ 1e-8, truncation eps^2; parameters that cancel by symmetry (the key bias) are zero
        assert abs((vals[0] - vals[1]) / (2 * eps) - want) <= 1e-6 * max(1.0, abs(want)), name


def test_configuration_refusals():
    with pytest.raises(ValueError):
        ModelConfig(TRANSFORMER_ATTENTION="linear")
    with pytest.raises(ValueError):
        ModelConfig(TRANSFORMER_NORM="post")
    with pytest.raises(ValueError):
        ModelConfig(TRANSFORMER_ATTENTION="relative", TRANSFORMER_DIM=36, TRANSFORMER_HEADS=3)
    with pytest.raises(ValueError):
        ModelConfig(TRANSFORMER_ATTENTION="differential", TRANSFORMER_DIM=96, TRANSFORMER_HEADS=3)
    ModelConfig(TRANSFORMER_ATTENTION="relative", TRANSFORMER_DIM=96, TRANSFORMER_HEADS=3)
    env, mc = _small("relative", "sandwich")
    layer = AlphaTriangleNet(mc, env).transformer_body.layers[0]
    with pytest.raises(ValueError):
        layer(torch.zeros(12, 1, 32))
    env, mc = _small("relative", "pre")
    with pytest.raises(ValueError):
        AlphaTriangleNet(mc, env).transformer_body.layers[0](torch.zeros(12, 1, 32), src_mask=torch.zeros(12, 12))


def test_inference_engine_refuses_the_variants():
    from alphatriangle_amd.ops.inference import engine_supports

    assert engine_supports(ModelConfig(), EnvConfig(), "fp32")[0]
    for change in (dict(TRANSFORMER_ATTENTION="relative"), dict(TRANSFORMER_NORM="sandwich")):
        ok, why = engine_supports(ModelConfig(**change), EnvConfig(), "fp32")
        assert not ok and "encoder" in why


def test_command_line_options():
    from typer.testing import CliRunner

    from alphatriangle_amd.cli import app

    out = CliRunner().invoke(app, ["train", "--attention", "cosine"])
    assert out.exit_code != 0 and "attention" in out.output


@pytest.mark.gpu
@pytest.mark.parametrize("attention,norm", VARIANTS)
@pytest.mark.parametrize("bf16", [False, True])
def test_gpu_network_against_the_host(attention: str, norm: str, bf16: bool):
    """The default-sized network's outputs and every gradient: GPU kernels against the host's formulas in 64 bits."""
    env = EnvConfig()
    mc = ModelConfig(TRANSFORMER_ATTENTION=attention, TRANSFORMER_NORM=norm, USE_BATCH_NORM=False)
    torch.manual_seed(3)
    net = AlphaTriangleNet(mc, env)
    _randomise(net)
    net.eval()  # dropout off
    host = AlphaTriangleNet(mc, env).double().eval()
    host.load_state_dict(net.state_dict())
    net.cuda()
    tokens = torch.randn(120, 8, 128, generator=torch.Generator().manual_seed(4))
    weight = torch.randn(120, 8, 128, generator=torch.Generator().manual_seed(5))
    x = tokens.cuda().requires_grad_(True)
    with torch.autocast("cuda", torch.bfloat16, enabled=bf16):
        y = net.transformer_body(x)
    y.backward(weight.cuda().to(y.dtype))
    xr = tokens.double().requires_grad_(True)
    yr = host.transformer_body(xr)
    yr.backward(weight.double())

    def rel(a: torch.Tensor, b: torch.Tensor) -> float:
        return float((a.double().cpu() - b).norm() / b.norm())

    # two layers, each a chain of about ten products.  fp32: the learner's linear layers carry 16 bits per operand (2^-17, errors
    # of sums like independent ones, so about sqrt(20) 2^-17 = 3.4e-5 forward, twice that back; ten times for sums that
    # cancel).  bf16: every operand and result of the chain is rounded to 2^-9 rms at most: sqrt(40) 2^-9 = 1.2e-2 forward.
    # Gradients pass ReLUs: a hidden unit within the forward error e of zero may be open on one side only.  Of unit-variance
    # pre-images 2 * 0.4 e lie that near, and each takes or drops its whole share, so sqrt(0.8 e) of a layer's gradient may
    # differ: 5e-3 at e = 3.4e-5 (7e-3 over two layers), 1e-1 at e = 1.2e-2.
    assert rel(y.detach(), yr.detach()) <= (5e-2 if bf16 else 1e-4)
    assert rel(x.grad, xr.grad) <= (2e-1 if bf16 else 7e-3)
    for (name, p), pr in zip(net.transformer_body.named_parameters(), host.transformer_body.parameters()):
        if name.endswith("in_proj_bias"):
            d = 128  # the key bias takes no gradient (it shifts a row's scores alike)
            keep = torch.cat([torch.arange(d), torch.arange(2 * d, 3 * d)])
            assert rel(p.grad.cpu()[keep], pr.grad[keep]) <= (2e-1 if bf16 else 1e-2), name
        else:
            assert rel(p.grad, pr.grad) <= (2e-1 if bf16 else 1e-2), name


@pytest.mark.gpu
def test_learner_steps_with_a_variant():
    """The trainer's step (autocast, flat optimizer) on a network of every new part, three times; parameters move and stay finite."""
    from alphatriangle_amd.config import TrainConfig
    from alphatriangle_amd.models.network import NeuralNetwork
    from alphatriangle_amd.rl.core.trainer import Trainer
    from tests.conftest import make_experience

    import numpy as np

    dev = torch.device("cuda")
    env = EnvConfig()
    mc = ModelConfig(TRANSFORMER_ATTENTION="differential", TRANSFORMER_NORM="sandwich")
    tc = TrainConfig(DEVICE="cuda", BATCH_SIZE=16, USE_PER=False, MAX_TRAINING_STEPS=100, MIN_BUFFER_SIZE_TO_TRAIN=16, BUFFER_CAPACITY=100)
    net = NeuralNetwork(mc, env, tc, dev)
    assert net.engine is None
    trainer = Trainer(net, tc, env)
    rng = np.random.default_rng(0)
    before = {n: p.detach().clone() for n, p in net.model.named_parameters()}
    for _ in range(3):
        batch = [make_experience(mc, env, rng) for _ in range(16)]
        info = trainer.train_step({"batch": batch, "indices": np.arange(16), "weights": np.ones(16, dtype=np.float32)})
        assert info is not None
    torch.cuda.synchronize()
    moved = sum(not torch.equal(before[n], p) for n, p in net.model.named_parameters())
    assert moved >= 0.9 * len(before) and all(bool(torch.isfinite(p).all()) for p in net.model.parameters())


def test_command_line_options_reach_the_model(monkeypatch):
    from typer.testing import CliRunner

    import alphatriangle_amd.training.runner as runner
    from alphatriangle_amd.cli import app

    given = {}
    monkeypatch.setattr(runner, "run_training", lambda **kwargs: given.update(kwargs) or 0)
    for options, want in ((["--attention", "relative"], ("relative", "pre")), (["--encoder-norm", "sandwich"], ("softmax", "sandwich")),
                          (["--preset", "large", "--attention", "differential", "--encoder-norm", "sandwich"], ("differential", "sandwich"))):
        given.clear()
        out = CliRunner().invoke(app, ["train", *options])
        mc = given["model_config_override"]
        assert out.exit_code == 0 and (mc.TRANSFORMER_ATTENTION, mc.TRANSFORMER_NORM) == want
    for options in (["--attention", "relative"], ["--encoder-norm", "sandwich"], ["--attention", "softmax"]):
        for preset in ("tiny", "cnn"):
            given.clear()
            out = CliRunner().invoke(app, ["train", "--preset", preset, *options])
            assert out.exit_code != 0 and not given and "encoder" in out.output


@pytest.mark.gpu
@pytest.mark.parametrize("attention,norm", VARIANTS)
@pytest.mark.parametrize("bf16", [False, True])
def test_learner_step_of_a_variant_is_captured(attention: str, norm: str, bf16: bool):
    """The trainer's forward and backward pass is replayed from a graph that holds no memset node and reproduces the eager gradients."""
    from alphatriangle_amd.config import TrainConfig
    from alphatriangle_amd.models.network import NeuralNetwork
    from alphatriangle_amd.rl.core.trainer import TensorBatch, Trainer

    dev = torch.device("cuda")
    env, mc = EnvConfig(), ModelConfig(TRANSFORMER_ATTENTION=attention, TRANSFORMER_NORM=norm)
    tc = TrainConfig(DEVICE="cuda", BATCH_SIZE=32, MAX_TRAINING_STEPS=100, COMPILE_MODEL=True)
    torch.manual_seed(3)
    trainer = Trainer(NeuralNetwork(mc, env, tc, dev), tc, env, autocast_bf16=bf16)
    gen = torch.Generator().manual_seed(5)
    for _ in range(3):
        policy = torch.rand(32, env.ACTION_DIM, generator=gen)
        tb = TensorBatch(torch.randint(-1, 2, (32, 1, env.ROWS, env.COLS), generator=gen).float().to(dev),
                         torch.rand(32, mc.OTHER_NN_INPUT_FEATURES_DIM, generator=gen).to(dev), (policy / policy.sum(1, keepdim=True)).to(dev),
                         torch.empty(32).uniform_(-5, 5, generator=gen).to(dev), torch.ones(32, device=dev))
        info, _ = trainer.train_step_tensors(tb)
        torch.cuda.synchronize()
    report = trainer.graph_report
    assert trainer.use_graph and report["replayed"] and report["memset_nodes"] == 0 and report["max_rel_err"] <= 1e-3, report
    assert bool(torch.isfinite(info["total_loss"])) and bool(torch.isfinite(trainer.flat.flat_param).all())


@pytest.mark.gpu
@pytest.mark.parametrize("attention,norm", [("relative", "pre"), ("differential", "sandwich")])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_self_play_with_a_variant(attention: str, norm: str, dtype: str):
    """Games played on the device tree with leaves through the module (its encoder through the kernels), before and after the
    learner hands over new weights; the leaf values are the module's on the host in 64 bits."""
    from alphatriangle_amd.rl.self_play.gpu_actor import ModuleEvaluator
    from tests.test_gpu_engine import _actor

    mc = ModelConfig(TRANSFORMER_ATTENTION=attention, TRANSFORMER_NORM=norm)
    actor, replay, _ = _actor(games=24, sims=8, dtype=dtype, model=mc)
    assert actor.nn.engine is None and isinstance(actor.evaluator, ModuleEvaluator)
    for step in range(4):
        rep = actor.play_move()
        assert rep.moves == actor.G and rep.simulations >= actor.G * 8
        if step == 1:
            _randomise(actor.nn._orig_model)
            actor.sync_weights(1)
    n = len(replay)
    assert n > 0 and bool(torch.isfinite(replay.ret[:n]).all())
    assert torch.allclose(replay.policy[:n].sum(1), torch.ones(n, device=replay.policy.device), atol=1e-4)
    ev = actor.evaluator
    env = actor.nn.env_config
    gen = torch.Generator().manual_seed(1)
    grid, other = torch.randint(-1, 2, (24, env.ROWS * env.COLS), generator=gen).float(), torch.rand(24, mc.OTHER_NN_INPUT_FEATURES_DIM, generator=gen)
    ev.forward(grid.cuda(), other.cuda())
    host = AlphaTriangleNet(mc, env).double().eval()
    host.load_state_dict(actor.nn._orig_model.state_dict())
    with torch.no_grad():
        want = host(grid.double().view(24, 1, env.ROWS, env.COLS), other.double())[0]
    got = ev.logits[:24, : want.shape[1]].double().cpu()
    # bf16: about forty operands and results of the chain rounded to 2^-9 rms at most, sqrt(40) 2^-9 = 1.2e-2; fp32: library convolutions
    # and linear layers of 16 bits per operand, sqrt(40) 2^-17 = 5e-5; four times either for ReLUs and normalisations
    assert float((got - want).norm() / want.norm()) <= (5e-2 if dtype == "bf16" else 2e-4)
