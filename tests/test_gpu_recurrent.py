"""The recurrent model on the operators (phyz_b200.recurrent): its gradients against autograd in 64 bits on the same
weights, serving step by step against the whole sequence, and the example end to end."""
import sys
from pathlib import Path

import pytest
import torch

from phyz_b200.recurrent import RecurrentCfg, RecurrentModel

pytestmark = pytest.mark.gpu


def forward64(model, weights, obs, reset):
    """The model's formulas in 64 bits; weights: [(w, b)] of model.layers()."""
    d = model.cfg.width
    it = iter(weights)

    def layer(x):
        w, b = next(it)
        return x @ w.t() + b

    h = torch.nn.functional.silu(layer(obs))
    for _ in model.blocks:
        z = layer(h)
        x, a = z[..., :d], torch.sigmoid(z[..., d:])
        s, out = torch.zeros_like(x[:, 0]), []
        for t in range(obs.shape[1]):
            s = torch.where(reset[:, t, None] != 0, torch.zeros_like(s), s)
            s = a[:, t] * s + (1 - a[:, t]) * x[:, t]
            out.append(s)
        h = h + torch.nn.functional.gelu(layer(torch.stack(out, 1)), approximate="tanh")
    return layer(h)


def setup(worlds=6, steps=20, n_in=30, n_out=11, width=48):
    g = torch.Generator(device="cuda").manual_seed(5)
    model = RecurrentModel(RecurrentCfg(n_in=n_in, n_out=n_out, width=width, blocks=2), seed=3)
    obs = torch.randn(worlds, steps, n_in, generator=g, device="cuda").to(torch.bfloat16)
    reset = (torch.rand(worlds, steps, generator=g, device="cuda") < 0.15).to(torch.uint8)
    dy = (torch.randn(worlds, steps, n_out, generator=g, device="cuda") * 0.1).to(torch.bfloat16)
    return model, obs, reset, dy


def test_gradients_against_autograd():
    """A handful of bf16 roundings (2^-8 each, on values that partly cancel) lie between a gradient and its 64-bit
    value: 12 of them in the deepest path, so 12 * 2^-8 of its 2-norm."""
    model, obs, reset, dy = setup()
    y, _, saved = model.forward(obs, None, reset)
    model.backward(dy, saved, reset)
    weights = [(la.weight.double().requires_grad_(), la.bias.double().requires_grad_()) for la in model.layers()]
    want = forward64(model, weights, obs.double(), reset)
    assert (y.double() - want).norm() <= 12 * 2.0 ** -8 * want.norm()
    want.backward(dy.double())
    for la, (w, b) in zip(model.layers(), weights):
        assert (la.grad.double() - w.grad).norm() <= 12 * 2.0 ** -8 * w.grad.norm()
        assert (la.bias_grad.double() - b.grad).norm() <= 12 * 2.0 ** -8 * b.grad.norm()


def test_update_moves_every_layer_and_its_copy():
    model, obs, reset, dy = setup()
    before = [la.master.clone() for la in model.layers()]
    target = torch.zeros(obs.shape[0], obs.shape[1], model.cfg.n_out, device="cuda", dtype=torch.bfloat16)
    model.train_step(obs, target, reset)
    for la, old in zip(model.layers(), before):
        assert not torch.equal(la.master, old)
        assert torch.equal(la.weight, la.master.to(torch.bfloat16))


def test_serving_is_the_sequence():
    """Step by step the same roundings happen in the same places, but for sums in another order: a few bf16 ulps."""
    model, obs, reset, _ = setup(worlds=70)
    y, last, _ = model.forward(obs, None, reset, save=False)
    state = model.start(obs.shape[0])
    for t in range(obs.shape[1]):
        out, state = model.step(obs[:, t], state, reset[:, t])
        assert (out.float() - y[:, t].float()).abs().max() <= 8 * 2.0 ** -8 * y.float().abs().max()
    for a, b in zip(state, last):
        assert (a - b).abs().max() <= 8 * 2.0 ** -8 * b.abs().max()


def test_example_learns():
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    import learn_dynamics

    losses = learn_dynamics.main(["--worlds", "256", "--steps", "32", "--updates", "41"])
    assert losses[-1] < 0.8 * losses[0]
