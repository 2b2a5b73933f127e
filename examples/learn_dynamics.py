"""Learn the quadruped's next observation from its rollouts, then serve the model
step by step.

The simulator rolls a batch of quadrupeds under a random policy with its
on-device control loop; the policy history ([step][feature][world], on the GPU)
is the training data of a recurrent model (phyz_b200.recurrent), which sees an
observation and the action taken and predicts how the observation changes. Then
the model runs one control step at a time, its memory on the device.

    python examples/learn_dynamics.py [--worlds N] [--steps T] [--updates K] [--width D]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from phyz_b200 import BatchSim, configs, nn  # noqa: E402
from phyz_b200.policy import random_weights  # noqa: E402
from phyz_b200.recurrent import RecurrentCfg, RecurrentModel  # noqa: E402


def rollout(worlds: int, steps: int, seed: int):
    """(inputs [world, step, observation + action], change of the observation [world, step, observation]) of a rollout,
    both scaled per feature."""
    model = configs.quadruped()
    sim = BatchSim(model, worlds, precision="f32")
    sim.enable_ground_contact(*configs.CONFIGS["c3_quadruped"].contact)
    pd = configs.c5_pd_dofs(model)
    sim.enable_pd_control(pd)
    spec = configs.c5_policy_spec(model)
    spec.history_steps = steps + 1
    sim.enable_policy(spec)
    sim.set_policy_base_targets(np.zeros((worlds, len(pd))))
    sim.set_policy_weights(random_weights(spec, seed))
    sim.set_policy_std(np.full(spec.n_out, configs.C5_STD))
    sim.seed_policy(seed)
    q0, v0 = configs.initial_state("c3_quadruped", model, np.arange(worlds))
    sim.load_states(q0, v0)
    sim.policy_rollout(0, steps, 4)
    sim.run_policy(steps)
    sim.sync()
    obs, out = sim.readback_policy_history(0, steps + 1)  # [step][world][feature], rows for the host
    sim.close()
    obs = torch.from_numpy(obs).cuda().transpose(0, 1)
    act = torch.from_numpy(out[..., :-1].copy()).cuda().transpose(0, 1)
    x, change = torch.cat([obs, act], 2)[:, :-1], obs[:, 1:] - obs[:, :-1]
    keep = torch.isfinite(x).all(2).all(1) & torch.isfinite(change).all(2).all(1)

    def scaled(v):
        v = v[keep]
        return ((v - v.mean((0, 1))) / (v.std((0, 1)) + 1e-3)).clamp(-8, 8).to(torch.bfloat16).contiguous()

    return scaled(x), scaled(change)


def main(argv=None) -> list[float]:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--worlds", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--updates", type=int, default=100)
    ap.add_argument("--width", type=int, default=128)
    a = ap.parse_args(argv)
    x, change = rollout(a.worlds, a.steps, 7)
    model = RecurrentModel(RecurrentCfg(n_in=x.shape[2], n_out=change.shape[2], width=a.width))
    # two episodes of half the rollout each, as a training batch has them
    reset = torch.zeros(x.shape[:2], dtype=torch.uint8, device="cuda")
    reset[:, 0] = reset[:, a.steps // 2] = 1
    losses = []
    for k in range(a.updates):
        loss = model.train_step(x, change, reset)
        if k % 10 == 0 or k == a.updates - 1:
            losses.append(float(loss))
            print(f"update {k:4d}  mean squared error {losses[-1]:.4f}")
    # served step by step, the memory kept between calls
    y, _, _ = model.forward(x, None, reset, save=False)
    state, worst = model.start(x.shape[0]), 0.0
    for t in range(x.shape[1]):
        out, state = model.step(x[:, t], state, reset[:, t])
        worst = max(worst, float((out.float() - y[:, t].float()).abs().max()))
    nn.status()
    print(f"served {x.shape[1]} steps of {x.shape[0]} worlds: at most {worst:.3g} from the whole-sequence outputs")
    return losses


if __name__ == "__main__":
    main()
