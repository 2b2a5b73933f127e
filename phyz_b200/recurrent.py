"""A recurrent model of a rollout, on the operators of nn.py: what a policy or a
dynamics model with memory is made of.

    h = silu(obs W_in^T + b)
    per block:  (x | gate) = h W_z^T + b,  s = gated_scan(x, gate),  h = h + gelu(s W_o^T + b)
    y = h W_out^T + b

The layers multiply in bf16 from working copies of f32 weights; the memory is
f32. Training walks whole rollouts [world][step] with episode resets, backwards
through time with the operators' own gradients, and updates every matrix with
Muon (biases by momentum). Serving keeps the memory between control steps.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import nn


@dataclass
class RecurrentCfg:
    n_in: int
    n_out: int
    width: int = 128
    blocks: int = 2
    lr: float = 0.02         # of the matrices (Muon)
    bias_lr: float = 0.02
    momentum: float = 0.95
    weight_decay: float = 0.0


class _Layer:
    """A linear layer's f32 weights, their momentum, and the bf16 copy that multiplies."""

    def __init__(self, n_out: int, n_in: int, device, gen: torch.Generator, gain: float = 1.0):
        self.master = torch.randn(n_out, n_in, device=device, generator=gen) * (gain / math.sqrt(n_in))
        self.bias = torch.zeros(n_out, device=device)
        self.momentum, self.bias_momentum = torch.zeros_like(self.master), torch.zeros_like(self.bias)
        self.weight = self.master.to(torch.bfloat16)
        self.grad = self.bias_grad = None

    def __call__(self, x, **kw):
        return nn.linear(x, self.weight, self.bias, **kw)

    def backward(self, dy, x, pre=None, **kw):
        dx, self.grad, self.bias_grad = nn.linear_backward(dy, x, self.weight, pre, **kw)
        return dx

    def update(self, cfg: RecurrentCfg) -> None:
        nn.muon_update(self.master, self.grad, self.momentum, lr=cfg.lr, mu=cfg.momentum,
                       weight_decay=cfg.weight_decay, copy=self.weight)
        self.bias_momentum.mul_(cfg.momentum).add_(self.bias_grad)
        self.bias.add_(self.bias_momentum, alpha=-cfg.bias_lr)


class RecurrentModel:
    """Rows in and out are [worlds, steps, features] in bfloat16; reset [worlds, steps] marks episode starts.

    Nothing here waits for the device. `nn.status()` does, and raises if a kernel gave up a wait and left its outputs
    unfinished: to be called where a program waits anyway, such as before it saves a checkpoint."""

    def __init__(self, cfg: RecurrentCfg, device: int = 0, seed: int = 0):
        self.cfg, self.device = cfg, torch.device("cuda", device)
        gen = torch.Generator(device=self.device).manual_seed(seed)
        d = cfg.width
        self.inp = _Layer(d, cfg.n_in, self.device, gen)
        self.blocks = [(_Layer(2 * d, d, self.device, gen), _Layer(d, d, self.device, gen, 0.5))
                       for _ in range(cfg.blocks)]
        for z, _ in self.blocks:
            z.bias[d:] = torch.linspace(0.0, 4.0, d, device=self.device)  # memories of 2 to 50 steps
        self.out = _Layer(cfg.n_out, d, self.device, gen)

    def layers(self):
        return [self.inp, *(layer for block in self.blocks for layer in block), self.out]

    def start(self, worlds: int):
        """The memory of worlds at the start of an episode."""
        return [torch.zeros(worlds, self.cfg.width, device=self.device) for _ in self.blocks]

    def forward(self, obs, state=None, reset=None, save: bool = True):
        """(y [b, t, n_out], the memory after the last step, what `backward` needs)."""
        b, t, _ = obs.shape
        d = self.cfg.width
        state = self.start(b) if state is None else state
        x0 = obs.reshape(b * t, -1)
        h = self.inp(x0, activation="silu", save_pre=save)
        saved, last = [(x0, h[1])] if save else None, []
        h = h[0] if save else h
        for (zl, ol), s0 in zip(self.blocks, state):
            z = zl(h).view(b, t, 2 * d)
            s, end = nn.gated_scan(z[..., :d], z[..., d:], s0, reset)
            rows = s.view(b * t, d)
            y = ol(rows, activation="gelu", residual=h, save_pre=save)
            if save:
                saved.append((h, z, s, rows, s0, y[1]))
            h = y[0] if save else y
            last.append(end)
        y = self.out(h)
        if save:
            saved.append(h)
        return y.view(b, t, -1), last, saved

    def backward(self, dy, saved, reset=None) -> None:
        """Every layer's gradients from dy [b, t, n_out]."""
        b, t, _ = dy.shape
        d = self.cfg.width
        dh = self.out.backward(dy.reshape(b * t, -1), saved[-1])
        for (zl, ol), (h, z, s, rows, s0, pre) in zip(reversed(self.blocks), reversed(saved[1:-1])):
            ds = ol.backward(dh, rows, pre, activation="gelu")
            dz = torch.empty_like(z)
            nn.gated_scan_backward(ds.view(b, t, d), z[..., :d], z[..., d:], s, s0, reset,
                                   out=(dz[..., :d], dz[..., d:]))
            dh = dh + zl.backward(dz.view(b * t, 2 * d), h)
        x0, pre = saved[0]
        self.inp.backward(dh, x0, pre, activation="silu", need_dx=False)

    def update(self) -> None:
        for layer in self.layers():
            layer.update(self.cfg)

    def train_step(self, obs, target, reset=None) -> torch.Tensor:
        """One update on the mean squared error of y against target; returns the loss (on the device)."""
        y, _, saved = self.forward(obs, None, reset)
        off = y.float() - target.float()
        self.backward((off * (2.0 / off.numel())).to(torch.bfloat16), saved, reset)
        self.update()
        return (off * off).mean()

    def step(self, obs, state, reset=None):
        """One control step of every world: obs [worlds, n_in] -> (y [worlds, n_out], the memory after it)."""
        y, state, _ = self.forward(obs[:, None], state, None if reset is None else reset[:, None], save=False)
        return y[:, 0], state
