"""A small model of gated recurrent blocks, trained on windows and run on-line sample by sample.

    python examples/gated_block.py [--steps 200] [--device cuda]

Each block is ``norm -> projections -> gated recurrence -> gated norm -> projection`` beside a residual
stream; ``residual_norm`` joins a block to the next one. Training walks windows of a simulated
nonlinear system with ``gated_recurrence``; the on-line run carries each block's state and calls
``gated_recurrence_step`` once a sample, which gives what the whole-sequence pass gives. The example
prints the training loss and how far the two runs differ.
"""

from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from tsfast_amd.gated import gated_norm, gated_recurrence, gated_recurrence_step, residual_norm  # noqa: E402


class GatedBlock(nn.Module):
    """The block between two norms: ``width`` columns in and out, ``heads`` states of ``key x value``, queries and
    keys shared by groups of heads."""

    def __init__(self, width: int, heads: int, key_heads: int, key: int, value: int):
        super().__init__()
        self.heads, self.key_heads, self.key, self.value = heads, key_heads, key, value
        self.sizes = (key_heads * key, key_heads * key, heads * value, heads * value, heads)
        self.inp = nn.Linear(width, sum(self.sizes), bias=False)
        self.out = nn.Linear(heads * value, width, bias=False)
        self.head_norm = nn.Parameter(torch.ones(heads * value))
        # decays from a few steps to a few hundred at the start: exp(-rate softplus(.)) a step
        self.rate = nn.Parameter(torch.linspace(math.log(3e-3), math.log(0.3), heads))
        # what joins this block to the next: post-norm, residual scale, the next block's pre-norm
        self.post = nn.Parameter(torch.ones(width))
        self.scale = nn.Parameter(torch.full((width,), 0.5))
        self.next = nn.Parameter(torch.ones(width))

    def _projections(self, x):
        q, k, v, gate, decay = self.inp(x).split(self.sizes, -1)
        q = q.unflatten(-1, (self.key_heads, self.key)) / math.sqrt(self.key)
        k = F.normalize(k.unflatten(-1, (self.key_heads, self.key)), dim=-1)
        g = -self.rate.exp() * F.softplus(decay)
        return q, k, v.unflatten(-1, (self.heads, self.value)), gate, g

    def _output(self, o, gate, stream):
        y = gated_norm(o.flatten(-2), gate, self.head_norm, groups=self.heads)
        return residual_norm(self.out(y), stream, self.next, post_weight=self.post, scale=self.scale)

    def forward(self, x, stream, state=None):
        """``x [B, L, width]`` (normed), the residual stream: the new stream, the next block's input, the state."""
        q, k, v, gate, g = self._projections(x)
        o, state = gated_recurrence(q, k, v, g, state)
        return *self._output(o, gate, stream), state

    def step(self, x, stream, state):
        """The same for one sample ``[B, width]``; ``state`` is updated in place."""
        q, k, v, gate, g = self._projections(x)
        o = gated_recurrence_step(q, k, v, g, state)
        return self._output(o, gate, stream)

    def zero_state(self, batch: int, device):
        return torch.zeros(batch, self.heads, self.key, self.value, device=device)


class GatedModel(nn.Module):
    """Input signals to output signals through ``depth`` blocks."""

    def __init__(self, inputs: int, outputs: int, width: int = 64, depth: int = 2, heads: int = 4, key_heads: int = 2, key: int = 16, value: int = 24):
        super().__init__()
        self.embed = nn.Linear(inputs, width)
        self.first = nn.Parameter(torch.ones(width))
        self.blocks = nn.ModuleList(GatedBlock(width, heads, key_heads, key, value) for _ in range(depth))
        self.read = nn.Linear(width, outputs)

    def forward(self, u, states=None):
        """``u [B, L, inputs]``: outputs ``[B, L, outputs]`` and the blocks' states."""
        stream = self.embed(u)
        x, out = gated_norm(stream, None, self.first), []
        for block, state in zip(self.blocks, states or [None] * len(self.blocks)):
            stream, x, state = block(x, stream, state)
            out.append(state)
        return self.read(x), out

    @torch.no_grad()
    def step(self, u, states):
        """One sample ``[B, inputs]``; ``states`` are updated in place."""
        stream = self.embed(u)
        x = gated_norm(stream, None, self.first)
        for block, state in zip(self.blocks, states):
            stream, x = block.step(x, stream, state)
        return self.read(x)

    def zero_states(self, batch: int, device):
        return [block.zero_state(batch, device) for block in self.blocks]


def windows(batch: int, length: int, generator, device):
    """Inputs and outputs of a damped oscillator with a saturated input, ``[batch, length, 1]`` each."""
    u = torch.randn(batch, length, generator=generator).cumsum(1) * 0.2
    drive = torch.tanh(u)
    y, v, out = torch.zeros(batch), torch.zeros(batch), []
    for t in range(length):
        v = 0.96 * v + 0.1 * (drive[:, t] - y)
        y = y + 0.2 * v
        out.append(y)
    return u[..., None].to(device), torch.stack(out, 1)[..., None].to(device)


def train(model, steps: int, device, batch: int = 16, length: int = 200, seed: int = 0):
    """Trains on random windows; the loss of each step."""
    r = torch.Generator().manual_seed(seed)
    optim, losses = torch.optim.Adam(model.parameters(), lr=3e-3), []
    for _ in range(steps):
        u, y = windows(batch, length, r, device)
        loss = F.mse_loss(model(u)[0], y)
        optim.zero_grad()
        loss.backward()
        optim.step()
        losses.append(loss.item())
    return losses


@torch.no_grad()
def online(model, u):
    """The outputs sample by sample, as a program that receives ``u`` on-line has them."""
    states = model.zero_states(u.shape[0], u.device)
    return torch.stack([model.step(u[:, t], states) for t in range(u.shape[1])], 1)


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    args = parser.parse_args(argv)
    torch.manual_seed(0)
    model = GatedModel(1, 1).to(args.device)
    losses = train(model, args.steps, args.device)
    u, y = windows(4, 300, torch.Generator().manual_seed(1), args.device)
    with torch.no_grad():
        whole, _ = model(u)
    apart = (online(model, u) - whole).abs().max().item()
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}; validation {F.mse_loss(whole, y).item():.4f}; on-line against whole sequence {apart:.1e}")
    return losses, apart


if __name__ == "__main__":
    main()
