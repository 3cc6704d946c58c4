"""A model of logged frames with a state instead of a cache: decay attention and a gated feed-forward in every block.

Each replica of an ensemble logs a few numbers per frame (energy, temperature, pressure, ...) for as long as it runs. A cache
of all frames would grow with the run; here every head carries one matrix along, which forgets at the head's own rate, so that
a new frame costs the same after a million steps, and the order of the frames is in the decay: no table of positions ends. The
model runs the operators together as they are used:

* ``decay_attention``: whole packed histories with their gradients, and chunks of a history that follow a state;
* ``decay_attention_step``: one new frame of every replica, its state moved on in place;
* ``gated_feed_forward``: the other half of each block, forward and backward.

    python examples/frame_memory.py [--dtype float32|bfloat16] [--replicas 64] [--steps 20]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import nn
from torch.nn.functional import rms_norm

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from examples.frame_attention import made_up_log  # noqa: E402
from fastmd_b200.decay_attention import decay_attention, decay_attention_step  # noqa: E402
from fastmd_b200.gated_feed_forward import gated_feed_forward  # noqa: E402


class MemoryBlock(nn.Module):
    """Decay attention over a replica's frames and a gated feed-forward, both added to the rows they read."""

    def __init__(self, width: int, heads: int, dim: int, hidden: int):
        super().__init__()
        self.heads, self.dim = heads, dim
        self.norm_in, self.norm_feed = nn.LayerNorm(width), nn.LayerNorm(width)
        self.qkv = nn.Linear(width, 3 * heads * dim, bias=False)
        self.q_weight, self.k_weight, self.o_weight = (nn.Parameter(torch.ones(dim)) for _ in range(3))
        self.out = nn.Linear(heads * dim, width, bias=False)
        self.gate, self.up = nn.Linear(width, hidden, bias=False), nn.Linear(width, hidden, bias=False)
        self.down = nn.Linear(hidden, width, bias=False)

    def qkv_heads(self, x):
        """Queries and keys (each head of root mean square 1, times its weight) and values of the rows."""
        q, k, v = self.qkv(self.norm_in(x)).unflatten(1, (-1, self.dim)).split(self.heads, 1)
        return rms_norm(q, (self.dim,), self.q_weight, 1e-6), rms_norm(k, (self.dim,), self.k_weight, 1e-6), v

    def rest(self, x, read):
        # a replica's first frames can read next to nothing (a query almost at a right angle to the few keys): the constant
        # keeps their rounding errors, and their gradients, from being blown up to size one
        x = x + self.out(rms_norm(read, (self.dim,), self.o_weight, 0.1).flatten(1))
        return x + gated_feed_forward(self.norm_feed(x), self.gate.weight, self.up.weight, self.down.weight)


class MemoryModel(nn.Module):
    """Predicts the next frame's features from a replica's frames so far."""

    def __init__(self, features: int, *, width: int = 256, heads: int = 4, dim: int = 64, hidden: int = 512, layers: int = 2,
                 device=None, dtype=torch.float32):
        super().__init__()
        self.embed, self.read = nn.Linear(features, width), nn.Linear(width, features)
        self.blocks = nn.ModuleList(MemoryBlock(width, heads, dim, hidden) for _ in range(layers))
        # half-lives from one frame to some hundreds
        rate = 2.0 ** -(1 + 8 * (torch.arange(heads, device=device, dtype=torch.float64) + 0.5) / heads)
        self.register_buffer("log_decay", torch.log1p(-rate).float())
        self.to(device=device, dtype=dtype)

    def _apply(self, fn, *args, **kwargs):
        # the decays move with the model, but stay in FP32 whatever its type becomes
        given = self.log_decay
        super()._apply(fn, *args, **kwargs)
        self.log_decay = given.to(self.log_decay.device)
        return self

    def forward(self, frames, offsets, states=None, return_states=False):
        """Predictions after every frame: frames ``[rows, features]`` packed by ``offsets``. ``states``, one a block, are those
        that the last call returned (``new_states`` before the first)."""
        x, after = self.embed(frames), []
        for i, block in enumerate(self.blocks):
            read = decay_attention(*block.qkv_heads(x), self.log_decay, offsets, None if states is None else states[i],
                                   return_state=return_states)
            if return_states:
                read, state = read
                after.append(state)
            x = block.rest(x, read)
        return (self.read(x), after) if return_states else self.read(x)

    def new_states(self, replicas: int):
        block = self.blocks[0]
        shape = (replicas, block.heads, block.dim, block.dim)
        return [torch.zeros(shape, device=self.embed.weight.device) for _ in self.blocks]

    @torch.no_grad()
    def step(self, frames, states):
        """Predictions after one new frame ``[replicas, features]`` of every replica; the states move on by it in place. No
        length is read on the host, so the call can be captured in a CUDA graph and replayed."""
        x = self.embed(frames)
        for block, state in zip(self.blocks, states):
            x = block.rest(x, decay_attention_step(*block.qkv_heads(x), self.log_decay, state))
        return self.read(x)


def next_frame_loss(model, frames, offsets):
    """Mean squared error of the prediction after every frame but the replicas' last ones."""
    predicted = model(frames, offsets).float()
    keep = torch.ones(frames.shape[0], dtype=torch.bool, device=frames.device)
    keep[offsets[1:] - 1] = False
    return (predicted[:-1] - frames[1:].float()).square().mean(1)[keep[:-1]].mean()


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--dtype", choices=("float32", "bfloat16"), default="float32")
    parser.add_argument("--replicas", type=int, default=64)
    parser.add_argument("--longest", type=int, default=500)
    parser.add_argument("--steps", type=int, default=20)
    args = parser.parse_args(argv)
    torch.manual_seed(0)
    dtype = getattr(torch, args.dtype)
    model = MemoryModel(4, device="cuda", dtype=dtype)
    frames, _, offsets = made_up_log(args.replicas, args.longest, 4, dtype=dtype)
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3)
    for i in range(args.steps):
        optimizer.zero_grad()
        loss = next_frame_loss(model, frames, offsets)
        loss.backward()
        optimizer.step()
        if i in (0, args.steps - 1):
            print(f"training step {i + 1}: loss {float(loss.detach()):.4f}")
    with torch.no_grad():
        predicted, states = model(frames, offsets, return_states=True)
    frame = predicted[offsets[1:] - 1]
    for _ in range(10):
        frame = model.step(frame, states)
    print(f"ten frames of {args.replicas} replicas rolled out; the first replica's last: "
          f"{[round(float(v), 3) for v in frame[0]]}")


if __name__ == "__main__":
    main()
