"""A small causal model of logged frames: packed training over whole histories, then one new frame at a time.

Each replica of an ensemble logs a few numbers per frame (energy, temperature, pressure, ...), each for as long as it has
run. The model reads the frames of all replicas as packed sequences and predicts every next frame. It runs the sequence
operators together as they are used:

* ``head_norm_rotary``: norm of the query and key heads and rotation by the frame's MD step, forward and backward;
* ``packed_attention``: causal attention within each replica's history, grouped heads, forward and backward; and its
  form for one new frame of every replica against a cache that holds the keys and values of the frames so far.

    python examples/frame_attention.py [--dtype float32|bfloat16] [--replicas 64] [--steps 20]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from fastmd_b200.head_rotary import head_norm_rotary, rotary_table  # noqa: E402
from fastmd_b200.packed_attention import packed_attention  # noqa: E402


class FrameBlock(nn.Module):
    """Attention over a replica's frames and an MLP, both added to the rows they read."""

    def __init__(self, width: int, heads: int, key_heads: int, dim: int):
        super().__init__()
        self.sizes = (heads, key_heads, key_heads)
        self.dim = dim
        self.norm_in, self.norm_mlp = nn.LayerNorm(width), nn.LayerNorm(width)
        self.qkv = nn.Linear(width, sum(self.sizes) * dim, bias=False)
        self.q_weight, self.k_weight = nn.Parameter(torch.ones(dim)), nn.Parameter(torch.ones(dim))
        self.out = nn.Linear(heads * dim, width, bias=False)
        self.mlp = nn.Sequential(nn.Linear(width, 2 * width), nn.SiLU(), nn.Linear(2 * width, width))

    def heads(self, x, steps, table):
        """Queries, keys (both with norm and rotation) and values of the rows: three views of one projection."""
        q, k, v = self.qkv(self.norm_in(x)).unflatten(1, (-1, self.dim)).split(self.sizes, 1)
        q, k = head_norm_rotary(q, k, steps, *table, self.q_weight, self.k_weight)
        return q, k, v

    def rest(self, x, attended):
        x = x + self.out(attended.flatten(1))
        return x + self.mlp(self.norm_mlp(x))


class FrameModel(nn.Module):
    """Predicts the next frame's features from a replica's frames so far."""

    def __init__(self, features: int, *, width: int = 256, heads: int = 8, key_heads: int = 2, dim: int = 64,
                 layers: int = 2, max_steps: int = 10_000, device=None, dtype=torch.float32):
        super().__init__()
        self.embed, self.read = nn.Linear(features, width), nn.Linear(width, features)
        self.blocks = nn.ModuleList(FrameBlock(width, heads, key_heads, dim) for _ in range(layers))
        self.to(device=device, dtype=dtype)
        self.table = rotary_table(max_steps, dim, device=device)

    def forward(self, frames, steps, offsets):
        """Predictions after every frame: frames ``[rows, features]`` packed by ``offsets``, their MD steps int64."""
        x = self.embed(frames)
        for block in self.blocks:
            q, k, v = block.heads(x, steps, self.table)
            x = block.rest(x, packed_attention(q, k, v, offsets, causal=True))
        return self.read(x)

    def new_cache(self, replicas: int, capacity: int):
        """Room for the last `capacity` frames of each replica: a slot per replica, filled as far as its count."""
        if capacity < 1:
            raise ValueError(f"a cache needs room for a frame, got {capacity}")
        weight = self.embed.weight
        shape = (replicas * capacity, self.blocks[0].sizes[1], self.blocks[0].dim)
        layers = [tuple(torch.zeros(shape, device=weight.device, dtype=weight.dtype) for _ in "kv")
                  for _ in self.blocks]
        starts = torch.arange(replicas + 1, device=weight.device) * capacity
        return {"layers": layers, "starts": starts, "counts": torch.zeros_like(starts[1:]),
                "frames": torch.zeros_like(starts[1:]), "capacity": capacity,
                "rows": torch.arange(replicas + 1, device=weight.device)}

    @torch.no_grad()
    def step(self, frames, steps, cache):
        """Predictions after one new frame ``[replicas, features]`` of every replica; the cache grows by it. In a full
        slot it takes the oldest frame's place: a new row sees all keys of its slot, and their order does not count. No
        length is read on the host, so the call can be captured in a CUDA graph and replayed."""
        at = cache["starts"][:-1] + cache["frames"] % cache["capacity"]
        cache["frames"] += 1
        torch.clamp(cache["frames"], max=cache["capacity"], out=cache["counts"])
        x = self.embed(frames)
        for block, (keys, values) in zip(self.blocks, cache["layers"]):
            q, k, v = block.heads(x, steps, self.table)
            keys.index_copy_(0, at, k)
            values.index_copy_(0, at, v)
            x = block.rest(x, packed_attention(q, keys, values, cache["rows"], cache["starts"], cache["counts"],
                                               causal=True))
        return self.read(x)


def made_up_log(replicas: int, longest: int, features: int, *, seed: int = 0, device="cuda", dtype=torch.float32):
    """Packed frames of damped oscillations with noise: ``(frames, steps, offsets)``, replica lengths 2 .. longest."""
    gen = torch.Generator().manual_seed(seed)
    lengths = torch.randint(2, longest + 1, (replicas,), generator=gen)
    offsets = torch.cat((torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)))
    steps = torch.cat([torch.arange(int(n)) for n in lengths])
    replica = torch.repeat_interleave(torch.arange(replicas), lengths)
    rate, phase = torch.rand(replicas, features, generator=gen), 6.3 * torch.rand(replicas, features, generator=gen)
    frames = torch.cos(0.3 * rate[replica] * steps[:, None] + phase[replica]) * torch.exp(-steps[:, None] / longest)
    frames = frames + 0.05 * torch.randn(frames.shape, generator=gen)
    return frames.to(device=device, dtype=dtype), steps.to(device), offsets.to(device)


def next_frame_loss(model, frames, steps, offsets):
    """Mean squared error of the prediction after every frame but the replicas' last ones."""
    predicted = model(frames, steps, offsets).float()
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
    model = FrameModel(4, device="cuda", dtype=dtype, max_steps=max(10_000, args.longest))
    log = made_up_log(args.replicas, args.longest, 4, dtype=dtype)
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3)
    for i in range(args.steps):
        optimizer.zero_grad()
        loss = next_frame_loss(model, *log)
        loss.backward()
        optimizer.step()
        if i in (0, args.steps - 1):
            print(f"training step {i + 1}: loss {float(loss.detach()):.4f}")
    cache = model.new_cache(args.replicas, args.longest)
    frame = log[0][log[2][:-1]]
    for i in range(10):
        frame = model.step(frame, torch.full((args.replicas,), i, device="cuda"), cache)
    print(f"ten frames of {args.replicas} replicas rolled out; the first replica's last: "
          f"{[round(float(v), 3) for v in frame[0]]}")


if __name__ == "__main__":
    main()
