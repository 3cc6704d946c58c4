"""The example model of logged frames: its packed form, its step form and plain torch operations agree (GPU)."""
import importlib.util

import pytest
import torch

from conftest import ROOT

gpu = pytest.mark.gpu


def load():
    spec = importlib.util.spec_from_file_location("frame_attention", ROOT / "examples" / "frame_attention.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_made_up_log_on_the_host():
    frames, steps, offsets = load().made_up_log(5, 9, 3, device="cpu")
    assert frames.shape == (int(offsets[-1]), 3) and steps.shape == (int(offsets[-1]),)
    assert all(int(steps[a]) == 0 for a in offsets[:-1]) and int(offsets.diff().max()) <= 9


def plain_forward(model, frames, steps, offsets):
    """The model in 64 bits with elementary operations, a replica at a time."""
    wide = {n: p.detach().double() for n, p in model.named_parameters()}
    cos, sin = (t.double() for t in model.table)
    out = []
    for a, b in zip(offsets.tolist(), offsets.tolist()[1:]):
        x = frames[a:b].double() @ wide["embed.weight"].T + wide["embed.bias"]
        c, s = cos[steps[a:b]][:, None], sin[steps[a:b]][:, None]
        for i, block in enumerate(model.blocks):
            w = {n.split(".", 2)[2]: p for n, p in wide.items() if n.startswith(f"blocks.{i}.")}
            h = torch.nn.functional.layer_norm(x, x.shape[-1:], w["norm_in.weight"], w["norm_in.bias"])
            q, k, v = (h @ w["qkv.weight"].T).unflatten(1, (-1, block.dim)).split(block.sizes, 1)

            def turned(y, weight):
                y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight
                one, two = y.chunk(2, -1)
                return torch.cat((one * c - two * s, two * c + one * s), -1)

            q, k = turned(q, w["q_weight"]), turned(k, w["k_weight"])
            k, v = (t.repeat_interleave(q.shape[1] // t.shape[1], 1) for t in (k, v))
            score = torch.einsum("ihd,jhd->hij", q, k) * block.dim ** -0.5
            score = score.masked_fill(torch.ones(b - a, b - a, device=x.device).triu(1).bool(), float("-inf"))
            x = x + torch.einsum("hij,jhd->ihd", score.softmax(-1), v).flatten(1) @ w["out.weight"].T
            h = torch.nn.functional.layer_norm(x, x.shape[-1:], w["norm_mlp.weight"], w["norm_mlp.bias"])
            h = torch.nn.functional.silu(h @ w["mlp.0.weight"].T + w["mlp.0.bias"])
            x = x + h @ w["mlp.2.weight"].T + w["mlp.2.bias"]
        out.append(x @ wide["read.weight"].T + wide["read.bias"])
    return torch.cat(out)


@gpu
def test_packed_steps_and_plain_agree(cuda):
    """float32: two layers of a few hundred FP32 roundings each, of values of size one, stay below 1e-4."""
    example = load()
    torch.manual_seed(1)
    model = example.FrameModel(4, device="cuda")
    frames, steps, offsets = example.made_up_log(6, 150, 4)
    whole = model(frames, steps, offsets).detach()
    want = plain_forward(model, frames, steps, offsets)
    assert float((whole.double() - want).abs().max()) <= 1e-4
    cache = model.new_cache(6, 160)
    shortest = int(offsets.diff().min())
    for i in range(shortest):
        rows = offsets[:-1] + i
        got = model.step(frames[rows], steps[rows], cache)
        assert float((got.double() - want[rows]).abs().max()) <= 1e-4
    assert cache["counts"].tolist() == [shortest] * 6


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_training_lowers_the_loss(cuda, dtype):
    example = load()
    torch.manual_seed(2)
    model = example.FrameModel(4, device="cuda", dtype=getattr(torch, dtype))
    log = example.made_up_log(8, 100, 4, dtype=getattr(torch, dtype))
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3)
    losses = []
    for _ in range(15):
        optimizer.zero_grad()
        loss = example.next_frame_loss(model, *log)
        loss.backward()
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in model.parameters())
        optimizer.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < 0.7 * losses[0]


def plain_operators(example, monkeypatch):
    """Stand-ins on the host for the two operators of the step form (queries and keys as they are, plain attention)."""

    def attend(q, k, v, offsets, key_offsets, key_counts, causal):
        out = []
        for b in range(q.shape[0]):
            at = slice(int(key_offsets[b]), int(key_offsets[b] + key_counts[b]))
            x, y = (t[at].repeat_interleave(q.shape[1] // k.shape[1], 1) for t in (k, v))
            weight = torch.softmax(torch.einsum("hd,jhd->hj", q[b], x) * q.shape[2] ** -0.5, 1)
            out.append(torch.einsum("hj,jhd->hd", weight, y))
        return torch.stack(out)

    monkeypatch.setattr(example, "packed_attention", attend)
    monkeypatch.setattr(example, "head_norm_rotary", lambda q, k, *rest: (q, k))


def test_a_full_cache_keeps_the_last_frames_on_the_host(monkeypatch):
    """More frames than a slot holds: the oldest make room, in their own slot, and the prediction is that of a fresh
    cache that has read the last ones alone."""
    example = load()
    plain_operators(example, monkeypatch)
    torch.manual_seed(3)
    model = example.FrameModel(3, width=16, heads=2, key_heads=1, dim=8, layers=1, device="cpu")
    frames, at = torch.randn(7, 2, 3), torch.arange(7)[:, None].expand(7, 2)
    cache = model.new_cache(2, 4)
    for i in range(7):
        got = model.step(frames[i], at[i], cache)
    assert cache["counts"].tolist() == [4, 4]
    fresh = model.new_cache(2, 4)
    for i in range(3, 7):
        want = model.step(frames[i], at[i], fresh)
    # one layer: what is kept of a frame does not depend on the frames before it; sums of four terms in another order
    assert torch.allclose(got, want, atol=1e-5)


def test_a_cache_without_room_is_refused_on_the_host():
    with pytest.raises(ValueError):
        load().FrameModel(3, width=16, heads=2, key_heads=1, dim=8, layers=1, device="cpu").new_cache(2, 0)


def test_the_table_covers_the_longest_history_on_the_host(monkeypatch):
    """A position outside the table would be flagged and its row not turned."""
    example = load()

    class Seen(Exception):
        pass

    def record(*args, max_steps=10_000, **kwargs):
        raise Seen(max_steps)

    monkeypatch.setattr(example, "FrameModel", record)
    for longest in (500, 10_001, 20_000):
        with pytest.raises(Seen) as seen:
            example.main(["--longest", str(longest)])
        assert seen.value.args[0] >= longest
