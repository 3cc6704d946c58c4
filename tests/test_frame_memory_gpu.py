"""The example model with states: packed histories, chunks, single steps and plain torch operations agree, and so do the
gradients (GPU)."""
import importlib.util
import sys

import pytest
import torch

from conftest import ROOT

gpu = pytest.mark.gpu


def load():
    spec = importlib.util.spec_from_file_location("frame_memory", ROOT / "examples" / "frame_memory.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def log(example, replicas, longest):
    frames, _, offsets = sys.modules[example.made_up_log.__module__].made_up_log(replicas, longest, 4)
    return frames, offsets


def plain_forward(model, wide, frames, offsets):
    """The model with elementary operations of the parameters ``wide``, a replica at a time."""
    decay = model.log_decay.double()
    out = []
    for a, b in zip(offsets.tolist(), offsets.tolist()[1:]):
        x = frames[a:b].double() @ wide["embed.weight"].T + wide["embed.bias"]
        at = torch.arange(b - a, device=x.device, dtype=torch.float64)
        gap = at[:, None] - at
        weight = torch.where(gap >= 0, (gap.clamp(min=0) * decay[:, None, None]).exp(), 0.0)
        for i, block in enumerate(model.blocks):
            w = {n.split(".", 2)[2]: p for n, p in wide.items() if n.startswith(f"blocks.{i}.")}

            def unit(y, by, least=1e-6):
                return y / (y.square().mean(-1, keepdim=True) + least).sqrt() * by

            h = torch.nn.functional.layer_norm(x, x.shape[-1:], w["norm_in.weight"], w["norm_in.bias"])
            q, k, v = (h @ w["qkv.weight"].T).unflatten(1, (-1, block.dim)).split(block.heads, 1)
            q, k = unit(q, w["q_weight"]), unit(k, w["k_weight"])
            read = torch.einsum("hts,shd->thd", torch.einsum("thd,shd->hts", q, k) * weight, v) * block.dim ** -0.5
            x = x + unit(read, w["o_weight"], 0.1).flatten(1) @ w["out.weight"].T
            h = torch.nn.functional.layer_norm(x, x.shape[-1:], w["norm_feed.weight"], w["norm_feed.bias"])
            gate = h @ w["gate.weight"].T
            x = x + (gate * torch.sigmoid(gate) * (h @ w["up.weight"].T)) @ w["down.weight"].T
        out.append(x @ wide["read.weight"].T + wide["read.bias"])
    return torch.cat(out)


@gpu
def test_histories_chunks_and_steps_agree(cuda):
    """float32: two layers of a few hundred FP32 roundings each, of values of size one, stay below 1e-4."""
    example = load()
    torch.manual_seed(1)
    model = example.MemoryModel(4, device="cuda")
    frames, offsets = log(example, 6, 300)
    with torch.no_grad():
        whole, last = model(frames, offsets, return_states=True)
        want = plain_forward(model, {n: p.double() for n, p in model.named_parameters()}, frames, offsets)
        assert float((whole.double() - want).abs().max()) <= 1e-4
        shortest, states, done = int(offsets.diff().min()), model.new_states(6), 0
        for n in (min(5, shortest), shortest - min(5, shortest)):  # two chunks of every replica, each behind its state
            rows = torch.cat([torch.arange(int(a) + done, int(a) + done + n) for a in offsets[:-1]]).cuda()
            got, states = model(frames[rows], torch.arange(7, device="cuda") * n, states, return_states=True)
            assert float((got.double() - want[rows]).abs().max()) <= 1e-4
            done += n
    fresh = model.new_states(6)
    for i in range(shortest):
        rows = offsets[:-1] + i
        assert float((model.step(frames[rows], fresh).double() - want[rows]).abs().max()) <= 1e-4
    for a, b, c in zip(fresh, states, last):
        assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max())
        assert a.shape == c.shape


@gpu
def test_gradients_agree(cuda):
    """Of every parameter, against 64 bits, to 1e-5 of each gradient's norm. A read's terms are of size 8 (q k / 8 of rows of
    root mean square 1) and it is divided by 0.3 at least, so its roundings count up to 25-fold: some hundred of FP32's steps of
    6e-8 in all."""
    example = load()
    torch.manual_seed(2)
    model = example.MemoryModel(4, device="cuda")
    frames, offsets = log(example, 5, 200)
    g = torch.randn(frames.shape, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    got = torch.autograd.grad(model(frames, offsets), model.parameters(), g)
    wide = {n: p.detach().double().requires_grad_() for n, p in model.named_parameters()}
    want = torch.autograd.grad(plain_forward(model, wide, frames, offsets), wide.values(), g.double())
    for (name, _), x, y in zip(model.named_parameters(), got, want):
        assert float((x.double() - y).norm()) <= 1e-5 * float(y.norm()), name


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_training_and_rolling_out_run(cuda, dtype, capsys):
    example = load()
    example.main(["--dtype", dtype, "--replicas", "5", "--longest", "60", "--steps", "3"])
    assert "rolled out" in capsys.readouterr().out


@gpu
def test_a_captured_step_is_replayed(cuda):
    example = load()
    torch.manual_seed(3)
    model = example.MemoryModel(4, device="cuda", dtype=torch.bfloat16)
    frames = torch.randn(8, 5, 4, device="cuda").bfloat16()
    states, fresh, now = model.new_states(5), model.new_states(5), frames[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model.step(now, states)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.step(now, states)
    for state in states:
        state.zero_()
    for frame in frames:
        now.copy_(frame)
        graph.replay()
        assert torch.equal(out, model.step(frame, fresh))


def test_the_decays_on_the_host():
    model = load().MemoryModel(3, width=16, heads=8, dim=8, hidden=24, layers=1, device="cpu")
    rate = 1 - model.log_decay.double().exp()
    assert bool((rate.diff() < 0).all()) and 0.2 < float(rate[0]) < 0.5 and float(rate[-1]) < 0.01
    assert [s.shape for s in model.new_states(2)] == [(2, 8, 8, 8)]


def test_the_decays_belong_to_the_model():
    """They move with it and are saved with it, and no change of its type rounds them: the operators take them in FP32."""
    def make(heads):
        return load().MemoryModel(3, width=16, heads=heads, dim=8, hidden=24, layers=1, device="cpu")

    model, want = make(8), make(8).log_decay.clone()
    assert "log_decay" not in dict(model.named_parameters())
    for kind in (torch.bfloat16, torch.float64, torch.float32):
        model.to(kind)
        assert model.embed.weight.dtype == kind and torch.equal(model.log_decay, want) and model.log_decay.dtype == torch.float32
    saved = model.state_dict()
    saved["log_decay"] = 0.5 * want
    model.load_state_dict(saved)
    assert torch.equal(model.log_decay, 0.5 * want)
    assert model.to("meta").log_decay.device.type == "meta"
