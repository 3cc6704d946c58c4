"""Packed attention and its gradients against the formulas in 64 bits (GPU), and the refusals.

The bounds follow the roundings: u = half the distance of neighbouring values of the stored type (2^-24 or 2^-8
relative), t = the rounding of the weights p and their gradients for the products (2^-8 in 16 bits, none in 32), and
e = the error of a score in FP32, at most (dim + 4) 2^-24 sum |q||k| scale, with that of exp2 and of the row sum."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from fastmd_b200 import _lib
from fastmd_b200.packed_attention import packed_attention

gpu = pytest.mark.gpu
F32, B16 = torch.float32, torch.bfloat16
E32 = 2.0 ** -24


def reference(q, k, v, offsets, key_offsets, counts, causal, scale, g=None, glse=None):
    """Outputs, gradients and the error bound of each, in 64 bits, a sequence and a head at a time."""
    unit = E32 if q.dtype == F32 else 2.0 ** -8
    split = 0.0 if q.dtype == F32 else 2.0 ** -8
    dim, group = q.shape[2], q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    out = {n: torch.zeros_like(t) for n, t in dict(out=q, dq=q, dk=k, dv=v).items()}
    err = {n: torch.zeros_like(t) for n, t in out.items()}
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    lse_err = torch.zeros_like(lse)
    for b in range(len(offsets) - 1):
        r = slice(offsets[b], offsets[b + 1])
        n = counts[b] if counts is not None else key_offsets[b + 1] - key_offsets[b]
        c = slice(key_offsets[b], key_offsets[b] + n)
        m = r.stop - r.start
        if m == 0 or n == 0:
            continue
        seen = torch.ones(m, n, dtype=torch.bool, device=q.device)
        if causal:
            seen = torch.arange(n, device=q.device) <= torch.arange(m, device=q.device)[:, None] + n - m
        for h in range(q.shape[1]):
            x, y, z = q[r, h], k[c, h // group], v[c, h // group]
            s = torch.where(seen, scale * (x @ y.T), -math.inf)
            top = s.amax(1, keepdim=True).nan_to_num(neginf=0.0)
            p = torch.exp(s - top)
            l = p.sum(1, keepdim=True)
            lse[r, h] = (top + l.log())[:, 0]
            p = p / l.clamp(min=1e-300)
            # a score's error, the rounding of its difference to the maximum, exp2's (2^-22) and the row sum's
            e = E32 * ((dim + 4) * scale * (x.abs() @ y.abs().T) + 4 * s.abs().nan_to_num(posinf=0.0) + 8)
            e = e + (e * p).sum(1, keepdim=True) + E32 * (4 + n / 16)
            o = p @ z
            out["out"][r, h] = o
            err["out"][r, h] = unit * o.abs() + (p * (split + e)) @ z.abs() + E32 * (n / 16) * (p @ z.abs())
            lse_err[r, h] = (e * p).sum(1) + E32 * (4 + n / 16 + 4 * lse[r, h].abs().nan_to_num(posinf=0.0))
            if g is None:
                continue
            w = g[r, h].double()
            dp = w @ z.T
            dp_err = E32 * (dim + 4) * (w.abs() @ z.abs().T)
            delta = (w * o).sum(1, keepdim=True)
            delta_err = (w.abs() * err["out"][r, h]).sum(1, keepdim=True) + E32 * dim * (w * o).abs().sum(1, keepdim=True)
            if glse is not None:
                delta = delta - glse[r, h, None].double()
            ds = p * (dp - delta)
            # a backward weight is exp(s - lse): the errors of both
            we = e + lse_err[r, h, None]
            ds_err = ds.abs() * (split + we) + p * (dp_err + delta_err + 4 * E32 * (dp.abs() + delta.abs()))
            out["dv"][c, h // group] += p.T @ w
            err["dv"][c, h // group] += (p * (split + we)).T @ w.abs() + E32 * (m / 16) * (p.T @ w.abs())
            out["dq"][r, h] = scale * (ds @ y)
            err["dq"][r, h] = scale * ((ds_err + E32 * (n / 16) * ds.abs()) @ y.abs())
            out["dk"][c, h // group] += scale * (ds.T @ x)
            err["dk"][c, h // group] += scale * ((ds_err + E32 * (m / 16) * ds.abs()).T @ x.abs())
    for n in ("dq", "dk", "dv"):
        err[n] += unit * (out[n].abs() + err[n])
    return out, err, lse, lse_err


def check(got, want, err, what):
    got = got.double()
    assert bool(torch.isfinite(got).all()), what
    over = ((got - want).abs() - err - 1e-30).amax() if got.numel() else torch.tensor(0.0)
    ratio = ((got - want).abs() / (err + 1e-30)).amax() if got.numel() else torch.tensor(0.0)
    assert float(over) <= 0, f"{what}: {float(ratio):.3g} times its bound"


def starts(sizes):
    return [sum(sizes[:i]) for i in range(len(sizes) + 1)]


def make(rows, slots, hq, hk, dim, dtype, seed=0, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    q = (torch.randn(sum(rows), hq, dim, generator=gen) * spread).to(dtype).cuda()
    k, v = (torch.randn(sum(slots), hk, dim, generator=gen).to(dtype).cuda() for _ in range(2))
    g = torch.randn(q.shape, generator=gen).to(dtype).cuda()
    return q, k, v, g


def on_device(values):
    return torch.tensor(values, dtype=torch.int64, device="cuda")


def run_case(rows, slots, counts, hq, hk, dim, dtype, causal, seed=0, spread=1.0, lse_grad=False):
    q, k, v, g = make(rows, slots, hq, hk, dim, dtype, seed, spread)
    ro, ko = starts(rows), starts(slots)
    if counts is not None:  # what lies behind a count is never used
        for b, n in enumerate(counts):
            k[ko[b] + n:ko[b + 1]] = float("nan")
            v[ko[b] + n:ko[b + 1]] = float("inf")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    scale = dim ** -0.5
    out, lse = packed_attention(q, k, v, on_device(ro), on_device(ko), None if counts is None else on_device(counts),
                                causal=causal, return_lse=True)
    glse = torch.randn(lse.shape, generator=torch.Generator().manual_seed(9)).cuda() if lse_grad else None
    grads = torch.autograd.grad((out, lse) if lse_grad else out, leaves, (g, glse) if lse_grad else g)
    alone = packed_attention(q.detach(), k.detach(), v.detach(), on_device(ro), on_device(ko),
                             None if counts is None else on_device(counts), causal=causal)
    clean = [torch.nan_to_num(t.detach(), 0.0, 0.0, 0.0) if counts is not None else t.detach() for t in (k, v)]
    want, err, want_lse, lse_err = reference(q.detach(), *clean, ro, ko, counts, causal, scale, g, glse)
    check(out.detach(), want["out"], err["out"], "out")
    check(alone, want["out"], err["out"], "out without gradients")
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), empty)
    check(lse.detach().masked_fill(empty, 0.0), want_lse.masked_fill(empty, 0.0), lse_err, "lse")
    for name, got in zip(("dq", "dk", "dv"), grads):
        check(got, want[name], err[name], name)


SEQUENCES = {
    "one": ([1], [1], None),
    "atoms": ([135, 135, 135], [135, 135, 135], None),
    "edges": ([127, 128, 129, 1, 0, 255], [127, 128, 129, 1, 0, 255], None),
    "cross": ([5, 64, 0, 3, 200], [300, 65, 17, 0, 131], None),
    "more_rows": ([200, 70], [90, 70], None),  # with causal the first 110 rows see nothing
    "step": ([1, 1, 1, 1], [400, 400, 400, 400], [400, 1, 129, 0]),
    "chunk": ([33, 33, 7], [700, 700, 700], [700, 40, 260]),
    "long": ([1100], [1100], None),
}


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("name", list(SEQUENCES))
def test_sequences(cuda, name, causal, dtype):
    rows, slots, counts = SEQUENCES[name]
    run_case(rows, slots, counts, 4, 2, 64, dtype, causal)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("hq,hk,dim", [(1, 1, 8), (3, 1, 32), (8, 1, 128), (5, 5, 96), (6, 2, 72), (16, 4, 40),
                                       (64, 1, 16), (24, 2, 128), (2, 2, 120)])
def test_heads_and_sizes(cuda, hq, hk, dim, dtype):
    run_case([70, 1, 190], [70, 1, 190], None, hq, hk, dim, dtype, True, seed=hq + dim)
    run_case([2, 1], [150, 333], [150, 201], hq, hk, dim, dtype, True, seed=hq + dim, lse_grad=True)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_large_scores(cuda, dtype):
    """Scores of some hundreds: the running maximum moves by far more than a weight's range."""
    run_case([300, 40], [300, 40], None, 2, 1, 64, dtype, False, spread=60.0)
    run_case([1, 3], [900, 257], None, 4, 2, 64, dtype, False, spread=60.0)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_layouts_are_the_packed_ones(cuda, dtype):
    """Views of a fused projection, a head-major tensor and an unaligned base give the packed tensor's bits."""
    rows, hq, hk, dim = 150, 4, 2, 64
    gen = torch.Generator().manual_seed(5)
    fused = torch.randn(rows, hq + 2 * hk, dim, generator=gen).to(dtype).cuda()
    parts = fused.split((hq, hk, hk), 1)
    offsets = on_device([0, 100, 150])
    want = packed_attention(*[p.contiguous() for p in parts], offsets, causal=True)
    assert torch.equal(packed_attention(*parts, offsets, causal=True), want)
    turned = [p.transpose(0, 1).contiguous().transpose(0, 1) for p in parts]
    assert torch.equal(packed_attention(*turned, offsets, causal=True), want)
    columns = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in parts]
    assert torch.equal(packed_attention(*columns, offsets, causal=True), want)
    odd = torch.empty(rows * hq * dim + 1, dtype=dtype, device="cuda")
    odd[1:] = parts[0].reshape(-1)
    assert torch.equal(packed_attention(odd[1:].view(rows, hq, dim), *parts[1:], offsets, causal=True), want)
    leaves = [p.detach().requires_grad_() for p in parts]
    out = packed_attention(*leaves, offsets, causal=True)
    spread_grad = torch.autograd.grad(out.sum(), leaves)  # an expanded gradient of stride 0
    out = packed_attention(*leaves, offsets, causal=True)
    full_grad = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert all(torch.equal(a, b) for a, b in zip(spread_grad, full_grad))


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_neighbours_do_not_matter(cuda, dtype):
    """A sequence's bits are its own: the others may hold NaN and infinities, and more of them may follow."""
    rows = [130, 77, 45]
    q, k, v, g = make(rows, rows, 4, 2, 64, dtype, seed=3)
    ro = starts(rows)

    def whole(q, k, v, g):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = packed_attention(*leaves, on_device(ro), causal=False)
        return out.detach(), *torch.autograd.grad(out, leaves, g)

    want = whole(q, k, v, g)
    for t, bad in ((q, "nan"), (k, "inf"), (v, "nan"), (g, "inf")):
        t[:130] = float(bad)
        t[207:] = float(bad)
    got = whole(q, k, v, g)
    for a, b in zip(got, want):
        assert torch.equal(a[130:207], b[130:207])


@gpu
def test_non_finite_values_stay_visible(cuda):
    """A row with a NaN query is NaN; the rows of other heads and tokens are not touched by it."""
    q, k, v, _ = make([40], [40], 2, 2, 32, F32)
    want = packed_attention(q, k, v, on_device([0, 40]))
    q[7, 1] = float("nan")
    got = packed_attention(q, k, v, on_device([0, 40]))
    assert bool(torch.isnan(got[7, 1]).all())
    q[7, 1], got[7, 1], want[7, 1] = 0, 0, 0
    assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_repeatable(cuda, dtype):
    rows = [700, 3, 512]
    q, k, v, g = make(rows, rows, 8, 2, 64, dtype)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    runs = []
    for _ in range(2):
        out = packed_attention(*leaves, on_device(starts(rows)), causal=True)
        runs.append([out.detach(), *torch.autograd.grad(out, leaves, g)])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@gpu
def test_gradient_against_differences(cuda):
    """Directional derivatives of sum(out c) + sum(lse d) by central differences of the FP32 operator: a step of
    2^-6 leaves a truncation near h^2 and a rounding near 2^-24 / h of the sum of the terms' sizes."""
    rows = [9, 5]
    q, k, v, c = make(rows, rows, 2, 1, 16, F32, seed=11)
    gen = torch.Generator().manual_seed(12)
    d = torch.randn(14, 2, generator=gen).cuda()
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    offsets, h = on_device(starts(rows)), 2.0 ** -6

    def value(args):
        out, lse = packed_attention(*args, offsets, causal=True, return_lse=True)
        return (out * c).double().sum() + (lse * d).double().sum()

    grads = torch.autograd.grad(value(leaves), leaves)
    for i in range(3):
        step = torch.randn(leaves[i].shape, generator=gen).cuda()
        up, down = ([t.detach() + sign * h * step if j == i else t.detach() for j, t in enumerate(leaves)]
                    for sign in (1, -1))
        slope = float(value(up) - value(down)) / (2 * h)
        size = float((grads[i].abs() * step.abs()).sum())
        assert abs(slope - float((grads[i] * step).double().sum())) <= 2.0 ** -9 * size


@gpu
def test_only_what_is_asked_for(cuda):
    q, k, v, g = make([50], [50], 2, 1, 32, B16)
    offsets = on_device([0, 50])
    both = [t.clone().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(packed_attention(*both, offsets), both, g)
    alone = q.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(packed_attention(alone, k, v, offsets), alone, g)[0], want[0])
    alone = v.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(packed_attention(q, k, alone, offsets), alone, g)[0], want[2])
    lse_only = q.clone().requires_grad_()
    _, lse = packed_attention(lse_only, k, v, offsets, return_lse=True)
    (dq,) = torch.autograd.grad(lse.sum(), lse_only)  # the gradient of lse alone: the mean key
    p = torch.softmax(32 ** -0.5 * torch.einsum("thd,sd->ths", q.double(), k[:, 0].double()), -1)
    want = 32 ** -0.5 * torch.einsum("ths,sd->thd", p, k[:, 0].double())
    assert float((dq.double() - want).abs().max()) <= 2.0 ** -6 * float(want.abs().max())


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("scale", [0.0, 0.7])
def test_scale(cuda, scale, dtype):
    """A scale of its own; 0 takes the mean of the values."""
    q, k, v, _ = make([150], [150], 2, 1, 64, dtype)
    got = packed_attention(q, k, v, on_device([0, 150]), scale=scale)
    want, err, _, _ = reference(q, k, v, [0, 150], [0, 150], None, False, scale)
    check(got, want["out"], err["out"], "out")


@gpu
@pytest.mark.parametrize("dtype,dim", [(F32, 64), (F32, 128), (B16, 64)], ids=["f32", "f32_wide", "b16"])
def test_scale_of_zero_gradients(cuda, dtype, dim):
    """Scores that do not count: queries and keys get nothing, each value the mean of the gradients. The tail of a tile
    is masked, so a masked score times 0 would show."""
    q, k, v, g = make([150], [150], 2, 1, dim, dtype)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out = packed_attention(*leaves, on_device([0, 150]), scale=0.0)
    out.backward(g)
    assert float(leaves[0].grad.abs().max()) < 1e-30 and float(leaves[1].grad.abs().max()) < 1e-30
    want = g.double().sum((0, 1)) / 150
    # 300 rounded products a sum, and the rounding of 1/150 and of the result
    unit = 2.0 ** -8 if dtype == B16 else 2.0 ** -20
    err = 2 * unit * g.double().abs().sum((0, 1)) / 150
    assert bool(((leaves[2].grad.double() - want).abs() <= err).all())


@gpu
def test_captured_in_a_graph(cuda):
    """A captured call reads offsets and counts when it is replayed."""
    q, k, v, _ = make([1, 1], [300, 300], 4, 2, 64, B16)
    counts = on_device([10, 300])
    args = (q, k, v, on_device([0, 1, 2]), on_device([0, 300, 600]), counts)
    packed_attention(*args, causal=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = packed_attention(*args, causal=True)
    for n in ([10, 300], [299, 1], [0, 150]):
        counts.copy_(on_device(n))
        graph.replay()
        assert torch.equal(out, packed_attention(*args, causal=True))


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_gradients_captured_in_a_graph(cuda, dtype):
    """Forward and backward in one graph: replays give the eager pass's bits for new values."""
    rows = [200, 1, 90]
    q, k, v, g = make(rows, rows, 4, 2, 64, dtype)
    leaves, offsets = [t.requires_grad_() for t in (q, k, v)], on_device(starts(rows))

    def step():
        out = packed_attention(*leaves, offsets, causal=True)
        return out.detach(), *torch.autograd.grad(out, leaves, g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (21, 22):
        with torch.no_grad():
            for t, new in zip((*leaves, g), make(rows, rows, 4, 2, 64, dtype, seed)):
                t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step()))


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
def test_many_sequences(cuda, causal, dtype):
    """More sequences than a warp ranks, empty ones and single rows among them."""
    rows = [(37 * b * b + 11 * b) % 150 if b % 7 else b % 2 for b in range(75)]
    run_case(rows, rows, None, 4, 2, 32, dtype, causal)


@gpu
def test_a_cache_past_32_bits(cuda):
    """Slots whose values lie more than 2^32 bytes and 2^31 elements into the cache are read as those of a small one."""
    rows, dim, slot = 20_000_000, 128, 300
    gen = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.empty(rows, 1, dim, dtype=B16, device="cuda") for _ in range(2))
    ends = [torch.randn(slot, 1, dim, generator=gen, device="cuda").to(B16) for _ in range(2)]
    k[-slot:], v[-slot:] = ends
    k[:50], v[:50] = ends[0][:50], ends[1][:50]
    q = torch.randn(2, 4, dim, generator=gen, device="cuda").to(B16)
    got = packed_attention(q, k, v, on_device([0, 1, 2]), on_device([0, rows - slot, rows]), on_device([50, 277]))
    small = [torch.cat((e[:50], e)) for e in ends]
    want = packed_attention(q, *small, on_device([0, 1, 2]), on_device([0, 50, 50 + slot]), on_device([50, 277]))
    # another number of splits: the roundings of the sums differ, not the values
    assert float((got.double() - want.double()).abs().max()) <= 2.0 ** -7 * float(want.abs().max())


@gpu
def test_another_stream(cuda):
    q, k, v, _ = make([100], [100], 2, 2, 64, B16)
    offsets = on_device([0, 100])
    want = packed_attention(q, k, v, offsets)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = packed_attention(q, k, v, offsets)
    side.synchronize()
    assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_bad_offsets_are_flagged(cuda, dtype):
    """Offsets and counts that leave the arrays are held inside and flagged."""
    q, k, v, _ = make([60], [60], 2, 2, 32, dtype)
    word = _lib.flags_word(q.device)
    good = on_device([0, 30, 60])
    for offsets, key_offsets, counts in ((on_device([0, 30, 70]), good, None), (on_device([0, -5, 60]), good, None),
                                         (good, on_device([0, 90, 60]), None), (good, good, on_device([31, 30])),
                                         (good, good, on_device([-1, 30])), (on_device([3, 30, 60]), good, None),
                                         (good, on_device([0, 30, 50]), None)):
        word.zero_()
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = packed_attention(*leaves, offsets, key_offsets, counts)
        torch.autograd.grad(out.sum(), leaves)
        assert int(word.item()) & 1
    word.zero_()
    packed_attention(q, k, v, good)
    assert int(word.item()) == 0


@gpu
def test_empty(cuda):
    q, k, v, _ = make([0], [0], 2, 1, 32, B16)
    assert packed_attention(q, k, v, on_device([0])).shape == (0, 2, 32)
    assert packed_attention(q, k, v, on_device([0, 0, 0])).shape == (0, 2, 32)
    q, k, v, _ = make([0], [40], 2, 1, 32, B16)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = packed_attention(*leaves, on_device([0, 0]), on_device([0, 40]))
    grads = torch.autograd.grad(out.sum(), leaves)
    assert not grads[1].any() and not grads[2].any()
    q, k, v, _ = make([40], [0], 2, 1, 32, F32)
    out, lse = packed_attention(q, k, v, on_device([0, 40]), on_device([0, 0]), return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())


@gpu
def test_refusals(cuda):
    q, k, v, _ = make([6], [6], 4, 2, 32, F32)
    offsets = on_device([0, 6])
    with pytest.raises(_lib.FastMDLibraryError):
        packed_attention(q, k.cpu(), v, offsets)
    for bad in (dict(q=q.half(), k=k.half(), v=v.half()), dict(k=k.bfloat16()), dict(v=v[:5]), dict(q=q[0]),
                dict(q=q[..., :12], k=k[..., :12], v=v[..., :12]), dict(q=q[:, :3]), dict(offsets=offsets.int()),
                dict(offsets=offsets[None]), dict(q=q[:5]), dict(offsets=offsets[:1]),
                dict(key_offsets=on_device([0, 3, 6])), dict(key_counts=on_device([3, 3])),
                dict(q=q.repeat(1, 33, 1)), dict(scale=-0.1), dict(scale=float("nan")), dict(scale=float("inf"))):
        with pytest.raises(ValueError):
            packed_attention(**(dict(q=q, k=k, v=v, offsets=offsets) | bad))


def test_abi_refuses_on_the_host():
    lib = _lib.lib()
    base = dict(q=1 << 20, k=1 << 20, v=1 << 20, offsets=1 << 20, key_offsets=1 << 20, key_counts=None, rows=0, keys=0,
                q_row=64, q_head=64, k_row=64, k_head=64, v_row=64, v_head=64, scale=0.125, type=1, batch=1, heads=1,
                key_heads=1, dim=64, causal=0)
    assert lib.fmd_packed_attention(_lib.FmdAttention(**base), None, None, None, 0, None, None) == 0  # no rows
    for bad in (dict(type=2), dict(heads=3, key_heads=2), dict(key_heads=0), dict(dim=12), dict(dim=136),
                dict(rows=-1), dict(batch=0, rows=1), dict(rows=1, q=None), dict(keys=1, v=None),
                dict(offsets=None), dict(heads=65), dict(scale=-1.0), dict(scale=math.nan)):
        assert lib.fmd_packed_attention(_lib.FmdAttention(**(base | bad)), None, None, None, 0, None, None) == 1
    for bad in (dict(rows=1, q=(1 << 20) + 2), dict(keys=1, k_row=65), dict(rows=1, q_head=4), dict(rows=1 << 40)):
        assert lib.fmd_packed_attention(_lib.FmdAttention(**(base | bad)), 1 << 20, None, None, 0, None, None) == 3
    assert lib.fmd_packed_attention(_lib.FmdAttention(**(base | dict(rows=1))), None, None, None, 0, None, None) == 1


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_a_second_derivative_is_refused(cuda, dtype):
    """Gradients taken with create_graph are first derivatives: to differentiate them raises and drops no term, with a
    gradient that depends on the inputs and with one that does not. Where nothing is differentiated again they are the
    same."""
    q, k, v, g = make([30], [30], 2, 1, 32, dtype)
    leaves, offsets = [t.requires_grad_() for t in (q, k, v)], on_device([0, 30])
    out, lse = packed_attention(*leaves, offsets, return_lse=True)
    once = torch.autograd.grad(out, leaves, g, retain_graph=True)
    again = torch.autograd.grad(out, leaves, g, create_graph=True, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(once, again))
    for i in range(3):
        with pytest.raises(RuntimeError, match="first derivatives"):
            torch.autograd.grad(again[i].sum() + leaves[0].square().sum(), leaves[0], retain_graph=True)
    (dq,) = torch.autograd.grad(lse.square().sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match="first derivatives"):
        (dq.square().sum() + leaves[0].square().sum()).backward()


@gpu
def test_forward_mode_is_refused(cuda):
    """A tangent on any of the three raises: it is not passed by."""
    args, offsets = make([20], [20], 2, 1, 32, F32)[:3], on_device([0, 20])
    with forward_ad.dual_level():
        for i in range(3):
            dual = list(args)
            dual[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError):
                packed_attention(*dual, offsets)
            with torch.no_grad(), pytest.raises(RuntimeError):
                packed_attention(*dual, offsets, return_lse=True)
        packed_attention(*args, offsets)


@gpu
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_values_at_the_end_of_float32(cuda, dim):
    """Finite values whose nearest bfloat16 is an infinity. A row of one key returns its value: a weight of 1 and, in
    planes, three exact products of it, which the sum may cut below 2^-22 each. Keys of zero score zero whatever the
    query holds: the mean of the values."""
    top = torch.finfo(F32).max
    q, k, v, _ = make([3], [3], 2, 1, dim, F32)
    v[:, :, 0], v[:, :, 1], v[:, :, 2] = top, -top, 3.3961775e38
    one = on_device([0, 1, 2, 3])  # three sequences of a row
    got = packed_attention(q, k, v, one)
    want = v.double().expand(3, 2, dim)
    assert bool(((got.double() - want).abs() <= 2.0 ** -20 * want.abs()).all())
    q, k, v, _ = make([3], [3], 2, 1, dim, F32)
    q[:, :, 0], q[:, :, 1], k[:] = top, -top, 0.0
    got = packed_attention(q, k, v, on_device([0, 3]))
    want = v.double().mean(0, keepdim=True).expand(3, 2, dim)
    assert bool(((got.double() - want).abs() <= 2.0 ** -20 * v.double().abs().amax(0)).all())


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_infinite_values_stay_not_finite(cuda, dim):
    """An infinite value leaves no finite number in its column of the rows that see it, and the other columns and the
    rows of other key heads as they are."""
    q, k, v, _ = make([40], [40], 4, 2, dim, F32)
    want = packed_attention(q, k, v, on_device([0, 40]))
    v[7, 1, 5] = float("inf")
    got = packed_attention(q, k, v, on_device([0, 40]))
    assert not bool(torch.isfinite(got[:, 2:, 5]).any())
    got[:, 2:, 5] = want[:, 2:, 5]
    assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("dtype,dim", [(F32, 32), (F32, 96), (B16, 32)], ids=["f32", "f32_wide", "b16"])
def test_offsets_that_fall_among_many_are_flagged(cuda, dtype, dim):
    """Forty sequences: one offset far ahead of its neighbours, whose sequence no tile's search ends at."""
    q, k, v, _ = make([2000], [2000], 1, 1, dim, dtype)
    good = torch.arange(41) * 50
    bad = good.clone()
    bad[5] = 1900
    word = _lib.flags_word(q.device)
    word.zero_()
    packed_attention(q, k, v, good.cuda())
    assert int(word.item()) == 0
    packed_attention(q, k, v, bad.cuda(), good.cuda())
    assert int(word.item()) & 1
    word.zero_()
    packed_attention(q, k, v, good.cuda(), bad.cuda())
    assert int(word.item()) & 1
    leaf = q.clone().requires_grad_()
    out = packed_attention(leaf, k, v, bad.cuda(), good.cuda())
    word.zero_()
    torch.autograd.grad(out.sum(), leaf)  # the backward pass by itself
    assert int(word.item()) & 1
    word.zero_()


def takes_two_tiles(rows, slots, hq, hk):
    """The rule of the forward pass in 16 bits for heads of more than 64 values: two tiles of rows a block."""
    blocks = (sum(rows) // (2 * (128 // (hq // hk))) + len(rows)) * hk
    return blocks >= 148 and sum(slots) // len(rows) >= 1024


@gpu
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("rows,slots,counts,hq,hk,dim", [
    ([2100, 1301], [2100, 1301], None, 16, 8, 64),  # last tiles of 52 and 21 rows; blocks without a second tile
    ([2100, 1301], [2100, 1301], None, 12, 12, 128),
    ([2100, 1301], [2100, 1301], None, 24, 8, 32),  # 42 tokens of three heads: rows of a tile that hold nothing
    ([1000, 1500], [1700, 1033], None, 30, 5, 96),  # 21 tokens of six heads; more keys than rows and the reverse
    ([1430, 1300], [1100, 1030], None, 16, 8, 72),  # causal: 330 rows see nothing, a first tile among them
    ([700, 1300, 0, 1], [1500, 1300, 1400, 1200], [1333, 1300, 5, 0], 32, 4, 64),
    ([1153] * 30, [1153] * 30, None, 2, 2, 40),
    ([2100, 1301], [2100, 1301], None, 24, 8, 72),
    ([2100, 1301], [2100, 1301], None, 16, 8, 120),
    ([700, 1300, 0, 1], [1500, 1300, 1400, 1200], [1333, 1300, 5, 0], 32, 4, 128),
    ([1153] * 30, [1153] * 30, None, 2, 2, 96),
    ([1040 + b % 5 for b in range(40)], [1040 + b % 5 for b in range(40)], None, 2, 1, 128),
], ids=["pairs", "single", "three", "six", "more_rows", "cache", "thirty", "three_wide", "pairs_wide",
        "cache_wide", "thirty_wide", "forty"])
def test_two_tiles_a_block(cuda, rows, slots, counts, hq, hk, dim, causal):
    """Long sequences in 16 bits: the tiles of a block share their keys and may see different numbers of them."""
    assert takes_two_tiles(rows, slots, hq, hk)
    run_case(rows, slots, counts, hq, hk, dim, B16, causal, seed=dim)


@gpu
@pytest.mark.parametrize("batch,slot,hq,hk,dim", [(64, 2000, 8, 2, 64), (3, 40_000, 32, 4, 64), (64, 1500, 4, 4, 32)])
def test_rows_against_long_caches_in_float32(cuda, batch, slot, hq, hk, dim):
    """Keys and values that come from memory late (caches larger than L2, read by all blocks at once): no wait runs out,
    in many passes, and all have the same bits."""
    gen = torch.Generator(device="cuda").manual_seed(batch)
    q, k, v = (torch.randn(n, h, dim, generator=gen, device="cuda") for n, h in ((batch, hq), (batch * slot, hk),
                                                                               (batch * slot, hk)))
    rows, keys = list(range(batch + 1)), starts([slot] * batch)
    args = (q, k, v, on_device(rows), on_device(keys), on_device([slot] * batch))
    word = _lib.flags_word(q.device)
    word.zero_()
    first = packed_attention(*args, causal=True)
    others = torch.empty(2 ** 26, device="cuda")
    for _ in range(20):
        others.zero_()  # 256 MB: the caches leave L2
        assert torch.equal(packed_attention(*args, causal=True), first)
    assert int(word.item()) == 0
    want, err, _, _ = reference(q, k, v, rows, keys, None, True, dim ** -0.5)
    check(first, want["out"], err["out"], "out")


@gpu
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("rows,hq,hk,dim", [([1, 2, 3] * 20, 2, 2, 32), ([2, 8] * 10, 8, 2, 64), ([11, 33, 5], 3, 1, 96),
                                            ([16, 17, 15], 4, 4, 128), ([88, 4], 16, 4, 72)])
def test_gradients_of_few_keys_in_16_bits(cuda, rows, hq, hk, dim, causal):
    """The gradients of q and k lose little beyond the rounding of the result where rows see few keys, though ds cancels
    most there: delta's error (from the stored output's two roundings) would reach them as n^-1/2 of that rounding for n
    keys, at 17 keys 0.35 with the average of g and v. The two planes of ds add 2^-16, FP32 sums less: 1.3 in all."""
    q, k, v, g = make(rows, rows, hq, hk, dim, B16, seed=dim, spread=1.2)
    leaves, ro = [t.requires_grad_() for t in (q, k, v)], starts(rows)
    out = packed_attention(*leaves, on_device(ro), causal=causal)
    grads = torch.autograd.grad(out, leaves, g)
    want, _, _, _ = reference(*(t.detach() for t in leaves), ro, ro, None, causal, dim ** -0.5, g)
    for name, got in zip(("dq", "dk"), grads):
        rounding = (want[name].to(B16).double() - want[name]).norm()
        assert float((got.double() - want[name]).norm()) <= 1.3 * float(rounding), name


@gpu
@pytest.mark.parametrize("dim", [64, 72])
def test_sums_over_many_keys_in_float32(cuda, dim):
    """Values near 1 and 4,000 keys in one walk: 4,000 additions in a row would leave 0.29 sqrt(4000 / 3) = 11 units of 2^-24
    (root mean square), the tiles' sums one after the other 1.3 (tiles of 64), as much again in the denominator, and the
    last operations about one each: 5 in all."""
    batch, slot, heads = 64, 4000, 8
    gen = torch.Generator(device="cuda").manual_seed(dim)
    q, k, v = (torch.randn(n, heads, dim, generator=gen, device="cuda") for n in (batch, batch * slot, batch * slot))
    v = 1.0 + 0.1 * v
    got = packed_attention(q, k, v, on_device(list(range(batch + 1))), on_device(starts([slot] * batch)))
    square = 0.0
    for b in range(0, batch, 8):
        x, y = (t[b * slot:(b + 1) * slot].double() for t in (k, v))
        p = torch.softmax(dim ** -0.5 * torch.einsum("hd,jhd->hj", q[b].double(), x), 1)
        want = torch.einsum("hj,jhd->hd", p, y)
        square += float(((got[b].double() - want) / want).square().mean()) / (batch // 8)
    assert math.sqrt(square) <= 5 * E32


@gpu
@pytest.mark.parametrize("dtype,dim", [(F32, 32), (F32, 128), (B16, 64)], ids=["f32", "f32_wide", "b16"])
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
def test_one_key_has_no_gradient_of_its_score(cuda, causal, dtype, dim):
    """The softmax of one score is 1: rows that see one key give nothing to queries and keys, to the bit, and a key that is
    alone gets nothing; with a gradient of lse they get that."""
    rows, slots = [1, 1, 5, 3, 1], [1, 4, 5, 1, 1]
    q, k, v, g = make(rows, slots, 6, 2, dim, dtype, seed=dim)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    ro, ko = starts(rows), starts(slots)
    out, lse = packed_attention(*leaves, on_device(ro), on_device(ko), causal=causal, return_lse=True)
    dq, dk, dv = torch.autograd.grad(out, leaves, g, retain_graph=True)
    alone_q = [0, 7, 8, 9, 10] + ([2] if causal else [])  # causal: the first of five frames, and two rows that see nothing
    assert not dq[alone_q].any() and not dk[[0, 10, 11]].any()
    assert bool(dq[1].any()) and bool(dq[3:7].any()) and bool(dk[1:10].any()) and bool(dv[[0, 10, 11]].any())
    glse = torch.randn(lse.shape, generator=torch.Generator().manual_seed(2)).cuda()
    dq, dk, _ = torch.autograd.grad((out, lse), leaves, (g, glse))
    want, err, _, _ = reference(q.detach(), k.detach(), v.detach(), ro, ko, None, causal, dim ** -0.5, g, glse)
    check(dq, want["dq"], err["dq"], "dq")
    check(dk, want["dk"], err["dk"], "dk")
    assert bool(dq[0].any()) and bool(dk[0].any())
