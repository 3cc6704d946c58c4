"""Decay attention, its gradients and its single rows against the formulas in 64 bits (GPU), and the refusals.

The bounds follow the roundings: u = half the distance of neighbouring values of the stored type (2^-24 or 2^-8 relative)
for the result; in 16 bits t = 2^-8 for the pairs' weights and the decayed rows, as operands of products; and in FP32 a decay
l^n, whose exponent is rounded ((n |log l| + 4) 2^-24 relative), and sums of dim products, of a chunk's rows (128 at most)
and of the chunks, one after the other."""
import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

from fastmd_b200 import _lib
from fastmd_b200.decay_attention import decay_attention, decay_attention_step

gpu = pytest.mark.gpu
F32, B16 = torch.float32, torch.bfloat16
E32 = 2.0 ** -24


def starts(sizes):
    return [sum(sizes[:i]) for i in range(len(sizes) + 1)]


def decays(heads, device="cuda"):
    """From one half-life a row to one in some hundreds; the last head of three or more forgets nothing."""
    log = torch.log1p(-(2.0 ** (-1 - 8 * (torch.arange(heads, dtype=torch.float64) + 0.5) / heads))).float()
    if heads >= 3:
        log[-1] = 0.0
    return log.to(device)


def mixed(a, b, c, log, gap):
    """sum_s e^{log gap} (a_t . b_s) c_s where gap >= 0, and its absolute sum and that with the decays' own errors."""
    w = torch.where(gap >= 0, torch.exp(log * gap.clamp(min=0)), 0.0)
    own = w * (4 + gap.clamp(min=0) * abs(log))
    bare = a.abs() @ b.abs().T
    return (w * (a @ b.T)) @ c, (w * bare) @ c.abs(), (own * bare) @ c.abs()


def reference(q, k, v, log, sizes, state, scale, g=None, gafter=None):
    dtype = q.dtype
    unit, t = (E32, 0.0) if dtype == F32 else (2.0 ** -8, 2.0 ** -8)
    heads, dim = q.shape[1:]
    q, k, v, log = (x.detach().double() for x in (q, k, v, log))
    g = torch.zeros_like(q) if g is None else g.double()
    first = torch.zeros(len(sizes), heads, dim, dim, device=q.device, dtype=torch.float64)
    last = torch.zeros_like(first)
    if state is not None:
        first = state.detach().double()
    if gafter is not None:
        last = gafter.double()
    want = {n: torch.zeros_like(x) for n, x in dict(out=q, dq=q, dk=k, dv=v, after=first, dstate=first).items()}
    err = {n: torch.zeros_like(x) for n, x in want.items()}
    for i, n in enumerate(sizes):
        row = slice(sum(sizes[:i]), sum(sizes[:i]) + n)
        at = torch.arange(n, device=q.device, dtype=torch.float64)
        gap = at[:, None] - at
        rough = E32 * (dim + 128 + n / 64 + 8)
        for h in range(heads):
            x, y, z, d, lg = q[row, h], k[row, h], v[row, h], g[row, h] * scale, float(log[h])
            since, until = torch.exp(lg * (at + 1))[:, None], torch.exp(lg * (n - 1 - at))[:, None]
            own_since, own_until = since * (4 + (at + 1) * -lg)[:, None], until * (4 + (n - 1 - at) * -lg)[:, None]
            whole, own_whole = math.exp(lg * n), math.exp(lg * n) * (4 + n * -lg)
            s, e = first[i, h], last[i, h]

            def put(name, index, parts, stored, cut):
                """parts: (value, absolute value, that with the decays' errors)"""
                value = sum(p[0] for p in parts)
                want[name][index] = value
                bound = sum((rough + cut) * p[1] + E32 * p[2] for p in parts)
                err[name][index] = bound + stored * (value.abs() + bound)

            def far(w, own, m, matrix):
                return w * (m @ matrix), w * (m.abs() @ matrix.abs()), own * (m.abs() @ matrix.abs())

            def outer(w, own, m, o):
                return (w * m).T @ o, (w * m.abs()).T @ o.abs(), (own * m.abs()).T @ o.abs()

            scaled = [scale * p for p in mixed(x, y, z, lg, gap)]
            put("out", (row, h), [scaled, [scale * p for p in far(since, own_since, x, s)]], unit, t)
            put("after", (i, h), [outer(until, own_until, y, z), (whole * s, whole * s.abs(), own_whole * s.abs())], E32, 0)
            put("dq", (row, h), [mixed(d, z, y, lg, gap), far(since, own_since, d, s.T)], unit, t)
            put("dk", (row, h), [mixed(z, d, x, lg, gap.T), far(until, own_until, z, e.T)], unit, t)
            put("dv", (row, h), [mixed(y, x, d, lg, gap.T), far(until, own_until, y, e)], unit, t)
            put("dstate", (i, h), [outer(since, own_since, x, d), (whole * e, whole * e.abs(), own_whole * e.abs())], E32, 0)
    return want, err


def check(got, want, err, what):
    assert got.shape == want.shape and bool(torch.isfinite(got).all()), what
    if not got.numel():
        return
    off = (got.double() - want).abs()
    assert bool((off <= err + 1e-30).all()), f"{what}: {float((off / (err + 1e-30)).amax()):.3g} times its bound"
    if got.dtype == B16 and got.numel() >= 40_000:
        # besides the result's own rounding one of each pair's weight or decayed row, as large on average: sqrt 2 in all,
        # and 6 % for the planes of the matrix and how far sums of thousands of roundings stray
        rounding = (want.to(B16).double() - want).norm()
        assert float(off.norm()) <= 1.5 * float(rounding), f"{what}: {float(off.norm() / rounding):.3f} times its rounding"


def make(sizes, heads, dim, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rows = sum(sizes)
    q, k, v, g = (torch.randn(rows, heads, dim, generator=gen).to(dtype).cuda() for _ in range(4))
    state, gafter = (torch.randn(len(sizes), heads, dim, dim, generator=gen).cuda() for _ in range(2))
    return q, k, v, g, state, gafter, torch.tensor(starts(sizes), device="cuda")


def run_case(sizes, heads, dim, dtype, with_state, seed=0):
    q, k, v, g, state, gafter, offsets = make(sizes, heads, dim, dtype, seed)
    log = decays(heads)
    want, err = reference(q, k, v, log, sizes, state if with_state else None, dim ** -0.5, g,
                          gafter if with_state else None)
    alone = decay_attention(q, k, v, log, offsets, state if with_state else None)
    check(alone, want["out"], err["out"], "out without gradients")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    if not with_state:
        out = decay_attention(q, k, v, log, offsets)
        check(out.detach(), want["out"], err["out"], "out")
        grads = torch.autograd.grad(out, leaves, g)
    else:
        leaves.append(state.requires_grad_())
        out, after = decay_attention(q, k, v, log, offsets, state, return_state=True)
        check(out.detach(), want["out"], err["out"], "out")
        check(after.detach(), want["after"], err["after"], "after")
        grads = torch.autograd.grad((out, after), leaves, (g, gafter))
    for name, got in zip(("dq", "dk", "dv", "dstate"), grads):
        check(got, want[name], err[name], name)


SEQUENCES = {
    "one": [1], "two": [2, 1], "frames": [135, 135, 135], "edges": [63, 64, 65, 1, 0, 127, 128, 129, 255, 0],
    "ragged": [5, 200, 0, 3, 311], "long": [1500], "zeros": [0, 0, 70], "short": [3, 0, 17, 1, 40, 5, 4, 8, 9], "single": [1] * 5,
}


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("with_state", [False, True], ids=["zeros", "state"])
@pytest.mark.parametrize("name", list(SEQUENCES))
@pytest.mark.parametrize("heads,dim", [(1, 8), (3, 64), (4, 128), (2, 32)])
def test_against_the_formulas(cuda, heads, dim, name, with_state, dtype):
    run_case(SEQUENCES[name], heads, dim, dtype, with_state, seed=dim + heads)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("dim", [16, 24, 40, 48, 56, 72, 80, 88, 96, 104, 112, 120])
def test_every_head_size_row_by_row(cuda, dim, dtype):
    run_case([5, 13, 0, 8, 1], 2, dim, dtype, True)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("dim", [16, 24, 40, 48, 56, 72, 80, 88, 96, 104, 112, 120])
def test_every_head_size(cuda, dim, dtype):
    run_case([150, 0, 77], 3, dim, dtype, True, seed=dim)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("sizes,heads,dim", [([3000], 1, 64), ([1100, 2, 1900, 700], 5, 64), ([2600, 601], 8, 128),
                                             ([700] * 3, 16, 96), ([20] * 400, 2, 32), ([257] * 40, 8, 64)],
                         ids=["one", "ragged", "two", "three", "many", "forty"])
def test_segments(cuda, sizes, heads, dim, dtype):
    """Sequences that are cut into segments, and many that are not."""
    run_case(sizes, heads, dim, dtype, True, seed=1)
    run_case(sizes, heads, dim, dtype, False, seed=2)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("seqs,heads,dim", [(1, 1, 8), (64, 8, 64), (5, 3, 24), (7, 16, 128), (3, 2, 120)])
def test_single_rows(cuda, seqs, heads, dim, dtype):
    """A step moves the state on and gives the row that the whole sequence has; its strides are free."""
    q, k, v, _, state, _, _ = make([1] * seqs, heads, dim, dtype, seed=dim)
    log = decays(heads)
    want, err = reference(q, k, v, log, [1] * seqs, state, dim ** -0.5)
    fused = torch.cat((q, k, v), 1)[:, :, None].expand(-1, -1, 2, -1).contiguous()[:, :, 0]
    now = state.clone()
    out = decay_attention_step(*fused.split(heads, 1), log, now)
    check(out, want["out"], err["out"], "out")
    check(now, want["after"], err["after"], "state")
    again = state.clone()
    assert torch.equal(decay_attention_step(q, k, v, log, again), out) and torch.equal(again, now)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_a_log_in_pieces(cuda, dtype):
    """One call, chunks of any lengths and single rows one after the other: the same outputs and states within bounds."""
    sizes, heads, dim = [300, 171], 4, 64
    q, k, v, _, state, _, offsets = make(sizes, heads, dim, dtype)
    log = decays(heads)
    want, err = reference(q, k, v, log, sizes, state, dim ** -0.5)
    now, done = state.clone(), 0
    for n in (1, 64, 3, 100, 0, 2):
        rows = torch.cat([torch.arange(offsets[b] + done, offsets[b] + done + n) for b in range(2)]).cuda()
        out, now = decay_attention(q[rows], k[rows], v[rows], log, torch.tensor([0, n, 2 * n], device="cuda"), now,
                                   return_state=True)
        check(out, want["out"][rows], err["out"][rows], f"rows {done}..")
        done += n
    rows = (offsets[:-1] + done)
    out = decay_attention_step(q[rows], k[rows], v[rows], log, now)
    check(out, want["out"][rows], err["out"][rows], "step")


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_other_sequences_do_not_count(cuda, dtype):
    """Values of other sequences, finite or not, and rows behind the last chunk do not reach a sequence."""
    sizes, heads, dim = [70, 130, 33], 3, 64
    q, k, v, g, state, gafter, offsets = make(sizes, heads, dim, dtype)
    log = decays(heads)

    def all_(q, k, v, g, state, gafter):
        leaves = [t.clone().requires_grad_() for t in (q, k, v, state)]
        out, after = decay_attention(*leaves[:3], log, offsets, leaves[3], return_state=True)
        return out.detach(), after.detach(), *torch.autograd.grad((out, after), leaves, (g, gafter))

    want = all_(q, k, v, g, state, gafter)
    for t in (q, k, v, g):
        t[70:200:2], t[71:200:2] = float("nan"), float("inf")
    state[1], gafter[1] = float("nan"), float("inf")
    got = all_(q, k, v, g, state, gafter)
    for i, (x, y) in enumerate(zip(want, got)):
        keep = [0, 2] if i in (1, 5) else [*range(70), *range(200, 233)]
        assert torch.equal(x[keep], y[keep]), i


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_strong_and_no_decay(cuda, dtype):
    """Decays of 0 keep all, of -inf and far below leave a row itself, above 0 count as 0."""
    q, k, v, _, state, _, offsets = make([200], 4, 32, dtype)
    log = torch.tensor([0.0, -math.inf, -200.0, 1.0], device="cuda")
    out, after = decay_attention(q, k, v, log, offsets, state, return_state=True)
    want, err = reference(q, k, v, torch.tensor([0.0, -1e4, -200.0, 0.0], device="cuda"), [200], state, 32 ** -0.5)
    check(out, want["out"], err["out"], "out")
    check(after, want["after"], err["after"], "after")
    now = state.clone()
    decay_attention_step(q[:1], k[:1], v[:1], log, now)
    assert torch.isfinite(now).all()


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_row_by_row_and_by_chunks(cuda, dtype):
    """The same rows as a batch of short sequences and beside a long one: decays at their limits, values of other sequences
    that are not finite, parts of the gradients, and offsets that do not fit."""
    sizes, heads, dim = [7, 0, 12, 1, 4], 4, 72
    q, k, v, g, state, gafter, offsets = make(sizes + [900], heads, dim, dtype)
    log = torch.tensor([0.0, -math.inf, -200.0, 1.0], device="cuda")
    q.data[3:5], state[2] = float("nan"), float("inf")  # of sequences 0 and 2

    def run(q, k, v, state, offsets, g, gafter):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, state)]
        out, after = decay_attention(*leaves[:3], log, offsets, leaves[3], return_state=True)
        grads = torch.autograd.grad((out, after), leaves, (g, gafter), retain_graph=True)
        (dv,) = torch.autograd.grad(out, leaves[2], g, retain_graph=True)
        (dstate,) = torch.autograd.grad(after, leaves[3], gafter)
        return out.detach(), after.detach(), *grads, dv, dstate

    rows, places = slice(19, 24), [3, 4]  # of the two sequences that are finite
    args = [t[rows] for t in (q, k, v)], torch.tensor([0.0, -1e4, -200.0, 0.0], device="cuda"), [1, 4], state[places]
    bounds = [reference(*args[0], *args[1:], dim ** -0.5, *grads)
              for grads in ((g[rows], gafter[places]), (g[rows], None), (None, gafter[places]))]
    for got in (run(q[:24], k[:24], v[:24], state[:5], offsets[:6], g[:24], gafter[:5]),
                run(q, k, v, state, offsets, g, gafter)):
        for i, (name, x) in enumerate(zip(("out", "after", "dq", "dk", "dv", "dstate", "dv", "dstate"), got)):
            want, err = bounds[max(0, i - 5)]
            check(x[places if x.dim() == 4 else rows], want[name], err[name], f"{i} {name}")
        assert torch.equal(got[1][1], state[1])  # nothing happened there
    flags = _lib.flags_word(q.device)
    for bad in ([0, 9, 7, 24], [1, 5, 9, 24], [0, 5, 9, 20], [0, 5, 9, 90], [0, -9, 9, 24], [0, 2 ** 60, 9, 24]):
        flags.zero_()
        decay_attention(q[:24], k[:24], v[:24], log, torch.tensor(bad, device="cuda"), return_state=True)
        assert int(flags.item()) & 1, bad
    flags.zero_()


@gpu
@pytest.mark.parametrize("dtype,dim", [(F32, 64), (F32, 72), (B16, 64)], ids=["planes", "f32", "b16"])
def test_a_decay_of_nan_gives_nan(cuda, dtype, dim):
    """It is not taken for one of the values that count as 0, and other heads do not see it."""
    q, k, v, _, state, _, offsets = make([300, 7], 2, dim, dtype)
    log = torch.tensor([math.nan, -0.1], device="cuda")
    want = decay_attention(q, k, v, log.nan_to_num(), offsets, state, return_state=True)
    got = decay_attention(q, k, v, log, offsets, state, return_state=True)
    for x, y in zip(got, want):
        assert torch.equal(x[:, 1], y[:, 1])
    assert torch.isnan(got[1][0, 0]).all() and torch.isnan(got[0][:, 0]).all()
    now = state.clone()
    assert torch.isnan(decay_attention_step(q[:2], k[:2], v[:2], log, now)[:, 0]).all() and torch.isfinite(now[:, 1]).all()


@gpu
@pytest.mark.parametrize("dtype,heads,dim", [(F32, 17, 64), (F32, 17, 128), (B16, 17, 128)], ids=["planes", "f32", "b16"])
def test_arrays_past_32_bits(cuda, dtype, heads, dim):
    """More than 2^31 values an array: the last sequence's rows and those of its first state."""
    tail = 300
    rows = 2 ** 31 // (heads * dim) + 5000
    x = torch.zeros(rows, heads, dim, device="cuda", dtype=dtype)
    q, k, v, g, state, gafter, _ = make([tail], heads, dim, dtype)
    x[-tail:] = q
    y = x.clone()
    y[-tail:] = k
    offsets = torch.tensor([0, 900, rows - tail, rows], device="cuda")
    states = torch.cat((torch.zeros_like(state), torch.zeros_like(state), state))
    log = decays(heads)
    want, err = reference(q, k, k, log, [tail], state, dim ** -0.5)
    out, after = decay_attention(x, y, y, log, offsets, states, return_state=True)
    check(out[-tail:], want["out"], err["out"], "out")
    check(after[2:], want["after"], err["after"], "after")
    assert not out[:-tail].any() and not after[:2].any()
    del x, y, out
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_strides_and_parts(cuda, dtype):
    sizes, heads, dim = [100, 61], 3, 40
    q, k, v, g, state, gafter, offsets = make(sizes, heads, dim, dtype)
    log = decays(heads)
    want = decay_attention(q, k, v, log, offsets, state)
    fused = torch.cat((q, k, v), 1)
    assert torch.equal(decay_attention(*fused.split(heads, 1), log, offsets, state), want)
    odd = torch.empty(161 * heads * dim + 1, device="cuda", dtype=dtype)[1:].view(161, heads, dim)
    odd.copy_(k)
    far = torch.empty(3, heads, dim, dim, device="cuda")[::2]
    far.copy_(state)
    flip = v.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(decay_attention(q, odd, flip, log, offsets, far), want)
    leaves = [t.requires_grad_() for t in (q, k, v, state)]
    out, after = decay_attention(*leaves[:3], log, offsets, state, return_state=True)
    full = torch.autograd.grad((out, after), leaves, (g, gafter), retain_graph=True)
    for i in range(4):
        (one,) = torch.autograd.grad((out, after), leaves[i], (g, gafter), retain_graph=True)
        assert torch.equal(one, full[i]), i
    # of out alone, of the state alone, and of an expanded gradient
    parts = [torch.autograd.grad(o, leaves, go, retain_graph=True, allow_unused=True) for o, go in ((out, g), (after, gafter))]
    for i in range(4):
        total = parts[0][i].double() + (0 if parts[1][i] is None else parts[1][i].double())
        assert float((total - full[i].double()).norm()) <= (2.0 ** -7 if dtype == B16 and i < 3 else 2.0 ** -20) * \
            float(total.norm())
    (broad,) = torch.autograd.grad(out.sum(), q, retain_graph=True)
    (ones,) = torch.autograd.grad(out, q, torch.ones_like(out))
    assert torch.equal(broad, ones)


class Elsewhere(torch.autograd.graph.saved_tensors_hooks):
    """Brings what is saved back in memory that starts one value further than a tensor of its own."""

    def __init__(self):
        super().__init__(lambda t: t.detach().cpu(), self.back)

    @staticmethod
    def back(t):
        return torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)[1:].view(t.shape).copy_(t)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("sizes", [[9, 3], [100, 61], [2000]], ids=["rows", "chunks", "segments"])
def test_saved_tensors_that_come_back_otherwise(cuda, sizes, dtype):
    """Hooks that move what is saved (to the host and back) may give it another start: the gradients are the same, to the bit."""
    heads, dim = 3, 72
    q, k, v, g, state, gafter, offsets = make(sizes, heads, dim, dtype)
    leaves, grads = [t.requires_grad_() for t in (q, k, v, state)], (g, gafter)
    log = decays(heads)

    def call():
        return decay_attention(q, k, v, log, offsets, state, return_state=True)

    want = torch.autograd.grad(call(), leaves, grads)
    for hook in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True), Elsewhere()):
        with hook:
            both = call()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(both, leaves, grads), want))


@gpu
def test_gradients_against_differences(cuda):
    q, k, v, g, state, gafter, offsets = make([9, 40], 2, 16, F32)
    log = decays(2)
    leaves = [t.requires_grad_() for t in (q, k, v, state)]

    def value(args):
        out, after = decay_attention(*args[:3], log, offsets, args[3], return_state=True)
        return (out.double() * g).sum() + (after.double() * gafter).sum()

    out, after = decay_attention(q, k, v, log, offsets, state, return_state=True)
    grads = torch.autograd.grad((out, after), leaves, (g, gafter))
    gen = torch.Generator(device="cuda").manual_seed(1)
    for leaf, grad in zip(leaves, grads):  # linear in each: differences are exact but for roundings
        way = torch.randn(leaf.shape, generator=gen, device="cuda")
        ends = [value([t.detach() + sign * 0.5 * way if t is leaf else t.detach() for t in leaves]) for sign in (1, -1)]
        got, want = float(ends[0] - ends[1]), float((grad.double() * way).sum())
        assert abs(got - want) <= 1e-4 * (1 + abs(want)), (got, want)


@gpu
@pytest.mark.parametrize("dtype,sizes,dim", [(F32, [600, 250], 64), (B16, [600, 250], 64), (F32, [600, 250], 104),
                                             (F32, [900, 1400], 72), (F32, [9, 3], 72), (B16, [9, 3], 64)],
                         ids=["f32", "b16", "f32-parts", "f32-segments", "f32-few", "b16-few"])
def test_captured_and_repeated(cuda, dtype, sizes, dim):
    """Forward, backward and steps in a graph, replayed on other values and lengths; the same bits on every run."""
    heads = 3
    q, k, v, g, state, gafter, offsets = make(sizes, heads, dim, dtype)
    log = decays(heads)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    row, moving = [t.detach()[:2] for t in leaves], state.clone()

    def work():
        out, after = decay_attention(q, k, v, log, offsets, state, return_state=True)
        step = decay_attention_step(*row, log, moving)
        return out, after, step, *torch.autograd.grad((out, after), leaves, (g, gafter))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    with torch.no_grad():
        q.mul_(-1.5)
        offsets[1] = 130 if sizes[0] > 130 else 4
        moving.copy_(state)
    graph.replay()
    moving.copy_(state)
    graph.replay()
    moving.copy_(state)
    for a, b in zip(got, work()):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("sizes", [[64] * 100, [6000, 400]], ids=["chunks", "segments"])
def test_planes_that_are_handed_over_take_no_room(cuda, sizes):
    """float32: the forward pass's planes of q, k and v are not given room again. The backward pass allocates its gradients, the
    planes of the output's gradient (6 bytes a value) and the segments' matrices, and writes nothing behind its workspace."""
    heads, dim = 3, 72
    q, k, v, g, state, gafter, offsets = make(sizes, heads, dim, F32)
    log, leaves = decays(heads), [t.requires_grad_() for t in (q, k, v, state)]

    def step():
        both = decay_attention(q, k, v, log, offsets, state, return_state=True)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        grads = torch.autograd.grad(both, leaves, (g, gafter))
        return grads, torch.cuda.max_memory_allocated() - before

    step()
    want, used = step()
    values, matrices = q.numel(), 3 * (sum(sizes) // 256 + len(sizes)) * heads * dim * dim * 4
    assert used <= 3 * 4 * values + state.numel() * 4 + 6 * values + matrices + 2 ** 20

    def problem():
        return _lib.FmdDecay(q.data_ptr(), k.data_ptr(), v.data_ptr(), log.data_ptr(), offsets.data_ptr(), q.shape[0],
                             heads * dim, dim, heads * dim, dim, heads * dim, dim, dim ** -0.5, 0, len(sizes), heads, dim)

    def room(backward, guard=0):
        nbytes = ctypes.c_size_t()
        _lib.call("fmd_decay_attention_workspace_bytes", problem(), backward, nbytes)
        return torch.full((nbytes.value + guard,), 0xA5, device="cuda", dtype=torch.uint8), nbytes.value

    forward, size = room(0)
    flags, stream = _lib.flags_word(q.device).data_ptr(), _lib.stream(q.device)
    out, grads = torch.empty_like(q), [torch.empty_like(t) for t in leaves]
    _lib.call("fmd_decay_attention", problem(), state.data_ptr(), out.data_ptr(), None, forward.data_ptr(), size, flags, stream)
    for handed in (forward.data_ptr(), None):
        work, size = room(2 if handed else 1, 4096)
        for t in grads:
            t.fill_(float("nan"))
        _lib.call("fmd_decay_attention_bwd", problem(), state.data_ptr(), handed, g.data_ptr(), heads * dim, dim,
                  gafter.data_ptr(), *(t.data_ptr() for t in grads), work.data_ptr(), size, flags, stream)
        assert bool((work[size:] == 0xA5).all())
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_the_workspace_of_a_backward_pass_with_planes():
    lib, one, all_ = _lib.lib(), ctypes.c_size_t(), ctypes.c_size_t()
    for kind, rows, batch in ((0, 4000, 2), (0, 4000, 200), (0, 40, 2), (1, 4000, 2)):
        f = _lib.FmdDecay(1 << 20, 1 << 20, 1 << 20, 1 << 20, 1 << 20, rows, 32, 16, 32, 16, 32, 16, 1.0, kind, batch, 2, 16)
        assert lib.fmd_decay_attention_workspace_bytes(f, 1, all_) == 0 and lib.fmd_decay_attention_workspace_bytes(f, 2, one) == 0
        planes = rows * 32 * 6 if kind == 0 and rows > 32 * batch else 0
        assert all_.value - one.value == 3 * planes and one.value >= planes
        p = ctypes.c_void_p(1 << 20)
        if one.value:
            assert lib.fmd_decay_attention_bwd(f, None, p, p, 32, 16, None, p, p, p, None, p, one.value - 1, None, None) == 4


@gpu
def test_two_streams_at_once(cuda):
    q, k, v, g, state, gafter, offsets = make([2100, 1300, 5], 6, 64, B16)
    log = decays(6)
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def grads():
        out, after = decay_attention(q, k, v, log, offsets, state, return_state=True)
        return torch.autograd.grad((out, after), leaves, (g, gafter))

    want = grads()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(grads())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for one in got for a, b in zip(one, want))


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_no_rows_and_no_sequences(cuda, dtype):
    q = torch.zeros(0, 2, 16, device="cuda", dtype=dtype, requires_grad=True)
    log = decays(2)
    state = torch.randn(3, 2, 16, 16, device="cuda", requires_grad=True)
    out, after = decay_attention(q, q, q, log, torch.zeros(4, dtype=torch.int64, device="cuda"), state, return_state=True)
    assert out.shape == (0, 2, 16) and torch.equal(after, state)
    g = torch.randn_like(after)
    dq, dstate = torch.autograd.grad((out, after), (q, state), (torch.zeros_like(out), g))
    assert dq.shape == q.shape and torch.equal(dstate, g)
    out, after = decay_attention(q, q, q, log, torch.zeros(1, dtype=torch.int64, device="cuda"), return_state=True)
    assert out.shape == (0, 2, 16) and after.shape == (0, 2, 16, 16)
    none = q.detach()
    assert decay_attention_step(none, none, none, log, torch.zeros(0, 2, 16, 16, device="cuda")).shape == (0, 2, 16)


@gpu
@pytest.mark.parametrize("offsets", [[0, 50, 40, 100], [5, 50, 60, 100], [0, 50, 60, 90], [0, 50, 60, 200], [0, -9, 60, 100],
                                     [0, 2 ** 40, 60, 100], [-(2 ** 40), 50, 60, 100]])
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_bad_offsets_are_flagged(cuda, offsets, dtype):
    q, k, v, g, state, gafter, _ = make([50, 10, 40], 2, 16, dtype)
    word = _lib.flags_word(q.device)
    for keep in (False, True):
        word.zero_()
        leaves = [t.detach().requires_grad_() for t in (q, k, v, state)]
        out = decay_attention(*leaves[:3], decays(2), torch.tensor(offsets, device="cuda"), leaves[3], return_state=keep)
        assert int(word.item()) & 1
        torch.autograd.grad(out, leaves, (g, gafter) if keep else g)
        torch.cuda.synchronize()
    word.zero_()


@gpu
@pytest.mark.parametrize("dtype,sizes,dim", [(B16, [900, 1400], 64), (F32, [900, 1400], 64), (B16, [2300], 128)],
                         ids=["b16", "f32", "b16-one"])
def test_captured_segments(cuda, dtype, sizes, dim):
    """The same where sequences are cut into segments, and where they become so few rows that most segments are empty."""
    if len(sizes) == 2:
        test_captured_and_repeated(cuda, dtype, sizes, dim)
        return
    q, k, v, g, state, gafter, offsets = make(sizes, 3, dim, dtype)
    log, leaves = decays(3), [t.requires_grad_() for t in (q, k, v, state)]

    def work():
        out, after = decay_attention(q, k, v, log, offsets, state, return_state=True)
        return out, after, *torch.autograd.grad((out, after), leaves, (g, gafter))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for _ in range(2):
        with torch.no_grad():
            v.mul_(-0.5)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, work()))


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("sizes,heads,dim", [([200] + [0] * 20 + [3] * 5, 2, 64), ([0] * 15 + [1, 180], 3, 128),
                                             ([2000] + [50] * 30, 2, 64), ([40] * 9 + [1700] + [35] * 9, 3, 72)],
                         ids=["row_by_row", "last", "chunks", "between"])
def test_one_long_log_among_short_ones(cuda, sizes, heads, dim, dtype):
    """The choice of kernels goes by the average length. Row by row a decay l^n is a product of n numbers that are rounded once,
    n / 2 units of 2^-24: for the 200 rows here less than the 128 units of a chunk's sum, which is not taken."""
    run_case(sizes, heads, dim, dtype, True, seed=dim)


@gpu
@pytest.mark.parametrize("offsets", [[0, 900, 700, 2300], [5, 900, 1400, 2300], [0, 900, 1400, 2200], [0, 900, 1400, 2400],
                                     [0, -9, 1400, 2300], [0, 2 ** 40, 1400, 2300], [-(2 ** 40), 900, 1400, 2300],
                                     [0, 2300, 0, 2300], [2300, 2300, 2300, 2300]])
@pytest.mark.parametrize("dtype,dim", [(F32, 16), (F32, 72), (B16, 64)], ids=["planes", "parts", "b16"])
def test_bad_offsets_are_flagged_with_segments(cuda, offsets, dtype, dim):
    """Nothing outside the arrays is touched: sequences cut into segments, forward and backward."""
    sizes, heads = [900, 500, 900], 3
    q, k, v, g, state, gafter, good = make(sizes, heads, dim, dtype)
    word, log = _lib.flags_word(q.device), decays(heads)
    want = decay_attention(q, k, v, log, good, state)
    bad = torch.tensor(offsets, device="cuda")
    for keep in (False, True):
        word.zero_()
        leaves = [t.detach().requires_grad_() for t in (q, k, v, state)]
        out = decay_attention(*leaves[:3], log, bad, leaves[3], return_state=keep)
        assert int(word.item()) & 1
        torch.autograd.grad(out, leaves, (g, gafter) if keep else g)
        torch.cuda.synchronize()
    word.zero_()
    assert torch.equal(decay_attention(q, k, v, log, good, state), want) and int(word.item()) == 0


@gpu
def test_refusals(cuda):
    q, k, v, _, state, _, offsets = make([5, 3], 2, 16, B16)
    log = decays(2)
    for args, text in (((q, k[:, :1], v, log, offsets), "rows, heads, dim"), ((q, k, v.float(), log, offsets), "bfloat16"),
                       ((q[..., :12], k[..., :12], v[..., :12], log, offsets), "multiple of 8"),
                       ((q, k, v, log[:1], offsets), "log_decay"), ((q, k, v, log.double(), offsets), "log_decay"),
                       ((q, k, v, log, offsets.int()), "offsets"), ((q, k, v, log, offsets[:1]), "without a sequence"),
                       ((q, k, v, log, offsets, state[:1]), "state"), ((q, k, v, log, offsets, state.double()), "state")):
        with pytest.raises(ValueError, match=text):
            decay_attention(*args)
    with pytest.raises(ValueError, match="scale"):
        decay_attention(q, k, v, log, offsets, scale=-1.0)
    with pytest.raises(ValueError, match="log_decay has no gradient"):
        decay_attention(q, k, v, log.requires_grad_(), offsets)
    log = log.detach()
    with pytest.raises(ValueError, match="state"):
        decay_attention_step(q, k, v, log, state)
    whole = torch.zeros(8, 2, 16, 16, device="cuda")
    with pytest.raises(ValueError, match="contiguous"):
        decay_attention_step(q, k, v, log, whole.transpose(2, 3))
    with pytest.raises(ValueError, match="no gradient"):
        decay_attention_step(q.requires_grad_(), k, v, log, whole)
    out = decay_attention(q, k, v, log, offsets)
    (dq,) = torch.autograd.grad(out, q, torch.ones_like(out), create_graph=True)
    with pytest.raises(RuntimeError, match="first derivatives only"):
        torch.autograd.grad(dq.float().sum(), q)
    with forward_ad.dual_level(), pytest.raises(RuntimeError):
        decay_attention(forward_ad.make_dual(q.detach(), torch.ones_like(q)), k, v, log, offsets)
    saved = torch.zeros(8, 2, 16, 16, device="cuda", requires_grad=True)
    product = (saved * saved).sum()  # a state that autograd has saved and a step has changed is noticed
    with torch.no_grad():
        decay_attention_step(q.detach(), k, v, log, saved)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()


def test_cpu_tensors_are_refused():
    q, log = torch.zeros(4, 2, 16), torch.zeros(2)
    with pytest.raises(_lib.FastMDLibraryError):
        decay_attention(q, q, q, log, torch.tensor([0, 4]))
    with pytest.raises(_lib.FastMDLibraryError):
        decay_attention_step(q, q, q, log, torch.zeros(4, 2, 16, 16))


def test_bad_arguments_of_the_entry_points_launch_nothing():
    lib, p, odd = _lib.lib(), ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 4)
    nbytes = ctypes.c_size_t()

    def problem(**change):
        sizes = dict(q=1 << 20, k=1 << 20, v=1 << 20, log_decay=1 << 20, offsets=1 << 20, rows=8, q_row=32, q_head=16,
                     k_row=32, k_head=16, v_row=32, v_head=16, scale=1.0, type=1, batch=2, heads=2, dim=16)
        return _lib.FmdDecay(**{**sizes, **change})

    assert lib.fmd_decay_attention_workspace_bytes(problem(), 0, nbytes) == 0 and nbytes.value == 0
    assert lib.fmd_decay_attention_workspace_bytes(problem(rows=4000, type=0), 1, nbytes) == 0
    need = nbytes.value  # planes of four inputs and what the segments of three passes add
    assert need >= 4 * 4000 * 32 * 6 + 3 * 2 * 2 * 16 * 16 * 4
    for change in (dict(type=3), dict(rows=-1), dict(batch=-1), dict(heads=0), dict(dim=12), dict(dim=136), dict(scale=-1.0),
                   dict(scale=float("nan")), dict(q=None), dict(log_decay=None), dict(offsets=None), dict(batch=0)):
        assert lib.fmd_decay_attention_workspace_bytes(problem(**change), 0, nbytes) == 1, change
    for change in (dict(q=(1 << 20) + 2), dict(k_row=33), dict(v_head=12), dict(rows=1 << 30), dict(heads=2000)):
        assert lib.fmd_decay_attention_workspace_bytes(problem(**change), 0, nbytes) == 3, change
    f = problem()
    assert lib.fmd_decay_attention(None, None, p, None, None, 0, None, None) == 1
    assert lib.fmd_decay_attention(f, None, None, None, None, 0, None, None) == 1
    assert lib.fmd_decay_attention(problem(rows=4000, type=0), None, p, p, p, 8, None, None) == 4
    assert lib.fmd_decay_attention(f, odd, p, None, None, 0, None, None) == 3
    assert lib.fmd_decay_attention_bwd(f, None, None, None, 32, 16, None, p, p, p, None, None, 0, None, None) == 1
    assert lib.fmd_decay_attention_bwd(f, None, None, p, 33, 16, None, p, p, p, None, None, 0, None, None) == 3
    assert lib.fmd_decay_attention_bwd(problem(rows=4000, type=0), None, None, p, 32, 16, None, p, p, p, p, p, need - 1, None, None) == 4
    assert lib.fmd_decay_attention_step(f, None, p, None) == 1
    assert lib.fmd_decay_attention_step(f, odd, p, None) == 3
    assert lib.fmd_decay_attention_step(problem(rows=0), None, None, None) == 0
