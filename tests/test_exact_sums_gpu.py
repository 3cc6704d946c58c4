"""float32 results of decay attention and the gated feed-forward, and the states in both types, by their mean error (GPU).

A bound on each value by the sum of its terms' sizes has to allow for errors that all point one way; it would not see a
plane of the operands that went lost. The mean square of all values' errors is narrower. With T the root of the sum of a sum's
squared terms, in units of 2^-24 T:

* a product of planes adds its large part 16 terms at a time into FP32 that is cut off. A step cuts up to two units of the
  sum so far, one on average, and that sum, of terms of either sign, has grown to sqrt(k / K) T after k of K steps: 2/3 of K
  steps' units in all, of which the size of a normal variable (0.8) leaves 0.55. CUT = 0.6 a step, and ROUND = 2 for the
  roundings that follow or go before.
* a decay l^n is known to 4 + n |log l| units of itself, and each activation to 4.
* sums of parts of sums add a third of a unit for each, of random sign.

What the six products of planes leave out is below a unit. Any one of them that went lost is 20 units (2^-9 of a value in the
second plane, 2^-18 in the third, uniform): `test_a_lost_plane_is_seen` computes with five of them, in 64 bits on the CPU."""
import math

import pytest
import torch

from fastmd_b200.decay_attention import decay_attention
from fastmd_b200.gated_feed_forward import gated_feed_forward

gpu = pytest.mark.gpu
F32, B16 = torch.float32, torch.bfloat16
E32, CUT, ROUND = 2.0 ** -24, 0.6, 2.0


def units_of(steps, parts=1):
    return CUT * steps + ROUND + 0.33 * math.sqrt(parts)


def share_of(got, want, rms):
    """The error as a share of what is allowed."""
    assert got.shape == want.shape and bool(torch.isfinite(got).all())
    return float((got.double() - want).norm() / rms.norm())


def check(got, want, rms, what):
    share = share_of(got, want, rms)
    assert share <= 1.0, f"{what}: {share:.3f} times its bound"


# ------------------------------------------------------------ the feed-forward block

def activation(a, kind):
    share = torch.sigmoid(a) if kind == "silu" else 0.5 * torch.special.erfc(-a * math.sqrt(0.5))
    if kind == "silu":
        return a * share, share + a * share * (1 - share)
    return a * share, share + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)


def product(a, b, ea=None, eb=None):
    """a @ b.T and the root mean square of its error, from those of a and b (None: exact)."""
    n = a.shape[1]
    # a sum starts anew every 128 values
    square = (E32 * units_of(min(8, n / 16), math.ceil(n / 128))) ** 2 * (a.square() @ b.square().T)
    if ea is not None:
        square = square + ea.square() @ b.square().T
    if eb is not None:
        square = square + a.square() @ eb.square().T
    return a @ b.T, square.sqrt()


def feed_reference(x, wg, wu, wd, g, kind):
    (a, ea), (b, eb) = product(x, wg), product(x, wu)
    level, slope = activation(a, kind)
    # |act'| and |act''| are at most 1.13
    el, es = ((1.13 * ea).square() + (4 * E32 * (1 + v.abs())).square() for v in (level, slope))
    h, eh = level * b, (el * b.square() + level.square() * eb.square() + (E32 * level * b).square()).sqrt()
    dh, edh = product(g, wd.T)
    da, db = dh * b * slope, dh * level
    eda = (edh.square() * (b * slope).square() + (dh * slope * eb).square() + es * (dh * b).square() + (2 * E32 * da).square()).sqrt()
    edb = (edh.square() * level.square() + el * dh.square() + (E32 * db).square()).sqrt()
    both = torch.cat((da, db), 1), torch.cat((wg, wu)).T, torch.cat((eda, edb), 1)
    return {"y": product(h, wd, eh), "dx": product(*both), "dgate": product(da.T, x.T, eda.T), "dup": product(db.T, x.T, edb.T),
            "ddown": product(g.T, h.T, None, eh.T)}


def feed_values(rows, width, hidden, out, seed, device):
    gen = torch.Generator().manual_seed(seed)
    shapes = ((rows, width, 1.0), (hidden, width, 1.5 * width ** -0.5), (hidden, width, width ** -0.5),
              (out, hidden, hidden ** -0.5), (rows, out, 1.0))
    return [(torch.randn(m, n, generator=gen) * scale).to(device) for m, n, scale in shapes]


@gpu
@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("rows,width,hidden,out", [(33, 512, 1365, 512), (64, 256, 512, 256), (300, 513, 129, 65),
                                                   (1000, 256, 512, 256), (3001, 72, 200, 1030)])
def test_feed_forward(cuda, rows, width, hidden, out, kind):
    *leaves, g = feed_values(rows, width, hidden, out, rows, cuda)
    want = feed_reference(*(t.double() for t in (*leaves, g)), kind)
    check(gated_feed_forward(*leaves, activation=kind), *want["y"], "y without gradients")
    leaves = [t.requires_grad_() for t in leaves]
    y = gated_feed_forward(*leaves, activation=kind)
    check(y.detach(), *want["y"], "y")
    for name, got in zip(("dx", "dgate", "dup", "ddown"), torch.autograd.grad(y, leaves, g)):
        check(got, *want[name], name)


# ------------------------------------------------------------ decay attention

def mixed(a, b, c, log, gap, units):
    """sum e^{log gap} (a_t . b_s) c_s where gap >= 0, and the mean square of its error."""
    seen, n = gap >= 0, gap.clamp(min=0)
    weight = torch.where(seen, torch.exp(log * n), 0.0)
    score, pairs = a @ b.T, (E32 * units[0]) ** 2 * (a.square() @ b.square().T)
    own = (E32 * (units[1] ** 2 + (4 - log * n) ** 2).sqrt()) ** 2
    return (weight * score) @ c, (weight.square() * (pairs + own * score.square())) @ c.square()


def far(w, n, log, m, matrix, units):
    """w (m @ matrix) with a decay w of n rows for each row of m, and its mean square error."""
    own = (E32 * (units[1] ** 2 + (4 - log * n) ** 2).sqrt()) ** 2
    return w[:, None] * (m @ matrix), (w.square() * own)[:, None] * (m.square() @ matrix.square())


def decay_reference(q, k, v, log, sizes, state, g, gafter):
    """The results of decay attention and the roots of the mean squares of their errors."""
    heads, dim = q.shape[1:]
    names = dict(out=q, dq=q, dk=k, dv=v, after=state, dstate=state)
    want, square = ({n: torch.zeros_like(t) for n, t in names.items()} for _ in range(2))
    scale, row = dim ** -0.5, 0
    for i, count in enumerate(sizes):
        at = torch.arange(count, device=q.device, dtype=torch.float64)
        here, gap = slice(row, row + count), at[:, None] - at
        # pairs: the head's values, by parts of 64; then a chunk's 128 rows, and the chunks or segments before it
        units = units_of(min(dim, 64) / 16, dim / 64), units_of(8, 4 + count / 128)
        for h in range(heads):
            x, y, z, d, lg = q[here, h], k[here, h], v[here, h], g[here, h] * scale, float(log[h])
            since, until = torch.exp(lg * (at + 1)), torch.exp(lg * (count - 1 - at))
            behind, first, last = count - 1 - at, state[i, h], gafter[i, h]

            def put(name, index, *parts):
                want[name][index], square[name][index] = sum(p[0] for p in parts), sum(p[1] for p in parts)

            def scaled(part):
                return scale * part[0], scale ** 2 * part[1]

            def outer(w, n, m, o):
                own = (E32 * (units[1] ** 2 + (4 - lg * n) ** 2).sqrt()) ** 2
                return (w[:, None] * m).T @ o, ((w.square() * own)[:, None] * m.square()).T @ o.square()

            whole, own = math.exp(lg * count), (E32 * (4 - lg * count + units[1])) ** 2
            put("out", (here, h), scaled(mixed(x, y, z, lg, gap, units)), scaled(far(since, at + 1, lg, x, first, units)))
            put("after", (i, h), outer(until, behind, y, z), (whole * first, own * (whole * first).square()))
            put("dq", (here, h), mixed(d, z, y, lg, gap, units), far(since, at + 1, lg, d, first.T, units))
            put("dk", (here, h), mixed(z, d, x, lg, gap.T, units), far(until, behind, lg, z, last.T, units))
            put("dv", (here, h), mixed(y, x, d, lg, gap.T, units), far(until, behind, lg, y, last, units))
            put("dstate", (i, h), outer(since, at + 1, x, d), (whole * last, own * (whole * last).square()))
        row += count
    return {n: (want[n], square[n].sqrt()) for n in want}


def decay_values(sizes, heads, dim, dtype, seed, device):
    gen = torch.Generator().manual_seed(seed)
    q, k, v, g = (torch.randn(sum(sizes), heads, dim, generator=gen).to(dtype).to(device) for _ in range(4))
    state, gafter = (torch.randn(len(sizes), heads, dim, dim, generator=gen).to(device) for _ in range(2))
    log = torch.log1p(-(2.0 ** (-1 - 8 * (torch.arange(heads, dtype=torch.float64) + 0.5) / heads))).float()
    log[-1] = 0.0  # nothing is forgotten
    offsets = torch.tensor([sum(sizes[:i]) for i in range(len(sizes) + 1)])
    return q, k, v, g, state, gafter, log.to(device), offsets.to(device)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("heads,dim", [(3, 8), (4, 32), (3, 64), (3, 96), (4, 128)])
@pytest.mark.parametrize("sizes", [[1] * 40, [3, 17, 0, 9, 30], [135, 60, 250], [1500], [2000, 700]],
                         ids=["single", "rows", "chunks", "one", "segments"])
def test_decay_attention(cuda, sizes, heads, dim, dtype):
    """In bfloat16 the states alone, whose sums are exact to FP32 too."""
    q, k, v, g, state, gafter, log, offsets = decay_values(sizes, heads, dim, dtype, dim, cuda)
    want = decay_reference(*(t.double() for t in (q, k, v, log)), sizes, *(t.double() for t in (state, g, gafter)))
    leaves = [t.requires_grad_() for t in (q, k, v, state)]
    out, after = decay_attention(q, k, v, log, offsets, state, return_state=True)
    grads = torch.autograd.grad((out, after), leaves, (g, gafter))
    for name, got in zip(("out", "after", "dq", "dk", "dv", "dstate"), (out.detach(), after.detach(), *grads)):
        if dtype == F32 or name in ("after", "dstate"):
            check(got, *want[name], name)


# ------------------------------------------------------------ what the bounds see (CPU)

def planes(x, count=3):
    got, left = [], x.clone()
    for _ in range(count):
        got.append(left.float().bfloat16().double())
        left = left - got[-1]
    return got


SIX = [(2, 0), (1, 1), (0, 2), (1, 0), (0, 1), (0, 0)]


def by_planes(a, b, pairs):
    x, y = planes(a), planes(b)
    return sum(x[i] @ y[j].T for i, j in pairs)


@pytest.mark.parametrize("lost", [None, *SIX[:5]])
def test_a_lost_plane_is_seen(lost):
    """Each of the products of planes counts at least one and a half times the bounds, and all six together next to nothing."""
    pairs = [p for p in SIX if p != lost]
    x, wg, wu, wd, g = (t.double() for t in feed_values(64, 256, 512, 256, 1, "cpu"))
    shares = []
    for a, b in ((x, wg), (g, wd.T), (torch.cat((g.T, g.T), 1), torch.cat((x.T, x.T), 1))):
        want, rms = product(a, b)
        shares.append(share_of(by_planes(a, b, pairs), want, rms))
    q, k, v, g, state, gafter, log, _ = decay_values([128], 2, 64, F32, 2, "cpu")
    q, k, v, g, state, gafter, log = (t.double() for t in (q, k, v, g, state, gafter, log))
    want = decay_reference(q, k, v, log, [128], torch.zeros_like(state), g, torch.zeros_like(state))
    at = torch.arange(128, dtype=torch.float64)
    out, again, after = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(state)
    for h in range(2):
        gap = at[:, None] - at
        weight = torch.where(gap >= 0, torch.exp(log[h] * gap.clamp(min=0)), 0.0) * 64 ** -0.5
        out[:, h] = (weight * by_planes(q[:, h], k[:, h], pairs)) @ v[:, h]  # lost among the scores
        again[:, h] = by_planes(weight * (q[:, h] @ k[:, h].T), v[:, h].T, pairs)  # and among the weights times values
        decayed = torch.exp(log[h] * (127 - at))[:, None] * k[:, h]
        after[0, h] = by_planes(decayed.T, v[:, h].T, pairs)
    shares += [share_of(t, *want[n]) for n, t in (("out", out), ("out", again), ("after", after))]
    assert max(shares) <= 0.1 if lost is None else min(shares) >= 1.5, shares


def test_a_lost_plane_of_the_decayed_rows_is_seen():
    """bfloat16: two planes of the decayed rows in place of three, in the states."""
    q, k, v, g, state, gafter, log, _ = decay_values([128], 2, 64, B16, 2, "cpu")
    none = torch.zeros_like(state).double()
    want = decay_reference(*(t.double() for t in (q, k, v, log)), [128], none, g.double(), none)
    at, k, v = torch.arange(128, dtype=torch.float64), k.double(), v.double()
    for count in (2, 3):
        after = torch.zeros_like(none)
        for h in range(2):
            decayed = (torch.exp(log[h].double() * (127 - at))[:, None] * k[:, h]).float().double()
            after[0, h] = sum(planes(decayed, count)).T @ v[:, h]
        # a head that forgets nothing needs one plane: its part of the state has no error
        share = share_of(after[:, :1], want["after"][0][:, :1], want["after"][1][:, :1])
        assert share >= 1.5 if count == 2 else share <= 0.5, share
