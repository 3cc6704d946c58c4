"""The sequence operators that are measured, their plain forms and their values in 64 bits.

Two operators of a transformer that reads the rows of many replicas as packed sequences (the atoms of a structure,
or the frames that a trajectory has logged so far):

* ``rotary``: an RMS norm of each head of the queries and keys with the rotation of their positions, with its
  backward pass where the case trains;
* ``attention``: softmax attention over packed sequences with grouped heads, with its backward pass where the case
  trains (a force is a gradient too), and its form for a few new rows against a long cache.

A case fixes the sizes and the lengths of its sequences; ``prepare`` draws the values from the seed.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
#: bounds of a drawn case: the score matrix of the plain form, the products of one pass, the rows of one pass
MOST_SCORES, MOST_FLOPS, MOST_ROWS = 1.2e9, 3.0e11, 32_000


def listed():
    return [
        # one new frame of each of 64 replicas: the launch is all there is
        dict(name="rotary_step_bf16", op="rotary", type="bf16", rows=64, hq=8, hk=2, d=64, rot=64, interleaved=False,
             norm=True, train=False),
        # the 5,000 atoms of the large cell in the framework's own type, pairs side by side, half of each head turned
        dict(name="rotary_atoms_fp32", op="rotary", type="fp32", rows=5000, hq=8, hk=8, d=64, rot=32,
             interleaved=True, norm=True, train=True),
        # an odd number of rows with no norm: rotation alone
        dict(name="rotary_only_bf16", op="rotary", type="bf16", rows=10007, hq=12, hk=12, d=96, rot=96,
             interleaved=True, norm=False, train=False),
        # 64 replicas of 500 frames each, grouped heads: a training step
        dict(name="rotary_frames_bf16", op="rotary", type="bf16", rows=32000, hq=16, hk=4, d=128, rot=128,
             interleaved=False, norm=True, train=True),
        # one new frame of each of 64 replicas against its own history of 1 to 1,000 frames
        dict(name="step_bf16", op="attention", type="bf16", seqs=64, fresh=1, low=1, high=1000, hq=8, hk=2, d=64,
             causal=True, cache=True, train=False),
        # three long trajectories: few rows, a long axis of keys
        dict(name="step_long_bf16", op="attention", type="bf16", seqs=3, fresh=1, low=20000, high=60000, hq=32, hk=4,
             d=128, causal=True, cache=True, train=False),
        # a chunk of 33 new frames of 8 replicas behind histories of up to 5,000 frames
        dict(name="chunk_bf16", op="attention", type="bf16", seqs=8, fresh=33, low=500, high=5000, hq=16, hk=4, d=128,
             causal=True, cache=True, train=False),
        # 64 replicas of the 135-atom cell: every atom sees its own structure, energy and forces in the framework's type
        dict(name="atoms_fp32", op="attention", type="fp32", seqs=64, fresh=0, low=135, high=135, hq=4, hk=4, d=32,
             causal=False, cache=False, train=True),
        # the large cell of 5,000 atoms as one sequence, in the framework's type
        dict(name="cell_fp32", op="attention", type="fp32", seqs=1, fresh=0, low=5000, high=5000, hq=4, hk=4, d=64,
             causal=False, cache=False, train=True),
        # 64 replicas of the 135-atom cell in 16 bits
        dict(name="atoms_bf16", op="attention", type="bf16", seqs=64, fresh=0, low=135, high=135, hq=8, hk=8, d=64,
             causal=False, cache=False, train=True),
        # 16 trajectories of 100 to 2,000 frames, packed: a training step
        dict(name="frames_bf16", op="attention", type="bf16", seqs=16, fresh=0, low=100, high=2000, hq=16, hk=4,
             d=128, causal=True, cache=False, train=True),
        # a whole history of 10,000 frames read at once
        dict(name="history_bf16", op="attention", type="bf16", seqs=1, fresh=0, low=10000, high=10000, hq=16, hk=2,
             d=128, causal=True, cache=False, train=False),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind, d = rng.choice(("bf16", "bf16", "fp32")), rng.choice((32, 64, 96, 128))
    hk, group = rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 1, 2, 3, 4, 8))
    if rng.random() < 0.35:
        rot = rng.choice((d, d, d // 2))
        rows = max(1, min(spread(1, MOST_ROWS), int(MOST_ROWS * 20 * 128 / ((hk * group + hk) * d))))
        norm = rng.random() < 0.75
        return dict(op="rotary", type=kind, rows=rows, hq=hk * group, hk=hk, d=d, rot=rot,
                    interleaved=rng.random() < 0.5, norm=norm, train=rng.random() < 0.5)
    form = rng.choice(("step", "chunk", "whole", "train", "train"))
    seqs = spread(1, 64)
    high = spread(1, 60000 if form == "step" else 10000)
    fresh = {"step": 1, "chunk": spread(2, 300)}.get(form, 0)
    fresh = min(fresh, high)
    causal = form in ("step", "chunk") or rng.random() < 0.5
    while True:
        case = dict(op="attention", type=kind, seqs=seqs, fresh=fresh, low=max(1, fresh, high // rng.choice((1, 3, 20))),
                    high=high, hq=hk * group, hk=hk, d=d, causal=causal, cache=fresh > 0, train=form == "train")
        scores = seqs * hk * group * (fresh or high) * high
        keys = seqs * high * hk * d * 2
        flops = work(case)["flops"] * (4 if kind == "fp32" else 1)
        if scores <= MOST_SCORES and keys <= 2.5e8 and flops <= MOST_FLOPS:
            return case
        if seqs > 1:
            seqs = max(1, seqs * 2 // 3)
        else:
            high = max(1, high * 2 // 3)
            fresh = min(fresh, high)


def lengths(case):
    """Keys of each sequence: spread evenly over low..high in an order of no pattern; the first has the most."""
    n, low, high = case["seqs"], case["low"], case["high"]
    got = [high - (high - low) * i // max(1, n - 1) for i in range(n)]
    rest = got[1:]
    random.Random(n).shuffle(rest)
    return got[:1] + rest


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] == "rotary":
        values = case["rows"] * (case["hq"] + case["hk"]) * case["d"]
        table = case["rows"] * (case["rot"] * 4 + 8)
        # forward: in, out; backward: the gradient and, through the norm, the input again; the input's gradient
        moved = values * size * (2 + (3 if case["norm"] else 2) * case["train"])
        return {"bytes": moved + table, "flops": values * (6 + 12 * case["train"])}
    pairs = rows = keys = 0
    for n in lengths(case):
        m = min(case["fresh"], n) or n
        rows, keys = rows + m, keys + n
        pairs += m * n - (m * (m - 1) // 2 if case["causal"] else 0)
    hq, hk, d = case["hq"], case["hk"], case["d"]
    moved = size * d * (2 * rows * hq + 2 * keys * hk)
    flops = 4 * pairs * hq * d
    if case["train"]:  # the output's gradient in, three gradients out; five products for the forward's two
        moved += size * d * (2 * rows * hq + 2 * keys * hk)
        flops += 10 * pairs * hq * d
    return {"bytes": moved, "flops": flops}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(kind)

    hq, hk, d, train = case["hq"], case["hk"], case["d"], case["train"]
    if case["op"] == "rotary":
        rows, rot = case["rows"], case["rot"]
        # queries, keys and values leave one projection side by side
        fused = normal(rows, hq + 2 * hk, d, scale=1.5)
        state = dict(q=fused[:, :hq], k=fused[:, hq:hq + hk], train=train, interleaved=case["interleaved"], wq=None,
                     wk=None)
        state["positions"] = torch.randint(0, 10000, (rows,), generator=gen, device="cuda")
        turn = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        angle = torch.arange(10000, device="cuda", dtype=torch.float64)[:, None] * turn
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        if case["norm"]:
            state["wq"], state["wk"] = 1 + normal(d, scale=0.2), 1 + normal(d, scale=0.2)
        if train:
            state["gq"], state["gk"] = normal(rows, hq, d), normal(rows, hk, d)
            state["leaves"] = [t.requires_grad_() for t in (state["q"], state["k"], state["wq"], state["wk"])
                               if t is not None]
        return state
    count = lengths(case)
    fresh = [min(case["fresh"], n) or n for n in count]
    rows, slot = sum(fresh), case["high"]
    at = lambda sizes: torch.tensor([0] + sizes, device="cuda").cumsum(0)  # noqa: E731
    state = dict(offsets=at(fresh), key_offsets=None, key_counts=None, causal=case["causal"], train=train,
                 most_rows=max(fresh), most_keys=max(count))
    if case["cache"]:  # each sequence has a slot of its own in the caches, filled as far as its count
        state["q"] = normal(rows, hq + 2 * hk, d, scale=1.3)[:, :hq]
        state["k"], state["v"] = (normal(len(count) * slot, hk, d) for _ in range(2))
        state["key_offsets"] = at([slot] * len(count))
        state["key_counts"] = torch.tensor(count, device="cuda")
    else:
        fused = normal(rows, hq + 2 * hk, d, scale=1.2)
        state["q"], state["k"], state["v"] = fused.split((hq, hk, hk), 1)
    if train:
        state["g"] = normal(rows, hq, d)
        # the three that gradients are asked for, each with the strides of the projection
        state["leaves"] = [t.detach().requires_grad_() for t in (state["q"], state["k"], state["v"])]
        state["q"], state["k"], state["v"] = state["leaves"]
    return state


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _rotary(state) if "positions" in state else _attention(state)


def _run_own(state):
    from fastmd_b200 import head_rotary, packed_attention

    if "positions" in state:
        args = (state["q"], state["k"], state["positions"], state["cos"], state["sin"], state["wq"], state["wk"])
        q, k = head_rotary.head_norm_rotary(*args, interleaved=state["interleaved"])
        if not state["train"]:
            return q, k
        grads = torch.autograd.grad((q, k), state["leaves"], (state["gq"], state["gk"]))
        return (q.detach(), k.detach(), *grads)
    out = packed_attention.packed_attention(state["q"], state["k"], state["v"], state["offsets"],
                                            state["key_offsets"], state["key_counts"], causal=state["causal"])
    if not state["train"]:
        return out
    return (out.detach(), *torch.autograd.grad(out, state["leaves"], state["g"]))


# ------------------------------------------------------------ the plain forms: 32 bits, rounded once at the end

EPS = 1e-6


def _turn(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    a, b = (x[..., :rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _head(x, w, cos, sin, interleaved):
    y = x.float()
    if w is not None:
        y = y * (y.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.float()
    return _turn(y, cos, sin, interleaved).to(x.dtype)


def _head_grads(x, w, g, cos, sin, interleaved):
    y = _turn(g.float(), cos, -sin, interleaved)
    if w is None:
        return y.to(x.dtype), None
    r = (x.float().square().mean(-1, keepdim=True) + EPS).rsqrt()
    unit = x.float() * r
    dw = (y * unit).sum((0, 1))
    y = y * w.float()
    return (r * (y - unit * (y * unit).mean(-1, keepdim=True))).to(x.dtype), dw.to(w.dtype)


def _rotary(s):
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    out = (_head(s["q"], s["wq"], cos, sin, s["interleaved"]), _head(s["k"], s["wk"], cos, sin, s["interleaved"]))
    if not s["train"]:
        return out
    dq, dwq = _head_grads(s["q"], s["wq"], s["gq"], cos, sin, s["interleaved"])
    dk, dwk = _head_grads(s["k"], s["wk"], s["gk"], cos, sin, s["interleaved"])
    return (*out, dq, dk) if dwq is None else (*out, dq, dk, dwq, dwk)


def _padded(x, start, count, most, heads):
    """[sequences, heads, group * most, d] of the packed rows, zeros behind each sequence's end."""
    at = torch.arange(most, device=x.device)
    there = at < count[:, None]
    rows = (start[:, None] + at).clamp(max=x.shape[0] - 1)
    y = torch.where(there[..., None, None], x[rows].float(), 0.0)
    y = y.unflatten(2, (heads, -1)).permute(0, 2, 3, 1, 4)
    return y.flatten(2, 3)


def _packed(y, start, rows, group):
    """The rows of ``_padded`` back in their order."""
    y = y.unflatten(2, (group, -1))
    row = torch.arange(rows, device=y.device)
    seq = torch.searchsorted(start[1:], row, right=True)
    return y[seq, :, :, row - start[seq]].flatten(1, 2)


def _attention(s):
    q, k, v, start = s["q"], s["k"], s["v"], s["offsets"]
    hk, group, scale = k.shape[1], q.shape[1] // k.shape[1], q.shape[2] ** -0.5
    rows = start.diff()
    at, keys = (start[:-1], rows) if s["key_offsets"] is None else (s["key_offsets"][:-1], s["key_counts"])
    a = _padded(q, start[:-1], rows, s["most_rows"], hk)
    b, c = _padded(k, at, keys, s["most_keys"], hk), _padded(v, at, keys, s["most_keys"], hk)
    row, col = (torch.arange(n, device=q.device) for n in (s["most_rows"], s["most_keys"]))
    seen = (col < keys[:, None])[:, None, :].expand(-1, row.numel(), -1)
    if s["causal"]:
        seen = seen & (col <= row[:, None] + (keys - rows)[:, None, None])
    seen = seen[:, None, None]
    score = (a @ b.transpose(2, 3)).mul_(scale).unflatten(2, (group, -1))
    score.masked_fill_(~seen, -math.inf)
    peak = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = score.sub_(peak).exp_().flatten(2, 3)
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.0)
    o = p @ c
    out = _packed(o, start, q.shape[0], group).to(q.dtype)
    if not s["train"]:
        return out
    g = _padded(s["g"], start[:-1], rows, s["most_rows"], hk)
    dv = p.transpose(2, 3) @ g
    ds = (g @ c.transpose(2, 3)).sub_((g * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = ds @ b, ds.transpose(2, 3) @ a
    return (out, _packed(dq, start, q.shape[0], group).to(q.dtype), _packed(dk, start, k.shape[0], 1).to(k.dtype),
            _packed(dv, start, v.shape[0], 1).to(v.dtype))


# ------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    s = {n: t.detach() if isinstance(t, torch.Tensor) else t for n, t in s.items()}
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    group, scale = case["hq"] // case["hk"], 1 / math.sqrt(case["d"])
    q, k, v = (s[n].double() for n in "qkv")
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    row = key = 0
    for n in lengths(case):
        m = min(case["fresh"], n) or n
        for h in range(case["hq"]):
            qs, ks = (slice(row, row + m), h), (slice(key, key + n), h // group)
            score = scale * torch.einsum("id,jd->ij", q[qs], k[ks])
            if case["causal"]:
                score += torch.full((m, n), -math.inf, device="cuda", dtype=torch.float64).triu(n - m + 1)
            p = torch.softmax(score, 1)
            del score
            out[qs] = torch.einsum("ij,jd->id", p, v[ks])
            if case["train"]:
                g = s["g"][qs].double()
                dv[ks] += torch.einsum("ij,id->jd", p, g)
                dp = torch.einsum("id,jd->ij", g, v[ks])
                dp -= torch.einsum("ij,ij->i", p, dp)[:, None]
                dp *= p
                dq[qs] = scale * torch.einsum("ij,jd->id", dp, k[ks])
                dk[ks] += scale * torch.einsum("ij,id->jd", dp, q[qs])
        row, key = row + m, key + (case["high"] if case["cache"] else n)
    return (out, dq, dk, dv) if case["train"] else out


def _exact_rotary(case, s):
    d, rot = case["d"], case["rot"]
    half = torch.arange(rot // 2, device="cuda")
    first, second = (2 * half, 2 * half + 1) if case["interleaved"] else (half, half + rot // 2)
    c, n = (s[t].double()[s["positions"]][:, None] for t in ("cos", "sin"))

    def of(x, w, g):
        x = x.double()
        r = 1 / torch.sqrt(torch.einsum("thd,thd->th", x, x) / d + EPS)[..., None] if w is not None else 1.0
        u = x * r
        y = u * w.double() if w is not None else u
        out = y.clone()
        out[..., first] = y[..., first] * c - y[..., second] * n
        out[..., second] = y[..., first] * n + y[..., second] * c
        if g is None:
            return out, None, None
        back = g.double()
        one, two = back[..., first], back[..., second]
        back[..., first], back[..., second] = c * one + n * two, c * two - n * one
        if w is None:
            return out, back, None
        dw = torch.einsum("thd,thd->d", back, u)
        du = back * w.double()
        dx = r * du - x * r ** 3 * torch.einsum("thd,thd->th", du, x)[..., None] / d
        return out, dx, dw

    q, dq, dwq = of(s["q"], s["wq"], s.get("gq"))
    k, dk, dwk = of(s["k"], s["wk"], s.get("gk"))
    if not case["train"]:
        return q, k
    return (q, k, dq, dk) if dwq is None else (q, k, dq, dk, dwq, dwk)
