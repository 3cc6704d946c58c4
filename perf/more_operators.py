"""More operators of learned models that are measured, their plain forms and their values in 64 bits.

Two halves of a block that reads logs without an end, beside the attention that reads them whole:

* ``feed``: a gated feed-forward block, ``(act(x Wg^T) * (x Wu^T)) Wd^T``, with its backward pass where the case trains;
* ``decay``: linear attention over packed sequences with a decay for each head, whose state takes the place of a cache:
  whole sequences with their backward pass, chunks behind a state, and (``step``) one new row of each sequence.

A case fixes the sizes and the lengths of its sequences; ``prepare`` draws the values from the seed.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
#: bounds of a drawn case: products of one pass (float32: a fourth), values of q and bytes of the states of one pass
MOST_FLOPS, MOST_VALUES, MOST_STATE = 2.4e12, 1.2e8, 5.4e8


def listed():
    return [
        # one new frame of each of 64 replicas through the block of the frame model: the launches are all there is
        dict(name="feed_step_bf16", op="feed", type="bf16", rows=64, width=256, hidden=512, act="silu", train=False),
        # a few new frames through wide layers: the weights are read once and little else
        dict(name="feed_wide_bf16", op="feed", type="bf16", rows=8, width=4096, hidden=11000, act="silu", train=False),
        # a chunk of 33 new frames in the framework's own type, an odd hidden size
        dict(name="feed_chunk_fp32", op="feed", type="fp32", rows=33, width=512, hidden=1365, act="gelu", train=False),
        # 64 replicas of the 135-atom cell: a training step in the framework's own type
        dict(name="feed_atoms_fp32", op="feed", type="fp32", rows=8640, width=256, hidden=512, act="silu", train=True),
        # an odd number of rows, sizes that no tile divides
        dict(name="feed_ragged_bf16", op="feed", type="bf16", rows=10007, width=264, hidden=1000, act="gelu",
             train=True),
        # 64 replicas of 500 frames: a training step of a larger model
        dict(name="feed_frames_bf16", op="feed", type="bf16", rows=32000, width=1024, hidden=4096, act="silu",
             train=True),
        # one new frame of each of 64 replicas: the launch is all there is
        dict(name="step_bf16", op="decay", type="bf16", form="step", seqs=64, low=1, high=1, heads=8, dim=64,
             state=True, train=False),
        # one new frame of each of 512 replicas of a larger model: the states are read and written
        dict(name="step_many_fp32", op="decay", type="fp32", form="step", seqs=512, low=1, high=1, heads=16, dim=128,
             state=True, train=False),
        # a chunk of 33 new frames of 8 replicas behind their states
        dict(name="chunk_bf16", op="decay", type="bf16", form="rows", seqs=8, low=33, high=33, heads=16, dim=128,
             state=True, train=False),
        # 64 replicas of 100 to 500 frames: a training step in the framework's own type
        dict(name="frames_fp32", op="decay", type="fp32", form="rows", seqs=64, low=100, high=500, heads=8, dim=64,
             state=False, train=True),
        # 16 trajectories of 100 to 2,000 frames, packed: a training step
        dict(name="frames_bf16", op="decay", type="bf16", form="rows", seqs=16, low=100, high=2000, heads=16, dim=128,
             state=False, train=True),
        # a whole history of 50,000 frames read at once, and its state kept
        dict(name="history_bf16", op="decay", type="bf16", form="rows", seqs=1, low=50000, high=50000, heads=16,
             dim=128, state=True, train=False),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind, train = rng.choice(("bf16", "bf16", "fp32")), rng.random() < 0.5
    if rng.random() < 0.5:
        odd = rng.random() < 0.3
        while True:
            width, hidden = spread(64, 4096), spread(64, 11264)
            if not odd:
                width, hidden = (width + 7) // 8 * 8, (hidden + 7) // 8 * 8
            case = dict(op="feed", type=kind, rows=spread(1, 32000), width=width, hidden=hidden,
                        act=rng.choice(("silu", "gelu")), train=train)
            if work(case)["flops"] * (4 if kind == "fp32" else 1) <= MOST_FLOPS:
                return case
    step = rng.random() < 0.3
    heads, dim = rng.choice((1, 2, 3, 4, 8, 16, 32)), rng.choice((32, 64, 64, 96, 128, 128, 8 * rng.randint(1, 16)))
    while True:
        seqs = spread(1, 512 if step else 64)
        high = 1 if step else spread(1, 50000)
        low = high if step else high // rng.choice((1, 3, 20, high + 1))
        case = dict(op="decay", type=kind, form="step" if step else "rows", seqs=seqs, low=low, high=high, heads=heads,
                    dim=dim, state=step or rng.random() < 0.5, train=train and not step)
        values = sum(lengths(case)) * heads * dim * (4 if train else 1) * (2 if kind == "fp32" else 1)
        if values <= MOST_VALUES and seqs * heads * dim * dim * 4 <= MOST_STATE and seqs * high <= 200_000:
            return case


def lengths(case):
    """Rows of each sequence: spread evenly over low..high in an order of no pattern; the first has the most."""
    n, low, high = case["seqs"], case["low"], case["high"]
    got = [high - (high - low) * i // max(1, n - 1) for i in range(n)]
    rest = got[1:]
    random.Random(n).shuffle(rest)
    return got[:1] + rest


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] == "feed":
        rows, width, hidden, train = case["rows"], case["width"], case["hidden"], case["train"]
        # rows in and out, the weights; backward: the output's gradient in, all gradients out
        moved = size * (2 * rows * width + 3 * width * hidden) * (2 if train else 1)
        return {"bytes": moved, "flops": 6 * rows * width * hidden * (3 if train else 1)}
    rows, heads, dim = sum(lengths(case)), case["heads"], case["dim"]
    values, states = rows * heads * dim, case["seqs"] * heads * dim * dim * 4
    # q, k, v in and the output out; backward: the output's gradient in, three gradients out (q, k, v stay)
    moved = values * size * (8 if case["train"] else 4) + case["state"] * states * (4 if case["train"] else 2)
    # by the recurrence: the state's update and what a row reads of it; each of q, k, v takes the same again
    return {"bytes": moved, "flops": 4 * values * dim * (4 if case["train"] else 1)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(kind)

    if case["op"] == "feed":
        rows, width, hidden = case["rows"], case["width"], case["hidden"]
        state = dict(op="feed", act=case["act"], train=case["train"], x=normal(rows, width),
                     w_gate=normal(hidden, width, scale=1.5 * width ** -0.5),
                     w_up=normal(hidden, width, scale=width ** -0.5),
                     w_down=normal(width, hidden, scale=hidden ** -0.5))
        if case["train"]:
            state["g"] = normal(rows, width)
            state["leaves"] = [state[n].requires_grad_() for n in ("x", "w_gate", "w_up", "w_down")]
        return state
    seqs, heads, dim, count = case["seqs"], case["heads"], case["dim"], lengths(case)
    fused = normal(sum(count), 3 * heads, dim)  # queries, keys and values leave one projection side by side
    state = dict(op="decay", step=case["form"] == "step", train=case["train"], longest=max(count),
                 offsets=torch.tensor([0] + count, device="cuda").cumsum(0), state=None, gstate=None)
    state["q"], state["k"], state["v"] = fused.split(heads, 1)
    # half-lives from one row to some hundreds, as many heads for each power of two
    place = (torch.arange(heads, device="cuda", dtype=torch.float64) + 0.5) / heads
    state["log_decay"] = torch.log1p(-(2.0 ** (-1 - 8 * place))).float()
    if case["state"]:
        state["state"] = torch.randn(seqs, heads, dim, dim, generator=gen, device="cuda")
    if case["train"]:
        state["g"] = normal(sum(count), heads, dim)
        state["leaves"] = [t.detach().requires_grad_() for t in (state["q"], state["k"], state["v"])]
        state["q"], state["k"], state["v"] = state["leaves"]
        if case["state"]:
            state["leaves"].append(state["state"].requires_grad_())
            state["gstate"] = torch.randn(seqs, heads, dim, dim, generator=gen, device="cuda")
    return state


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _feed(state) if state["op"] == "feed" else _step(state) if state["step"] else _decay(state)


def _run_own(s):
    from fastmd_b200 import decay_attention, gated_feed_forward

    if s["op"] == "feed":
        y = gated_feed_forward.gated_feed_forward(s["x"], s["w_gate"], s["w_up"], s["w_down"], activation=s["act"])
        return (y.detach(), *torch.autograd.grad(y, s["leaves"], s["g"])) if s["train"] else y
    if s["step"]:  # the state is the caller's and moves on in place
        out = decay_attention.decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"])
        return out, s["state"]
    keep = s["state"] is not None
    out = decay_attention.decay_attention(s["q"], s["k"], s["v"], s["log_decay"], s["offsets"], s["state"],
                                          return_state=keep)
    if not s["train"]:
        return out
    if not keep:
        return (out.detach(), *torch.autograd.grad(out, s["leaves"], s["g"]))
    out, after = out
    return (out.detach(), after.detach(), *torch.autograd.grad((out, after), s["leaves"], (s["g"], s["gstate"])))


# ------------------------------------------------------------ the plain forms: 32 bits, rounded once at the end

def _feed(s):
    kind = s["x"].dtype
    x, wg, wu, wd = (s[n].float() for n in ("x", "w_gate", "w_up", "w_down"))
    a, b = x @ wg.T, x @ wu.T
    if s["act"] == "silu":
        turn = 1 / (1 + (-a).exp())
        slope = turn * (1 + a * (1 - turn))
    else:
        turn = 0.5 * (1 + torch.erf(a * math.sqrt(0.5)))
        slope = turn + a * (-0.5 * a.square()).exp() * (1 / math.sqrt(2 * math.pi))
    act = a * turn
    h = act * b
    y = (h @ wd.T).to(kind)
    if not s["train"]:
        return y
    g = s["g"].float()
    dh = g @ wd
    da, db = dh * b * slope, dh * act
    return (y, (da @ wg + db @ wu).to(kind), (da.T @ x).to(kind), (db.T @ x).to(kind), (g.T @ h).to(kind))


def _step(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    now = s["state"]
    now.mul_(s["log_decay"].exp()[:, None, None]).add_(k[..., :, None] * v[..., None, :])
    out = (q[..., None, :] @ now)[..., 0, :] * q.shape[-1] ** -0.5
    return out.to(s["q"].dtype), now


CHUNK = 128


def _padded(x, start, count, most):
    """[sequences, heads, most, dim] of the packed rows, zeros behind each sequence's end."""
    at = torch.arange(most, device=x.device)
    rows = (start[:-1, None] + at).clamp(max=max(0, x.shape[0] - 1))
    return torch.where((at < count[:, None])[..., None, None], x[rows].float(), 0.0).transpose(1, 2)


def _mixed(a, b, c, log, later=False):
    """out_t = sum_s e^{log |t - s|} (a_t . b_s) c_s over s <= t, or with ``later`` s >= t: inside chunks pair by pair,
    from chunk to chunk by what each adds to the matrix that the next ones read. The rows are a multiple of CHUNK."""
    x, y, z = (t.unflatten(2, (-1, CHUNK)) for t in (a, b, c))
    log = log[:, None, None]

    def weights(gap, unit):  # e^{log gap}, nothing where the gap is below zero
        return torch.where(gap >= 0, (gap.clamp(min=0) * unit * log).exp(), 0.0)

    i, n = torch.arange(CHUNK, device=a.device), torch.arange(x.shape[2], device=a.device)
    gap, chunks = i[:, None] - i, n[:, None] - n - 1
    if later:
        gap, chunks = gap.T, chunks.T
    since, until = (CHUNK - i, i) if later else (i + 1, CHUNK - 1 - i)
    near = ((x @ y.transpose(3, 4)) * weights(gap, 1)[:, None]) @ z
    added = (weights(until[:, None], 1)[:, None] * y).transpose(3, 4) @ z
    matrix = (weights(chunks, CHUNK) @ added.flatten(3)).unflatten(3, added.shape[3:])
    return (near + weights(since[:, None], 1)[:, None] * (x @ matrix)).flatten(2, 3)


def _decay(s):
    q, k, v, start, log = s["q"], s["k"], s["v"], s["offsets"], s["log_decay"]
    count, kind, scale = start.diff(), q.dtype, q.shape[-1] ** -0.5
    row = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(start[1:], row, right=True)
    packed = lambda t: t.transpose(1, 2)[seq, row - start[seq]].to(kind)  # noqa: E731
    most = max(1, -(-s["longest"] // CHUNK)) * CHUNK
    a, b, c = (_padded(t, start, count, most) for t in (q, k, v))
    at, n = torch.arange(most, device=q.device), count[:, None, None]
    before = ((at + 1) * log[:, None]).exp()[..., None]  # of the state at the start, as row t reads it
    behind = torch.where(at < n, ((n - 1 - at).clamp(min=0) * log[:, None]).exp(), 0.0)[..., None]
    first, whole = s["state"], (count[:, None] * log).exp()[..., None, None]
    out, after = _mixed(a, b, c, log), (behind * b).transpose(2, 3) @ c
    if first is not None:
        out += before * (a @ first)
        after += whole * first
    out = packed(out * scale)
    if not s["train"]:
        return out if first is None else (out, after)
    g = _padded(s["g"], start, count, most) * scale
    dq, dk, dv = _mixed(g, c, b, log), _mixed(c, g, a, log, later=True), _mixed(b, a, g, log, later=True)
    if first is None:
        return out, packed(dq), packed(dk), packed(dv)
    gs = s["gstate"]
    dq += before * (g @ first.transpose(2, 3))
    dk += behind * (c @ gs.transpose(2, 3))
    dv += behind * (b @ gs)
    dfirst = whole * gs + (before * a).transpose(2, 3) @ g
    return out, after, packed(dq), packed(dk), packed(dv), dfirst


# ------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    s = {n: t.detach().double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t for n, t in s.items()}
    if case["op"] == "feed":
        return _exact_feed(case, s)
    return _exact_decay(case, s)


def _exact_feed(case, s):
    x, wg, wu, wd = s["x"], s["w_gate"], s["w_up"], s["w_down"]
    a, b = torch.einsum("rk,nk->rn", x, wg), torch.einsum("rk,nk->rn", x, wu)
    if case["act"] == "silu":
        act = a * torch.sigmoid(a)
        slope = torch.sigmoid(a) + act * torch.sigmoid(-a)
    else:
        share = torch.special.ndtr(a)
        act = a * share
        slope = share + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    y = torch.einsum("rn,kn->rk", act * b, wd)
    if not case["train"]:
        return y
    dwd = torch.einsum("rk,rn->kn", s["g"], act * b)
    dh = torch.einsum("rk,kn->rn", s["g"], wd)
    da, db = dh * b * slope, dh * act
    dx = torch.einsum("rn,nk->rk", da, wg) + torch.einsum("rn,nk->rk", db, wu)
    return y, dx, torch.einsum("rn,rk->nk", da, x), torch.einsum("rn,rk->nk", db, x), dwd


def _exact_decay(case, s):
    """Every pair of rows by itself, a block of rows at a time."""
    q, k, v, log, scale = s["q"], s["k"], s["v"], s["log_decay"], 1 / math.sqrt(case["dim"])
    heads, dim = case["heads"], case["dim"]
    out, dq, dk, dv = (torch.zeros_like(q) for _ in range(4))
    first = s["state"] if case["state"] else q.new_zeros(case["seqs"], heads, dim, dim)
    after, dfirst = torch.zeros_like(first), torch.zeros_like(first)
    row, block = 0, 1000
    for i, n in enumerate(lengths(case)):
        t = torch.arange(n, device=q.device, dtype=torch.float64)
        for h in range(heads):
            here = (slice(row, row + n), h)
            x, y, z = q[here], k[here], v[here]
            since, until = torch.exp(log[h] * (t + 1))[:, None], torch.exp(log[h] * (n - 1 - t))[:, None]
            after[i, h] = torch.exp(log[h] * n) * first[i, h] + torch.einsum("ta,tb->ab", until * y, z)
            if case["train"]:
                g = s["g"][here] * scale
                dq[here] = since * torch.einsum("tb,ab->ta", g, first[i, h])
                dfirst[i, h] = torch.einsum("ta,tb->ab", since * x, g)
                if case["state"]:
                    dk[here] = until * torch.einsum("tb,ab->ta", z, s["gstate"][i, h])
                    dv[here] = until * torch.einsum("ta,ab->tb", y, s["gstate"][i, h])
                    dfirst[i, h] += torch.exp(log[h] * n) * s["gstate"][i, h]
            for low in range(0, n, block):
                high = min(n, low + block)
                mine, all_ = slice(low, high), slice(0, high)
                weight = torch.exp(log[h] * (t[mine, None] - t[None, all_])).tril(low)
                score = torch.einsum("ta,sa->ts", x[mine], y[all_]) * weight
                out[row + low:row + high, h] = scale * (torch.einsum("ts,sb->tb", score, z[all_])
                                                        + since[mine] * torch.einsum("ta,ab->tb", x[mine], first[i, h]))
                if not case["train"]:
                    continue
                dv[row:row + high, h] += torch.einsum("ts,tb->sb", score, g[mine])
                weight *= torch.einsum("tb,sb->ts", g[mine], z[all_])
                dq[row + low:row + high, h] += torch.einsum("ts,sa->ta", weight, y[all_])
                dk[row:row + high, h] += torch.einsum("ts,ta->sa", weight, x[mine])
        row += n
    if not case["train"]:
        return (out, after) if case["state"] else out
    return (out, after, dq, dk, dv, dfirst) if case["state"] else (out, dq, dk, dv)
