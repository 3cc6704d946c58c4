"""The gated feed-forward block and its gradients against the formulas in 64 bits (GPU), and the refusals.

The bounds follow the roundings: u = half the distance of neighbouring values of the stored type (2^-24 or 2^-8 relative),
for the result and for h, da and db, which are operands of further products; and the sums: n products of bfloat16 are added
16 at a time into FP32 that is cut off, 2^-23 a step; in float32 a sum starts anew every 128 values (8 steps for the large
products, and what the small ones and the planes leave out is below 8 units of 2^-24), and the partial sums are added; a few
rows are added up on the FP32 cores, 32 sums side by side."""
import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

from fastmd_b200 import _lib
from fastmd_b200.gated_feed_forward import gated_feed_forward

gpu = pytest.mark.gpu
F32, B16 = torch.float32, torch.bfloat16
E32 = 2.0 ** -24


def sums(n, dtype):
    """Units of sum |a||b| that a sum of n products may be off by."""
    return E32 * (n / 8 + 8 if dtype == B16 else 24 + n / 32)


def act_of(a, kind):
    if kind == "silu":
        s = torch.sigmoid(a)
        return a * s, s + a * s * (1 - s)
    s = torch.special.ndtr(a)
    return a * s, s + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)


def reference(x, wg, wu, wd, g, kind):
    """Results in 64 bits and their bounds."""
    dtype, unit = x.dtype, E32 if x.dtype == F32 else 2.0 ** -8
    x, wg, wu, wd, g = (t.detach().double() for t in (x, wg, wu, wd, g))
    rows, width, hidden, out = *x.shape, *wd.T.shape
    a, b = x @ wg.T, x @ wu.T
    ea, eb = sums(width, dtype) * (x.abs() @ wg.abs().T), sums(width, dtype) * (x.abs() @ wu.abs().T)
    level, slope = act_of(a, kind)
    # |act'| and |act''| are at most 1.13; the functions' own errors are 2^-19 of |a| + 1 (16 bits), 2^-21 (32)
    own = (a.abs() + 1) * (2.0 ** -19 if dtype == B16 else 2.0 ** -21)
    el, es = 1.13 * ea + own, 1.13 * ea + own
    h = level * b
    eh = el * b.abs() + (level.abs() + el) * eb + 2 * unit * h.abs()
    y = h @ wd.T
    want, err = {"y": y}, {"y": eh @ wd.abs().T + sums(hidden, dtype) * (h.abs() @ wd.abs().T)}
    dh = g @ wd
    edh = sums(out, dtype) * (g.abs() @ wd.abs())
    da, db = dh * b * slope, dh * level
    eda = edh * (b * slope).abs() + (dh.abs() + edh) * (eb * slope.abs() + (b.abs() + eb) * es) + 2 * unit * da.abs()
    edb = edh * level.abs() + (dh.abs() + edh) * el + 2 * unit * db.abs()
    want["dx"] = da @ wg + db @ wu
    err["dx"] = eda @ wg.abs() + edb @ wu.abs() + sums(2 * hidden, dtype) * (da.abs() @ wg.abs() + db.abs() @ wu.abs())
    want["dgate"], err["dgate"] = da.T @ x, eda.T @ x.abs() + sums(rows, dtype) * (da.abs().T @ x.abs())
    want["dup"], err["dup"] = db.T @ x, edb.T @ x.abs() + sums(rows, dtype) * (db.abs().T @ x.abs())
    want["ddown"], err["ddown"] = g.T @ h, g.abs().T @ eh + sums(rows, dtype) * (g.abs().T @ h.abs())
    for n in want:
        err[n] = err[n] * (1 + unit) + unit * want[n].abs()
    return want, err


def check(got, want, err, what, operands=0):
    assert got.shape == want.shape and bool(torch.isfinite(got).all()), what
    if not got.numel():
        return
    off = (got.double() - want).abs()
    assert bool((off <= err + 1e-30).all()), f"{what}: {float((off / (err + 1e-30)).amax()):.3g} times its bound"
    if got.dtype == B16 and got.numel() >= 4000:
        # Besides the result's own rounding one of each operand, independent and on average as large: sqrt 2 in all. The
        # second is a sum over n operands' roundings, whose values are products of three normal ones: the square of one
        # has 27 times the mean square as its own, so that their sum strays by sqrt(27 / n) of itself, and three times that
        # is allowed; and 3 % for the rest (factors in FP32, sums that are cut off).
        rounding = (want.to(B16).double() - want).norm()
        most = 1.03 * math.sqrt(2 + 3 * math.sqrt(27 / operands))
        assert float(off.norm()) <= most * float(rounding), f"{what}: {float(off.norm() / rounding):.3f} times its rounding"


def make(rows, width, hidden, out, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    normal = lambda *shape, scale: (torch.randn(*shape, generator=gen) * scale).to(dtype).cuda()  # noqa: E731
    return (normal(rows, width, scale=1.0), normal(hidden, width, scale=1.5 * width ** -0.5),
            normal(hidden, width, scale=width ** -0.5), normal(out, hidden, scale=hidden ** -0.5),
            normal(rows, out, scale=1.0))


def run_case(rows, width, hidden, out, dtype, kind, seed=0):
    *leaves, g = make(rows, width, hidden, out, dtype, seed)
    alone = gated_feed_forward(*leaves, activation=kind)
    leaves = [t.requires_grad_() for t in leaves]
    y = gated_feed_forward(*leaves, activation=kind)
    grads = torch.autograd.grad(y, leaves, g)
    want, err = reference(*leaves, g, kind)
    check(alone, want["y"], err["y"], "y without gradients", rows * hidden)
    check(y.detach(), want["y"], err["y"], "y", rows * hidden)
    for name, got in zip(("dx", "dgate", "dup", "ddown"), grads):
        check(got, want[name], err[name], name, rows * hidden)


SIZES = [
    (1, 8, 8, 8), (1, 1, 1, 1), (3, 5, 7, 2), (33, 64, 128, 64), (64, 256, 512, 256), (65, 72, 200, 72),
    (127, 128, 64, 136), (129, 130, 257, 131), (200, 264, 1000, 264), (300, 513, 129, 65), (1000, 256, 512, 256),
    (8, 1024, 2000, 512), (16, 768, 1111, 768), (2, 4096, 136, 8), (5000, 64, 80, 40),
]


@gpu
@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("rows,width,hidden,out", SIZES, ids=["x".join(map(str, s)) for s in SIZES])
def test_against_the_formulas(cuda, rows, width, hidden, out, dtype, kind):
    run_case(rows, width, hidden, out, dtype, kind, seed=rows + width)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_many_tiles(cuda, dtype):
    """More tiles than SMs in every product, with last ones that are nearly empty."""
    run_case(6145, 520, 2056, 776, dtype, "silu")


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_strides_and_shapes(cuda, dtype):
    """Views, transposed and offset tensors give the bits of contiguous ones; leading dimensions are kept."""
    x, wg, wu, wd, g = make(60, 40, 72, 24, dtype)
    want = gated_feed_forward(x, wg, wu, wd)
    wide = torch.full((60, 100), float("nan"), device="cuda", dtype=dtype)
    wide[:, 8:48] = x
    odd = torch.full((60 * 41 + 1,), float("nan"), device="cuda", dtype=dtype)[1:].view(60, 41)
    odd[:, :40] = x
    fused = torch.cat((wg, wu))
    for other in (wide[:, 8:48], odd[:, :40], x.T.contiguous().T):
        assert torch.equal(gated_feed_forward(other, fused[:72], fused[72:], wd.T.contiguous().T), want)
    assert torch.equal(gated_feed_forward(x.view(3, 20, 40), wg, wu, wd), want.view(3, 20, 24))
    assert torch.equal(gated_feed_forward(x[7], wg, wu, wd), gated_feed_forward(x[7:8], wg, wu, wd)[0])
    assert torch.equal(gated_feed_forward(x[:1].expand(9, 40), wg, wu, wd), want[:1].expand(9, 24))
    # gradients through copies and of broadcast rows
    leaf = odd.requires_grad_()
    (dodd,) = torch.autograd.grad(gated_feed_forward(leaf[:, :40], wg, wu, wd), leaf, g)
    x.requires_grad_()
    (dx,) = torch.autograd.grad(gated_feed_forward(x, wg, wu, wd), x, g)
    assert torch.equal(dodd[:, :40], dx) and not dodd[:, 40:].any()
    one = x.detach()[:1].clone().requires_grad_()
    (done,) = torch.autograd.grad(gated_feed_forward(one.expand(60, 40), wg, wu, wd), one, g)
    rows = one.detach().expand(60, 40).contiguous().requires_grad_()
    (each,) = torch.autograd.grad(gated_feed_forward(rows, wg, wu, wd), rows, g)
    assert torch.equal(done, each.sum(0, keepdim=True))


@gpu
def test_rows_of_odd_length(cuda):
    """bfloat16 rows that are copied first, transposed ones among them: the bits of padded storage, gradients of the tensors
    themselves, and no second derivatives either."""
    given = make(50, 37, 51, 29, B16)
    padded = [torch.zeros(t.shape[0], 64, device="cuda", dtype=B16)[:, :t.shape[1]].copy_(t) for t in given]
    turned = [t.T.contiguous().T for t in given]
    results = []
    for *leaves, g in (given, padded, turned):
        leaves = [t.detach().requires_grad_() for t in leaves]
        y = gated_feed_forward(*leaves)
        grads = torch.autograd.grad(y, leaves, g, retain_graph=True, create_graph=True)
        with pytest.raises(RuntimeError, match="first derivatives"):
            torch.autograd.grad(grads[0].float().square().sum(), leaves[0])
        results.append((y.detach(), gated_feed_forward(*(t.detach() for t in leaves)), *(x.detach() for x in grads)))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


class Elsewhere(torch.autograd.graph.saved_tensors_hooks):
    """Brings what is saved back in memory that starts one value further than a tensor of its own."""

    def __init__(self):
        super().__init__(lambda t: t.detach().cpu(), self.back)

    @staticmethod
    def back(t):
        return torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)[1:].view(t.shape).copy_(t)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
@pytest.mark.parametrize("width,hidden,out", [(67, 101, 67), (72, 136, 72), (1, 1, 1)])
def test_saved_tensors_that_come_back_otherwise(cuda, width, hidden, out, dtype):
    """Hooks that move what is saved (to the host and back) may give it other strides and another start: padded rows come back
    without their padding. The gradients are those of the tensors as they were, to the bit."""
    *leaves, g = make(90, width, hidden, out, dtype)
    views = [torch.zeros(t.shape[0], t.shape[1] + 16, device="cuda", dtype=dtype)[:, 8:8 + t.shape[1]].copy_(t) for t in leaves]
    for some in (leaves, views, [t.T.contiguous().T for t in leaves]):
        some = [t.detach().requires_grad_() for t in some]
        want = torch.autograd.grad(gated_feed_forward(*some), some, g)
        for hook in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True), Elsewhere()):
            with hook:
                y = gated_feed_forward(*some)
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, some, g), want))


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_gradients_on_their_own(cuda, dtype):
    """Each gradient asked for by itself has the bits that it has among all, on every run."""
    *leaves, g = make(700, 136, 320, 136, dtype)
    all_ = [t.requires_grad_() for t in leaves]
    want = torch.autograd.grad(gated_feed_forward(*all_), all_, g)
    again = torch.autograd.grad(gated_feed_forward(*all_), all_, g)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    for i in range(4):
        some = [t.detach().requires_grad_(i == j) for j, t in enumerate(leaves)]
        (got,) = torch.autograd.grad(gated_feed_forward(*some), some[i], g)
        assert torch.equal(got, want[i]), i


@gpu
def test_gradients_against_differences(cuda):
    *leaves, g = make(20, 24, 40, 16, F32)
    leaves = [t.requires_grad_() for t in leaves]
    grads = torch.autograd.grad(gated_feed_forward(*leaves, activation="gelu"), leaves, g)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for leaf, grad in zip(leaves, grads):
        way = torch.randn(leaf.shape, generator=gen, device="cuda")
        step = 2.0 ** -8
        ends = []
        for sign in (1, -1):
            args = [t.detach() + sign * step * way if t is leaf else t.detach() for t in leaves]
            ends.append((gated_feed_forward(*args, activation="gelu").double() * g).sum())
        got, want = float((ends[0] - ends[1]) / (2 * step)), float((grad * way).sum())
        # the third derivative times step^2 / 6, and 2^-20 of the sum's terms over the step
        assert abs(got - want) <= 1e-3 * (1 + abs(want)), (got, want)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_no_rows(cuda, dtype):
    *leaves, g = make(0, 24, 40, 16, dtype)
    leaves = [t.requires_grad_() for t in leaves]
    y = gated_feed_forward(*leaves)
    assert y.shape == (0, 16)
    dx, *dw = torch.autograd.grad(y, leaves, g)
    assert dx.shape == (0, 24) and not any(t.any() for t in dw)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_values_that_are_not_finite_stay_in_their_row(cuda, dtype):
    x, wg, wu, wd, g = make(300, 80, 136, 72, dtype)
    want = gated_feed_forward(x, wg, wu, wd)
    x[17, 3], x[130, 0], x[299] = float("nan"), float("inf"), -float("inf")
    y = gated_feed_forward(x.requires_grad_(), wg, wu, wd)
    (dx,) = torch.autograd.grad(y, x, g)
    bad = torch.zeros(300, dtype=torch.bool)
    bad[[17, 130, 299]] = True
    assert torch.equal(y[~bad], want[~bad]) and not torch.isfinite(y[bad]).any()
    assert torch.isfinite(dx[~bad]).all()


@gpu
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_an_infinite_weight_leaves_other_units_their_gradients(cuda, kind):
    """act(a) of one hidden unit is infinite in some rows, those of its neighbours small or beyond float16: bfloat16."""
    x, wg, wu, wd, g = make(40, 16, 32, 24, B16)
    x = x.abs() + 0.1
    wg[5] = wg[5].abs() * 1e5
    wg[6] = wg[6].abs() * 1e-2
    wg[7, 0] = float("inf")
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    (dup,) = torch.autograd.grad(gated_feed_forward(*leaves, activation=kind), leaves[2:3], g)
    others = [i for i in range(32) if i != 7]
    want, err = reference(x, wg[others], wu[others], wd[:, others], g, kind)
    check(dup[others], want["dup"], err["dup"], "dup", 40)


@gpu
@pytest.mark.parametrize("dtype", [F32, B16], ids=["f32", "b16"])
def test_arrays_past_32_bits(cuda, dtype):
    """More than 2^31 values of the hidden rows: the last rows of the result and their gradient."""
    hidden, tail = 8200, 200
    rows = 2 ** 31 // hidden + 1000
    x, wg, wu, wd, g = make(tail, 16, hidden, 16, dtype)
    many, more = (torch.zeros(rows, 16, device="cuda", dtype=dtype) for _ in range(2))
    many[-tail:], more[-tail:] = x, g
    want, err = reference(x, wg, wu, wd, g, "silu")
    leaves = [t.requires_grad_() for t in (many, wg, wu, wd)]
    y = gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, more)
    check(y.detach()[-tail:], want["y"], err["y"], "y", tail * hidden)
    check(grads[0][-tail:], want["dx"], err["dx"], "dx", tail * hidden)
    for name, got in zip(("dgate", "dup", "ddown"), grads[1:]):
        check(got, want[name], err[name], name, tail * hidden)
    assert not y[:-tail].any() and not grads[0][:-tail].any()
    del y, grads, got
    torch.cuda.empty_cache()


@gpu
def test_large_values(cuda):
    """Projections far beyond the activations' range, and finite values beyond the largest bfloat16."""
    for dtype in (F32, B16):
        x, wg, wu, wd, g = make(64, 64, 64, 64, dtype)
        for kind in ("silu", "gelu"):
            big = (x * 2.0 ** 40).requires_grad_()
            y = gated_feed_forward(big, wg, wu, wd, activation=kind)
            (dx,) = torch.autograd.grad(y, big, g)
            want, _ = reference(big, wg, wu, wd, g, kind)
            for got, ref in ((y.detach(), want["y"]), (dx, want["dx"])):
                assert float((got.double() - ref).norm()) <= (2.0 ** -7 if dtype == B16 else 2.0 ** -19) * float(ref.norm())
    top = torch.finfo(F32).max
    x = torch.zeros(2, 8, device="cuda")
    x[0, 0], x[1, 1] = top, -top
    eye = torch.eye(8, device="cuda")
    y = gated_feed_forward(x, eye * 2.0 ** -120, eye * 2.0 ** -124, eye)
    want = (x.double() * 2.0 ** -120).relu() * (x.double() * 2.0 ** -124)
    assert torch.isfinite(y).all() and float((y.double() - want).abs().max()) <= 2.0 ** -20 * float(want.abs().max())


@gpu
@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("rows", [4, 300])
def test_gates_far_below_zero(cuda, rows, kind):
    """act(a) and act'(a) for a in [-9, -5], where they are 10^-6 to 10^-18 (GELU): bfloat16 keeps their leading bits. One
    value of x reaches each projection, down is the identity and every unit has a gradient in one row, so that nothing is
    summed: y is h as it was rounded (2^-8 of itself), dup and dgate are db and da (2^-8, and 2^-11 of the factor they are
    multiplied by). The functions' own errors count 2^-16 (the exponent of e^{-a a / 2}, up to 58, has 24 bits; the rest is
    2^-20), and act' is a difference whose smaller part is a thirtieth of the other."""
    hidden, width = 512, 8
    gen = torch.Generator().manual_seed(rows)
    x = torch.zeros(rows, width)
    x[:, 0] = 1.0
    gate, up = torch.zeros(hidden, width), torch.zeros(hidden, width)
    gate[:, 0] = torch.linspace(-9, -5, hidden)
    up[:, 0] = torch.randn(hidden, generator=gen)
    g = torch.zeros(rows, hidden)
    unit = torch.arange(hidden)
    g[unit % rows, unit] = torch.randn(hidden, generator=gen)
    x, gate, up, down, g = (t.to(B16).cuda() for t in (x, gate, up, torch.eye(hidden), g))
    leaves = [t.requires_grad_() for t in (gate, up)]
    y = gated_feed_forward(x, gate, up, down, activation=kind)
    dgate, dup = torch.autograd.grad(y, leaves, g)
    a, b, own = gate.detach()[:, 0].double(), up.detach()[:, 0].double(), g.sum(0).double()
    share = torch.sigmoid(a) if kind == "silu" else 0.5 * torch.special.erfc(-a * math.sqrt(0.5))
    level = a * share
    slope = share + (level * (1 - share) if kind == "silu" else a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi))
    step, function, factor = 2.0 ** -8, 2.0 ** -16, 2.0 ** -11
    for name, got, want, most in (("y", y.detach(), (level * b).expand(rows, hidden), step + 2 * function),
                                  ("dup", dup[:, 0], own * level, step + factor + 2 * function),
                                  ("dgate", dgate[:, 0], own * b * slope, step + factor + 4 * function)):
        off = ((got.double() - want).abs() / want.abs()).amax()
        assert float(off) <= most * (1 + step), f"{name}: off by {float(off):.4f} of itself, {most:.4f} allowed"
    assert not dgate[:, 1:].any() and not dup[:, 1:].any()


@gpu
def test_captured_with_gradients(cuda):
    """Forward and backward in a graph, replayed on other values, two graphs with workspaces of their own."""
    *leaves, g = make(500, 136, 320, 136, B16)
    leaves = [t.requires_grad_() for t in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(gated_feed_forward(*leaves), leaves, g)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for kind in ("silu", "gelu"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = gated_feed_forward(*leaves, activation=kind)
            grads = torch.autograd.grad(y, leaves, g)
        graphs.append((graph, kind, y, grads))
    with torch.no_grad():
        leaves[0].mul_(-1.5)
        g.mul_(0.5)
    for graph, *_ in graphs:
        graph.replay()
    for _, kind, y, grads in graphs:
        eager = gated_feed_forward(*leaves, activation=kind)
        want = torch.autograd.grad(eager, leaves, g)
        assert torch.equal(y, eager) and all(torch.equal(a, b) for a, b in zip(grads, want))


@gpu
def test_two_streams_at_once(cuda):
    *leaves, g = make(2000, 264, 1000, 264, B16)
    leaves = [t.requires_grad_() for t in leaves]
    want = torch.autograd.grad(gated_feed_forward(*leaves), leaves, g)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(torch.autograd.grad(gated_feed_forward(*leaves), leaves, g))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for grads in got for a, b in zip(grads, want))


@gpu
def test_refusals(cuda):
    x, wg, wu, wd, g = make(8, 16, 24, 16, B16)
    for bad, text in (((x, wg, wu, wd.T), "down"), ((x[:, :8], wg, wu, wd), "width"), ((x, wg, wu[:8], wd), "up"),
                      ((x.float(), wg, wu, wd), "float32 or bfloat16"), ((x, wg, wu, wd.half()), "float32 or bfloat16"),
                      ((x[:, :0], wg[:, :0], wu[:, :0], wd), "between 1")):
        with pytest.raises(ValueError, match=text):
            gated_feed_forward(*bad)
    with pytest.raises(ValueError, match="activation"):
        gated_feed_forward(x, wg, wu, wd, activation="relu")
    x.requires_grad_()
    y = gated_feed_forward(x, wg, wu, wd)
    (dx,) = torch.autograd.grad(y, x, g, create_graph=True)
    with pytest.raises(RuntimeError, match="first derivatives only"):
        torch.autograd.grad(dx.float().sum(), x)
    with forward_ad.dual_level(), pytest.raises(RuntimeError):
        gated_feed_forward(forward_ad.make_dual(x.detach(), torch.ones_like(x)), wg, wu, wd)


def test_cpu_tensors_are_refused():
    w = torch.zeros(8, 8)
    with pytest.raises(_lib.FastMDLibraryError):
        gated_feed_forward(w, w, w, w)


def test_bad_arguments_of_the_entry_points_launch_nothing():
    lib, p = _lib.lib(), ctypes.c_void_p(1 << 20)
    kept, work, back = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()

    def problem(**change):
        sizes = dict(x=1 << 20, gate=1 << 20, up=1 << 20, down=1 << 20, rows=8, x_row=16, gate_row=16, up_row=16,
                     down_row=24, width=16, hidden=24, out=16, type=1, activation=0)
        return _lib.FmdFeedForward(**{**sizes, **change})

    def bytes_of(f, keep=0):
        return lib.fmd_gated_feed_forward_bytes(f, keep, kept, work, back)

    assert bytes_of(problem()) == 0 and kept.value >= 8 * 24 * 2
    assert bytes_of(problem(), 1) == 0 and kept.value >= 8 * 24 * 6 and back.value >= 8 * 24 * 4
    assert bytes_of(problem(type=0), 1) == 0 and kept.value >= 8 * 24 * 14 + 6 * (8 * 16 + 3 * 24 * 16)
    for change in (dict(type=2), dict(activation=2), dict(rows=-1), dict(width=0), dict(hidden=0), dict(out=0), dict(x=None),
                   dict(gate=None), dict(x_row=8), dict(down_row=16)):
        assert bytes_of(problem(**change)) == 1, change
    for change in (dict(x=(1 << 20) + 2), dict(x_row=17), dict(gate_row=20), dict(down_row=25), dict(rows=1 << 29)):
        assert bytes_of(problem(**change)) == 3, change
    assert bytes_of(problem(type=0, x=(1 << 20) + 4, x_row=17)) == 0  # float32: any rows
    assert bytes_of(problem(rows=0, x=None)) == 0
    f = problem()
    assert lib.fmd_gated_feed_forward(None, p, 0, p, 1 << 20, p, 1 << 20, None, None) == 1
    assert lib.fmd_gated_feed_forward(f, None, 0, p, 1 << 20, p, 1 << 20, None, None) == 1
    assert lib.fmd_gated_feed_forward(f, p, 0, p, 8, p, 1 << 20, None, None) == 4
    assert lib.fmd_gated_feed_forward(f, p, 0, None, 1 << 20, p, 1 << 20, None, None) == 4
    assert lib.fmd_gated_feed_forward(f, ctypes.c_void_p((1 << 20) + 8), 0, p, 1 << 20, p, 1 << 20, None, None) == 3
    assert lib.fmd_gated_feed_forward(problem(rows=0, x=None), None, 0, None, 0, None, 0, None, None) == 0
    assert lib.fmd_gated_feed_forward_bwd(f, p, 1 << 20, None, 16, p, p, p, p, p, 1 << 20, None, None) == 1
    assert lib.fmd_gated_feed_forward_bwd(f, p, 8, p, 16, p, p, p, p, p, 1 << 20, None, None) == 4
    assert lib.fmd_gated_feed_forward_bwd(f, p, 1 << 20, p, 16, p, p, p, p, p, 8, None, None) == 4
    assert lib.fmd_gated_feed_forward_bwd(f, p, 1 << 20, p, 17, p, p, p, p, p, 1 << 20, None, None) == 3
    one = dict(source=(1 << 20) + 2, to=1 << 20, rows=5, columns=17, from_row=17, from_column=1, to_row=24)

    def pad(count=1, **change):
        return lib.fmd_pad_rows((_lib.FmdPadded * 4)(_lib.FmdPadded(**{**one, **change})), count, None)

    assert lib.fmd_pad_rows(None, 1, None) == 1 and pad(0) == 1 and pad(5) == 1
    for change in (dict(rows=-1), dict(columns=0), dict(to_row=16), dict(to_row=25), dict(source=None), dict(to=None)):
        assert pad(**change) == 1, change
    assert pad(to=(1 << 20) + 8) == 3 and pad(rows=0, source=None, to=None) == 0
