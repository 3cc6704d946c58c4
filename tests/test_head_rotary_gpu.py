"""Norm and rotation of query and key heads against the formulas in 64 bits (GPU), and the table (CPU)."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from fastmd_b200 import _lib, head_rotary
from fastmd_b200.head_rotary import head_norm_rotary, rotary_table

gpu = pytest.mark.gpu


def turn64(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    a, b = (x[..., :rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def head64(x, w, cos, sin, interleaved, eps):
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    return turn64(x, cos.double()[:, None], sin.double()[:, None], interleaved)


def make(rows, hq, hk, dim, rot, dtype, norm, seed=0, weight_dtype=None, length=5000):
    gen = torch.Generator().manual_seed(seed)
    fused = torch.randn(rows, hq + 2 * hk, dim, generator=gen).to(dtype).cuda()
    positions = torch.randint(0, length, (rows,), generator=gen).cuda()
    cos, sin = rotary_table(length, rot, device="cuda")
    weights = [None, None]
    if norm:
        weights = [(1 + 0.3 * torch.randn(dim, generator=gen)).to(weight_dtype or dtype).cuda() for _ in range(2)]
    return fused[:, :hq], fused[:, hq:hq + hk], positions, cos, sin, weights


def unit(dtype):  # half the distance of neighbouring values, relative
    return 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8


CASES = [
    # rows, hq, hk, dim, rot, dtype, norm, interleaved
    (1, 1, 1, 8, 8, torch.float32, True, False),
    (1, 8, 2, 64, 64, torch.bfloat16, True, False),
    (7, 3, 1, 96, 48, torch.bfloat16, True, False),
    (7, 3, 1, 96, 24, torch.bfloat16, True, False),  # half of 12: four values a lane
    (33, 5, 5, 40, 40, torch.bfloat16, True, True),
    (130, 16, 4, 128, 128, torch.bfloat16, True, False),
    (130, 16, 4, 128, 64, torch.float32, True, True),
    (61, 12, 12, 96, 96, torch.float32, False, False),
    (61, 12, 2, 72, 8, torch.bfloat16, False, True),
    (257, 9, 3, 32, 32, torch.float32, True, False),
]


@gpu
@pytest.mark.parametrize("rows,hq,hk,dim,rot,dtype,norm,interleaved", CASES)
def test_forward_and_gradients(cuda, rows, hq, hk, dim, rot, dtype, norm, interleaved):
    q, k, positions, cos, sin, (wq, wk) = make(rows, hq, hk, dim, rot, dtype, norm)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk) if t is not None]
    args = leaves if norm else leaves + [None, None]
    out = head_norm_rotary(args[0], args[1], positions, cos, sin, args[2], args[3], interleaved=interleaved)
    gen = torch.Generator().manual_seed(1)
    g = [torch.randn(o.shape, generator=gen).to(dtype).cuda() for o in out]
    grads = torch.autograd.grad(out, leaves, g)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    wargs = wide if norm else wide + [None, None]
    ref = [head64(x, w, cos[positions], sin[positions], interleaved, 1e-6)
           for x, w in ((wargs[0], wargs[2]), (wargs[1], wargs[3]))]
    ref_grads = torch.autograd.grad(ref, wide, [t.double() for t in g])
    # one rounding of the stored value, and about ten FP32 roundings of terms as large as a head's largest value
    for got, want in zip(list(out) + list(grads[:2]), list(ref) + list(ref_grads[:2])):
        bound = unit(dtype) * want.abs() + 16 * 2.0 ** -24 * (want.abs().amax(-1, keepdim=True) + 1)
        assert bool(((got.double() - want).abs() <= bound).all())
    # a weight's gradient adds rows * heads terms in FP32: n roundings of partial sums no larger than the sum of |terms|
    for got, want, x, gx in zip(grads[2:], ref_grads[2:], wide[:2], g):
        terms = rows * x.shape[1]
        size = 3.0 * math.sqrt(dim) * gx.double().abs().amax()  # |u| is at most sqrt(dim), a turn keeps lengths
        bound = unit(dtype) * want.abs() + 2.0 ** -24 * min(terms, 64) * terms * size
        assert bool(((got.double() - want).abs() <= bound).all())


@gpu
def test_gradient_against_differences(cuda):
    """The directional derivative of sum(q' c) by central differences of the operator itself: FP32 values, a step
    of 2^-7, so a truncation of about h^2 / 6 of third derivatives of size one and a rounding of 2^-24 / h each."""
    q, k, positions, cos, sin, (wq, wk) = make(5, 2, 1, 16, 16, torch.float32, True, seed=3)
    gen = torch.Generator().manual_seed(4)
    c = torch.randn(5, 2, 16, generator=gen).cuda()
    dirs = [torch.randn(t.shape, generator=gen).cuda() for t in (q, wq)]
    leaves = [q.clone().requires_grad_(), wq.clone().requires_grad_()]
    out, _ = head_norm_rotary(leaves[0], k, positions, cos, sin, leaves[1], wk)
    grads = torch.autograd.grad((out * c).sum(), leaves)
    h = 2.0 ** -7

    def value(sign, which):
        args = [q.clone(), wq.clone()]
        args[which] = args[which] + sign * h * dirs[which]
        o, _ = head_norm_rotary(args[0], k, positions, cos, sin, args[1], wk)
        return float((o.double() * c.double()).sum())

    for which in range(2):
        slope = (value(1, which) - value(-1, which)) / (2 * h)
        want = float((grads[which].double() * dirs[which].double()).sum())
        size = float(dirs[which].abs().sum() * c.abs().max()) + abs(want)
        assert abs(slope - want) <= 2.0 ** -9 * size


@gpu
def test_mixed_weight_type_and_one_side(cuda):
    q, k, positions, cos, sin, (wq, _) = make(19, 4, 2, 64, 32, torch.bfloat16, True, weight_dtype=torch.float32)
    wq = wq.requires_grad_()
    qo, ko = head_norm_rotary(q, k, positions, cos, sin, wq, None)
    want = head64(q, wq.detach(), cos[positions], sin[positions], False, 1e-6)
    assert bool(((qo.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all())
    want = head64(k, None, cos[positions], sin[positions], False, 1e-6)
    assert bool(((ko.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all())
    (dw,) = torch.autograd.grad(qo.float().sum(), wq)  # only the queries' side runs backward
    assert dw.dtype == torch.float32 and bool(torch.isfinite(dw).all())


@gpu
def test_layouts_are_the_packed_ones(cuda):
    """Other strides, an unaligned base and a transposed head order give the bits of the packed tensor."""
    q, k, positions, cos, sin, (wq, wk) = make(21, 6, 2, 32, 32, torch.bfloat16, True)
    want = head_norm_rotary(q.contiguous(), k.contiguous(), positions, cos, sin, wq, wk)
    flat = torch.empty(21 * 6 * 32 + 1, device="cuda", dtype=q.dtype)
    flat[1:] = q.reshape(-1)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    for other in (flat[1:].view(21, 6, 32), turned, q.transpose(1, 2).contiguous().transpose(1, 2)):
        got = head_norm_rotary(other, k, positions, cos, sin, wq, wk)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
def test_repeatable_and_empty(cuda):
    q, k, positions, cos, sin, (wq, wk) = make(3001, 4, 4, 64, 64, torch.bfloat16, True)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    runs = []
    for _ in range(2):
        out = head_norm_rotary(leaves[0], leaves[1], positions, cos, sin, *leaves[2:])
        runs.append(torch.autograd.grad(sum(o.float().square().sum() for o in out), leaves))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    leaves = [q[:0].detach().requires_grad_(), k[:0].detach().requires_grad_(), *leaves[2:]]
    out = head_norm_rotary(leaves[0], leaves[1], positions[:0], cos, sin, *leaves[2:])
    grads = torch.autograd.grad(sum(o.float().sum() for o in out), leaves)
    assert out[0].shape == (0, 4, 64) and grads[0].shape == (0, 4, 64)
    assert not grads[2].any() and not grads[3].any()


@gpu
def test_position_outside_the_table_is_flagged(cuda):
    q, k, positions, cos, sin, _ = make(4, 2, 1, 16, 8, torch.float32, False, length=50)
    positions[2], positions[3] = 50, -1
    word = _lib.flags_word(q.device)
    word.zero_()
    qo, _ = head_norm_rotary(q, k, positions, cos, sin)
    assert int(word.item()) & 1
    word.zero_()
    assert not qo[2:, :, :8].any() and torch.equal(qo[2:, :, 8:], q[2:, :, 8:])


@gpu
def test_refusals(cuda):
    q, k, positions, cos, sin, (wq, wk) = make(4, 2, 1, 16, 16, torch.float32, True)
    with pytest.raises(_lib.FastMDLibraryError):
        head_norm_rotary(q.cpu(), k, positions, cos, sin)
    for bad in (dict(q=q.half(), k=k.half()), dict(q=q.bfloat16()), dict(q=q[:3]), dict(q=q[..., :12], k=k[..., :12]),
                dict(positions=positions.int()), dict(positions=positions[:2]), dict(cos=cos.double()),
                dict(cos=cos[:, :4]), dict(cos=cos[:, :2], sin=sin[:, :2]), dict(q_weight=wq[:8]),
                dict(q_weight=wq.half()), dict(q=q.reshape(4, 32))):
        args = dict(q=q, k=k, positions=positions, cos=cos, sin=sin, q_weight=wq, k_weight=wk) | bad
        with pytest.raises(ValueError):
            head_norm_rotary(**args)


def test_table_on_the_host():
    cos, sin = rotary_table(9, 8, base=100.0)
    want = torch.tensor([[p * 100.0 ** (-2 * i / 8) for i in range(4)] for p in range(9)], dtype=torch.float64)
    assert torch.equal(cos, want.cos().float()) and torch.equal(sin, want.sin().float())
    cos, _ = rotary_table(9, 8, base=100.0, factor=4.0, amplitude=0.5)
    assert torch.allclose(cos.double(), 0.5 * (want / 4).cos(), atol=1e-7)
    # over 60 steps pair 0 turns 9.5 times (kept above 8), pair 3 turns 0.3 times (divided)
    cos, _ = rotary_table(9, 8, base=100.0, factor=4.0, trained_length=60, turns=(1.0, 8.0))
    assert torch.allclose(cos[:, 0].double(), want[:, 0].cos(), atol=1e-7)
    assert torch.allclose(cos[:, 3].double(), (want[:, 3] / 4).cos(), atol=1e-7)
    turns = 60 * 100.0 ** -0.25 / (2 * math.pi)
    kept = (turns - 1) / 7
    assert torch.allclose(cos[:, 1].double(), (want[:, 1] * (kept + (1 - kept) / 4)).cos(), atol=1e-7)
    for bad in (dict(length=-1, rotary_dim=8), dict(length=2, rotary_dim=7), dict(length=2, rotary_dim=8, factor=0.0)):
        with pytest.raises(ValueError):
            rotary_table(**bad)


def test_abi_refuses_on_the_host():
    lib = _lib.lib()
    sides = (_lib.FmdHeadRotarySide * 2)()
    args = [sides, 0, 0, 0, 64, 64, 0, 1e-6, None, None, None, 0, 0, None, 0, None, None]
    assert lib.fmd_head_rotary(*args) == 0  # no rows: nothing to do
    for at, value in ((1, 7), (2, 1), (4, 12), (4, 136), (5, 72), (5, 4), (3, -1)):
        bad = list(args)
        bad[at] = value
        assert lib.fmd_head_rotary(*bad) == 1
    sides[0].w, sides[0].heads = 1 << 20, 1
    args[12] = 1
    assert lib.fmd_head_rotary(*args) == 4  # the backward pass with weights needs its workspace
    assert head_rotary.TYPES[torch.float32] == 0


@gpu
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("rows,hq,hk,dim,dtype", [(7, 3, 1, 96, torch.bfloat16), (13, 5, 6, 64, torch.float32),
                                                  (1, 3, 3, 32, torch.float32), (33, 1, 7, 48, torch.bfloat16)])
def test_gradients_without_an_eps(cuda, rows, hq, hk, dim, dtype, interleaved):
    """eps = 0: the lanes without a head or a row, which divide nothing by nothing, have no share in the sums. The
    bounds are those of test_forward_and_gradients: eps does not add a rounding."""
    q, k, positions, cos, sin, (wq, wk) = make(rows, hq, hk, dim, dim, dtype, True, seed=rows)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    out = head_norm_rotary(*leaves[:2], positions, cos, sin, *leaves[2:], eps=0.0, interleaved=interleaved)
    gen = torch.Generator().manual_seed(1)
    g = [torch.randn(o.shape, generator=gen).to(dtype).cuda() for o in out]
    grads = torch.autograd.grad(out, leaves, g)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    ref = [head64(x, w, cos[positions], sin[positions], interleaved, 0.0) for x, w in zip(wide[:2], wide[2:])]
    ref_grads = torch.autograd.grad(ref, wide, [t.double() for t in g])
    for got, want in zip(list(out) + list(grads[:2]), list(ref) + list(ref_grads[:2])):
        bound = unit(dtype) * want.abs() + 16 * 2.0 ** -24 * (want.abs().amax(-1, keepdim=True) + 1)
        assert bool(((got.double() - want).abs() <= bound).all())
    for got, want, x, gx in zip(grads[2:], ref_grads[2:], wide[:2], g):
        terms = rows * x.shape[1]
        size = 3.0 * math.sqrt(dim) * gx.double().abs().amax()
        bound = unit(dtype) * want.abs() + 2.0 ** -24 * min(terms, 64) * terms * size
        assert bool(((got.double() - want).abs() <= bound).all())


@gpu
@pytest.mark.parametrize("eps", [-1e-6, float("nan"), float("inf"), 1e39])
def test_an_eps_that_is_none_is_refused(cuda, eps):
    q, k, positions, cos, sin, (wq, wk) = make(4, 2, 1, 16, 16, torch.float32, True)
    with pytest.raises(ValueError):
        head_norm_rotary(q, k, positions, cos, sin, wq, wk, eps=eps)


@pytest.mark.parametrize("eps", [-1e-6, float("nan"), float("inf")])
def test_abi_refuses_an_eps_that_is_none(eps):
    sides = (_lib.FmdHeadRotarySide * 2)()
    assert _lib.lib().fmd_head_rotary(sides, 0, 0, 0, 64, 64, 0, eps, None, None, None, 0, 0, None, 0, None, None) == 1


@gpu
@pytest.mark.parametrize("norm", [False, True], ids=["turn", "norm"])
def test_a_second_derivative_is_refused(cuda, norm):
    """Gradients taken with create_graph are first derivatives: to differentiate them raises and drops no term, with a
    gradient that depends on the inputs and with one that does not. Where nothing is differentiated again they are the
    same."""
    q, k, positions, cos, sin, (wq, wk) = make(5, 2, 1, 16, 16, torch.float32, norm)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk) if t is not None]
    out = head_norm_rotary(leaves[0], leaves[1], positions, cos, sin, *leaves[2:])
    once = torch.autograd.grad(out[0].sum() + out[1].sum(), leaves, retain_graph=True)
    again = torch.autograd.grad(out[0].sum() + out[1].sum(), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(once, again))
    if norm:  # without a norm the gradient is the same for all inputs: no second derivative is lost
        with pytest.raises(RuntimeError, match="first derivatives"):
            torch.autograd.grad(again[0].sum() + leaves[0].square().sum(), leaves[0])
    (dq,) = torch.autograd.grad(head_norm_rotary(leaves[0], leaves[1], positions, cos, sin, *leaves[2:])[0].square().sum(),
                                leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match="first derivatives"):
        (dq.square().sum() + leaves[0].square().sum()).backward()


@gpu
def test_forward_mode_is_refused(cuda):
    """A tangent on any input raises: it is not passed by."""
    q, k, positions, cos, sin, (wq, wk) = make(5, 2, 1, 16, 16, torch.float32, True)
    args = [q, k, positions, cos, sin, wq, wk]
    with forward_ad.dual_level():
        for i in (0, 1, 3, 4, 5, 6):
            dual = list(args)
            dual[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError):
                head_norm_rotary(*dual)
            with torch.no_grad(), pytest.raises(RuntimeError):
                head_norm_rotary(*dual)
        head_norm_rotary(*args)
