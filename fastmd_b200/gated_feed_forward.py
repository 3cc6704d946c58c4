"""A gated feed-forward block, ``(act(x gate^T) * (x up^T)) down^T``, and its backward pass.

The other half of a block that attends (``packed_attention``, ``decay_attention``): both first projections, the activation
and the product are one kernel, the last projection another, and the backward pass three. The kernels are
``fmd_gated_feed_forward`` / ``fmd_gated_feed_forward_bwd`` (fastmd_b200/csrc/gated_feed_forward.cu). CUDA tensors only:
there is no CPU path.
"""
from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import Function

from . import _lib
from ._first_order import first_order, has_tangent
from ._lib import FmdFeedForward, FmdPadded, c_size_t, call, on_device, ptr, stream
from .head_rotary import TYPES, _aligned

ACTIVATIONS = {"silu": 0, "gelu": 1}


def _ready(x: Tensor) -> bool:
    """Whether the kernels read ``x`` as it is: unit stride inside a row and, in 16 bits, rows at multiples of 16 bytes."""
    row, unit = x.stride()
    rows, columns = x.shape
    whole = (unit == 1 or columns == 1) and (row >= columns or rows <= 1)
    return whole and (x.dtype == torch.float32 or not (x.data_ptr() % 16 or (row % 8 and rows > 1)))


def _rows(*tensors: Tensor) -> tuple[Tensor, ...]:
    """The tensors as the kernels read them; those that are not are copied, in 16 bits by one kernel, to padded rows. Not for
    autograd to see: the gradients belong to the tensors themselves."""
    some = [t for t in tensors if not _ready(t)]
    if not some:
        return tensors
    if some[0].dtype == torch.float32:
        copies = iter([t.contiguous() for t in some])
    else:
        wide = [(t.shape[1] + 7) // 8 * 8 for t in some]
        starts = [0]
        for t, row in zip(some, wide):
            starts.append(starts[-1] + (t.shape[0] * row + 127) // 128 * 128)
        room = torch.empty(starts[-1], device=some[0].device, dtype=some[0].dtype)
        made = [room.as_strided(t.shape, (row, 1), at) for t, row, at in zip(some, wide, starts)]
        call("fmd_pad_rows", (FmdPadded * len(some))(*((t.data_ptr(), m.data_ptr(), *t.shape, *t.stride(), row)
                                                       for t, m, row in zip(some, made, wide))), len(some), stream(room.device))
        copies = iter(made)
    return tuple(t if _ready(t) else next(copies) for t in tensors)


def _problem(x, gate, up, down, activation) -> FmdFeedForward:
    return FmdFeedForward(x.data_ptr(), gate.data_ptr(), up.data_ptr(), down.data_ptr(), x.shape[0], x.stride(0),
                          gate.stride(0), up.stride(0), down.stride(0), x.shape[1], gate.shape[0], down.shape[0],
                          TYPES[x.dtype], activation)


def _forward(x, gate, up, down, activation, keep):
    device = x.device
    y = torch.empty(x.shape[0], down.shape[0], device=device, dtype=x.dtype)
    problem = _problem(x, gate, up, down, activation)
    kept, forward, backward = c_size_t(), c_size_t(), c_size_t()
    call("fmd_gated_feed_forward_bytes", problem, keep, kept, forward, backward)
    size, more = kept.value, forward.value
    # as scratch of the call the two are one buffer (sizes are multiples of 256)
    room = torch.empty(size if keep else size + more, device=device, dtype=torch.uint8)
    workspace = torch.empty(more, device=device, dtype=torch.uint8) if keep and more else None
    start = room.data_ptr()
    call("fmd_gated_feed_forward", problem, y.data_ptr(), keep, start, size, ptr(workspace) if keep else start + size, more,
         _lib.flags_word(device).data_ptr(), stream(device))
    return y, room, backward.value


class _GatedFeedForward(Function):
    @staticmethod
    def forward(ctx, x, gate, up, down, activation):
        given = (x, gate, up, down)
        rows = _rows(*given)
        y, kept, ctx.size = _forward(*rows, activation, True)
        ctx.save_for_backward(*given, kept, *(None if a is b else a for a, b in zip(rows, given)))
        ctx.activation = activation
        return y

    @staticmethod
    def backward(ctx, g):
        *like, kept, x, gate, up, down = ctx.saved_tensors
        x, gate, up, down = (b if a is None else a for a, b in zip((x, gate, up, down), like))
        device, inputs = x.device, (g, *like)
        g, = _rows(g)
        # a hook may have moved what was saved: without the padding of its rows, or to another start
        kept, (x, gate, up, down) = _aligned(kept), _rows(x, gate, up, down)
        grads = [torch.empty(t.shape, device=device, dtype=t.dtype) if need else None
                 for t, need in zip(like, ctx.needs_input_grad)]
        workspace = torch.empty(ctx.size, device=device, dtype=torch.uint8)
        call("fmd_gated_feed_forward_bwd", _problem(x, gate, up, down, ctx.activation), kept.data_ptr(), kept.numel(),
             g.data_ptr(), g.stride(0), *(ptr(t) for t in grads), workspace.data_ptr(), ctx.size,
             _lib.flags_word(device).data_ptr(), stream(device))
        return *first_order("gated_feed_forward", grads, inputs), None


def gated_feed_forward(x: Tensor, gate: Tensor, up: Tensor, down: Tensor, *, activation: str = "silu") -> Tensor:
    """``(act(x gate^T) * (x up^T)) down^T``: ``[.., width] -> [.., out]``.

    x ``[.., width]``, gate and up ``[hidden, width]``, down ``[out, hidden]`` (as ``torch.nn.Linear`` keeps its weights),
    all float32 or all bfloat16. ``activation``: ``"silu"``, ``a / (1 + e^-a)``, or ``"gelu"``, ``a (1 + erf(a / sqrt 2)) /
    2``. Sizes are free, and so are strides; in bfloat16, rows that do not start at multiples of 16 bytes are copied first
    (keep weights of odd width in padded storage to save that).

    Differentiable in all four (first derivatives in reverse mode: others raise), with the same bits on every run. Sums are
    held in 32 bits; in bfloat16 the gated product and the gradients of the two projections are rounded to bfloat16 as
    operands of the next product, each of which costs a result about as much as its own rounding; the activation is good to
    2^-16 of itself, and its value and slope reach the gradients with 11 bits beside the largest of 16 units of a row (none are
    left below 2^-39 of it). In float32 each product is six of bfloat16 planes (a few rows without gradients: FP32). Rows do not see each other's values, finite or not; within
    a row an infinity may give NaN where the formula has an infinity. For the backward pass a call keeps 6.5 bytes a row and
    hidden unit (float32: 14, and one and a half times the bytes of x and the weights). As for any autograd function, a
    backward pass is captured in a CUDA graph only while no eager graph of the same leaves is alive."""
    _lib.require_cuda(x, gate, up, down)
    lead, weights, last = x.shape, gate.shape, down.shape
    if x.dim() < 1 or gate.dim() != 2 or up.shape != weights or down.dim() != 2 or lead[-1] != weights[1] \
            or last[1] != weights[0]:
        raise ValueError("x must be [.., width], gate and up [hidden, width] and down [out, hidden], got "
                         f"{tuple(lead)}, {tuple(weights)}, {tuple(up.shape)} and {tuple(last)}")
    kind = x.dtype
    if kind not in TYPES or gate.dtype != kind or up.dtype != kind or down.dtype != kind:
        raise ValueError("x and the weights must all be float32 or bfloat16, got "
                         f"{kind}, {gate.dtype}, {up.dtype} and {down.dtype}")
    index = x.get_device()
    if gate.get_device() != index or up.get_device() != index or down.get_device() != index:
        raise ValueError("x and the weights must be on one device")
    hidden, width, out = *weights, last[0]
    if not (0 < width <= 2 ** 20 and 0 < hidden <= 2 ** 20 and 0 < out <= 2 ** 20):
        raise ValueError(f"width, hidden and out must be between 1 and 2^20, got {width}, {hidden} and {out}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    flat = x if len(lead) == 2 else x.reshape(-1, width)
    args, kind = (flat, gate, up, down), ACTIVATIONS[activation]
    with on_device(x.device):
        if (torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or up.requires_grad or down.requires_grad)) \
                or has_tangent(x, gate, up, down):
            y = _GatedFeedForward.apply(*args, kind)
        else:
            y = _forward(*_rows(*args), kind, False)[0]
    return y if len(lead) == 2 else y.view(*lead[:-1], out)


__all__ = ["gated_feed_forward"]
