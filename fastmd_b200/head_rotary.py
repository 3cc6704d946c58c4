"""RMS norm of each query and key head with the rotation of its position, in one pass, and its backward pass.

``head_norm_rotary`` serves blocks that attend over packed rows (``packed_attention``): the frames a trajectory has
logged, with the MD step as position, or any other ordered rows. ``rotary_table`` makes the angles once per model.
The kernels are ``fmd_head_rotary`` (fastmd_b200/csrc/head_rotary.cu). CUDA tensors only: there is no CPU path.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch import Tensor
from torch.autograd import Function

from . import _lib
from ._first_order import first_order, has_tangent
from ._lib import FmdHeadRotarySide, call, ptr, stream

TYPES = {torch.float32: 0, torch.bfloat16: 1}


def rotary_table(length: int, rotary_dim: int, *, base: float = 10000.0, factor: float = 1.0,
                 trained_length: int | None = None, turns: tuple[float, float] = (1.0, 32.0), amplitude: float = 1.0,
                 device=None) -> tuple[Tensor, Tensor]:
    """``(cos, sin)`` float32 ``[length, rotary_dim / 2]`` of the angles ``position * base^(-2p / rotary_dim)``.

    For positions beyond those a model was trained on, ``factor`` divides the frequencies: all of them, or, with
    ``trained_length``, by how often pair ``p`` turns over that length: below ``turns[0]`` the whole factor, above
    ``turns[1]`` none, in between a linear blend. ``amplitude`` multiplies both tables. Computed in 64 bits."""
    length, rotary_dim = int(length), int(rotary_dim)
    if length < 0 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_table needs length >= 0 and an even rotary_dim >= 2, got {length}, {rotary_dim}")
    if base <= 0 or factor <= 0 or turns[0] >= turns[1] or (trained_length is not None and trained_length < 1):
        raise ValueError("rotary_table needs base > 0, factor > 0, trained_length >= 1 and turns[0] < turns[1]")
    frequency = float(base) ** (-torch.arange(0, rotary_dim, 2, device=device, dtype=torch.float64) / rotary_dim)
    if trained_length is None:
        frequency = frequency / factor
    else:
        kept = (trained_length * frequency / (2 * math.pi) - turns[0]) / (turns[1] - turns[0])
        kept = kept.clamp(0.0, 1.0)
        frequency = frequency * (kept + (1.0 - kept) / factor)
    angle = torch.arange(length, device=device, dtype=torch.float64)[:, None] * frequency
    return (angle.cos() * amplitude).float(), (angle.sin() * amplitude).float()


def _head_rows(x: Tensor) -> Tensor:
    """``x`` with unit stride inside a head and 16-byte rows, heads and base; copied only when needed."""
    row, head, unit = x.stride()
    width = 16 // x.element_size()
    if unit == 1 and row and head and not (row % width or head % width or x.data_ptr() % 16):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _aligned(table: Tensor) -> Tensor:
    table = table.contiguous()
    return table.clone() if table.data_ptr() % 16 else table


def _like(x: Tensor) -> Tensor:
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _launch(sides, x, weight, cos, sin, positions, interleaved, eps, backward):
    rows, _, dim = x.shape
    length, half = cos.shape
    device = x.device
    workspace, size = None, 0
    if backward and weight is not None:
        nbytes = ctypes.c_size_t()
        call("fmd_head_rotary_workspace_bytes", dim, nbytes)
        size = nbytes.value
        workspace = torch.empty(size, device=device, dtype=torch.uint8)
    kind = TYPES[x.dtype]
    call("fmd_head_rotary", sides, kind, kind if weight is None else TYPES[weight.dtype], rows, dim, 2 * half,
         interleaved, eps, positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), length, backward, ptr(workspace), size,
         ptr(_lib.flags_word(device)), stream(device))


def _forward(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved):
    q_out, k_out = _like(q), _like(k)
    sides = (FmdHeadRotarySide * 2)(
        FmdHeadRotarySide(q.data_ptr(), None, q_out.data_ptr(), ptr(q_weight), None, q.stride(0), q.stride(1), 0, 0,
                          q.shape[1]),
        FmdHeadRotarySide(k.data_ptr(), None, k_out.data_ptr(), ptr(k_weight), None, k.stride(0), k.stride(1), 0, 0,
                          k.shape[1]))
    _launch(sides, q, q_weight if q_weight is not None else k_weight, cos, sin, positions, interleaved, eps, False)
    return q_out, k_out


class _HeadNormRotary(Function):
    @staticmethod
    def forward(ctx, q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved):
        q_out, k_out = _forward(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved)
        # without a norm the gradient is a rotation of the output's: the input is not kept
        ctx.save_for_backward(q if q_weight is not None else None, k if k_weight is not None else None, positions,
                              cos, sin, q_weight, k_weight)
        ctx.eps, ctx.interleaved = eps, interleaved
        return q_out, k_out

    @staticmethod
    def backward(ctx, gq, gk):
        q, k, positions, cos, sin, q_weight, k_weight = ctx.saved_tensors
        sides = (FmdHeadRotarySide * 2)()
        grads, kept, weight = [], [], None
        for i, (x, g, w) in enumerate(((q, gq, q_weight), (k, gk, k_weight))):
            if not (ctx.needs_input_grad[i] or ctx.needs_input_grad[5 + i]):  # heads = 0: this side is left out
                grads.append((None, None))
                continue
            g = _head_rows(g)
            dx, dw = _like(g), torch.empty_like(w) if w is not None else None
            weight = w if w is not None else weight
            sides[i] = FmdHeadRotarySide(ptr(x), g.data_ptr(), dx.data_ptr(), ptr(w), ptr(dw),
                                         x.stride(0) if x is not None else 0, x.stride(1) if x is not None else 0,
                                         g.stride(0), g.stride(1), g.shape[1])
            grads.append((dx, dw))
            kept.append(g)
        if kept:
            _launch(sides, kept[0], weight, cos, sin, positions, ctx.interleaved, ctx.eps, True)
        (dq, dwq), (dk, dwk) = grads
        dq, dk, dwq, dwk = first_order("head_norm_rotary", (dq, dk, dwq, dwk), (gq, gk, q, k, q_weight, k_weight))
        return dq, dk, None, None, None, dwq, dwk, None, None


def head_norm_rotary(q: Tensor, k: Tensor, positions: Tensor, cos: Tensor, sin: Tensor,
                     q_weight: Tensor | None = None, k_weight: Tensor | None = None, *, eps: float = 1e-6,
                     interleaved: bool = False) -> tuple[Tensor, Tensor]:
    """``(q', k')`` for q ``[rows, q_heads, dim]`` and k ``[rows, k_heads, dim]`` (float32 or bfloat16, any strides;
    rows that are not 16-byte aligned are copied first).

    With its weight ``[dim]`` (float32 or the type of q and k; None: no norm) a head is divided by
    ``sqrt(mean(x^2) + eps)`` (``eps`` not negative) and multiplied by the weight. Then its first
    ``2 * cos.shape[1]`` values are turned by row ``positions[row]`` (int64) of the float32 tables: pairs
    ``(p, p + half)``, or ``(2p, 2p + 1)`` with ``interleaved``. ``dim`` is a multiple of 8 up to 128, the turned part a
    multiple of 8 up to ``dim``. A position outside the table raises ``FMD_FLAG_INDEX_RANGE`` in the device's flags word
    and the turned part is zero.
    Differentiable in q, k and the weights (first derivatives in reverse mode: others raise), with the same bits on every run;
    computed in 32 bits, rounded once."""
    _lib.require_cuda(q, k, positions, cos, sin, q_weight, k_weight)
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError("q and k must be [rows, heads, dim] with the same rows and dim, got "
                         f"{tuple(q.shape)} and {tuple(k.shape)}")
    if q.dtype not in TYPES or k.dtype != q.dtype:
        raise ValueError(f"q and k must both be float32 or bfloat16, got {q.dtype} and {k.dtype}")
    rows, _, dim = q.shape
    if dim % 8 or not 8 <= dim <= 128:
        raise ValueError(f"the head size must be a multiple of 8 up to 128, got {dim}")
    if max(q.shape[1], k.shape[1]) > 1024:
        raise ValueError(f"at most 1024 heads, got {q.shape[1]} and {k.shape[1]}")
    if positions.shape != (rows,) or positions.dtype != torch.int64:
        raise ValueError(f"positions must be int64 [{rows}], got {positions.dtype} {tuple(positions.shape)}")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be float32 tables of the same shape [positions, half]")
    if cos.shape[1] % 4 or not 4 <= cos.shape[1] <= dim // 2:
        raise ValueError(f"the turned part must be a multiple of 8 up to the head size, got {2 * cos.shape[1]}")
    for w in (q_weight, k_weight):
        if w is not None and (w.shape != (dim,) or w.dtype not in (torch.float32, q.dtype)):
            raise ValueError(f"a norm weight must be [{dim}] in float32 or the type of q and k")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("both norm weights must have the same type")
    eps = float(eps)
    if not 0.0 <= eps <= 1e38:
        raise ValueError(f"eps must be between 0 and 1e38, got {eps}")
    weights = [w if w is None or w.is_contiguous() else w.contiguous() for w in (q_weight, k_weight)]
    args = (_head_rows(q), _head_rows(k), positions.contiguous(), _aligned(cos), _aligned(sin), *weights,
            eps, bool(interleaved))
    trains = (q.requires_grad or k.requires_grad or (q_weight is not None and q_weight.requires_grad)
              or (k_weight is not None and k_weight.requires_grad))
    if (trains and torch.is_grad_enabled()) or has_tangent(q, k, cos, sin, q_weight, k_weight):
        return _HeadNormRotary.apply(*args)
    return _forward(*args)


__all__ = ["rotary_table", "head_norm_rotary"]
