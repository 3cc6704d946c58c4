"""Softmax attention over packed sequences, with grouped heads, its gradients and its form for a few rows.

The sequences of a batch lie one behind the other in the rows of one tensor, told apart by CSR offsets on the device:
the atoms of the replicas of a disjoint union (every atom of a structure attends to the others), or the frames that
each replica has logged (``causal``: a frame sees those before it). One call serves whole sequences, a chunk of new
rows behind a cache, and a single new row of each sequence. No call reads a length on the host, so every call can be
captured in a CUDA graph. The kernels are ``fmd_packed_attention`` / ``fmd_packed_attention_bwd``
(fastmd_b200/csrc/packed_attention*.cu). CUDA tensors only: there is no CPU path.
"""
from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import Function

from . import _lib
from ._first_order import first_order, has_tangent
from ._lib import FmdAttention, c_size_t, call, ptr, stream
from .head_rotary import TYPES, _head_rows, _like


def _problem(q, k, v, offsets, key_offsets, key_counts, causal, scale) -> FmdAttention:
    return FmdAttention(q.data_ptr(), k.data_ptr(), v.data_ptr(), offsets.data_ptr(), key_offsets.data_ptr(),
                        ptr(key_counts), q.shape[0], k.shape[0], q.stride(0), q.stride(1), k.stride(0), k.stride(1),
                        v.stride(0), v.stride(1), scale, TYPES[q.dtype], offsets.shape[0] - 1, q.shape[1], k.shape[1],
                        q.shape[2], causal)


def _workspace(problem: FmdAttention, backward: bool, device) -> tuple[Tensor | None, int]:
    nbytes = c_size_t()
    call("fmd_packed_attention_workspace_bytes", problem, backward, nbytes)
    size = nbytes.value
    return (torch.empty(size, device=device, dtype=torch.uint8) if size else None), size


def _forward(q, k, v, offsets, key_offsets, key_counts, causal, scale, lse):
    device = q.device
    out = _like(q)
    sums = torch.empty(q.shape[:2], device=device, dtype=torch.float32) if lse else None
    problem = _problem(q, k, v, offsets, key_offsets, key_counts, causal, scale)
    workspace, size = _workspace(problem, False, device)
    call("fmd_packed_attention", problem, out.data_ptr(), ptr(sums), ptr(workspace), size,
         _lib.flags_word(device).data_ptr(), stream(device))
    return out, sums


class _PackedAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, key_offsets, key_counts, causal, scale):
        out, lse = _forward(q, k, v, offsets, key_offsets, key_counts, causal, scale, True)
        ctx.save_for_backward(q, k, v, offsets, key_offsets, key_counts, out, lse)
        ctx.causal, ctx.scale = causal, scale
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    def backward(ctx, g, glse):
        q, k, v, offsets, key_offsets, key_counts, out, lse = ctx.saved_tensors
        if g is None and glse is None:
            return (None,) * 8
        inputs = (g, glse, q, k, v)
        g = torch.zeros_like(out) if g is None else _head_rows(g)
        glse = glse.contiguous() if glse is not None else None
        dq = _like(q) if ctx.needs_input_grad[0] else None
        dk, dv = (_like(k), _like(v)) if ctx.needs_input_grad[1] or ctx.needs_input_grad[2] else (None, None)
        problem = _problem(q, k, v, offsets, key_offsets, key_counts, ctx.causal, ctx.scale)
        workspace, size = _workspace(problem, True, q.device)
        call("fmd_packed_attention_bwd", problem, out.data_ptr(), lse.data_ptr(), g.data_ptr(), g.stride(0),
             g.stride(1), ptr(glse), ptr(dq), ptr(dk), ptr(dv), ptr(workspace), size,
             _lib.flags_word(q.device).data_ptr(), stream(q.device))
        return *first_order("packed_attention", (dq, dk, dv), inputs), None, None, None, None, None


def _check_offsets(name: str, t: Tensor, shape: tuple) -> Tensor:
    if t.dtype != torch.int64 or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be int64 {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def packed_attention(q: Tensor, k: Tensor, v: Tensor, offsets: Tensor, key_offsets: Tensor | None = None,
                     key_counts: Tensor | None = None, *, causal: bool = False, scale: float | None = None,
                     return_lse: bool = False) -> Tensor | tuple[Tensor, Tensor]:
    """``softmax(scale * q k^T) v`` for the rows and keys of each sequence: ``[rows, heads, dim]``.

    q ``[rows, heads, dim]``, k and v ``[keys, key_heads, dim]``, float32 or bfloat16; query head ``h`` reads key head
    ``h // (heads // key_heads)``. ``dim`` is a multiple of 8 up to 128. Strides are free; tensors whose heads have no
    unit stride or do not start at multiples of 16 bytes are copied first. ``scale`` (not negative) defaults to
    ``dim ** -0.5``.

    Sequence ``b`` has the rows ``offsets[b] .. offsets[b + 1] - 1`` and the keys ``key_offsets[b] ..`` (default:
    the same offsets), all up to ``key_offsets[b + 1]`` or the first ``key_counts[b]`` of them: a cache gives each
    sequence a slot and says how far it is filled; what lies behind is never used, whatever its values. With
    ``causal``, row ``t`` of ``m`` sees the first ``t + 1 + n - m`` of ``n`` keys (the last row sees all). A row that
    sees no key gets zeros. ``offsets``, ``key_offsets`` and ``key_counts`` are int64 on the device; those that do not
    start at 0, fall, end elsewhere than at the last row or overfill a slot raise ``FMD_FLAG_INDEX_RANGE`` in the
    device's flags word.

    ``return_lse`` also returns float32 ``[rows, heads]``: the logarithm of each row's softmax denominator (-inf for
    a row that sees no key). Both are differentiable in q, k and v (first derivatives in reverse mode: others raise),
    with the same bits on every run. Scores, softmax and sums are held in 32 bits. For bfloat16, weights are rounded to
    bfloat16 for their products with v and the output's gradient, their gradients to 16 significant bits for those with
    k and q, and the backward pass goes by the output as it is stored where a row sees more than 16 keys: errors are up
    to 1.4 times that of rounding an exact result. A key that a row does not see has no part in it, but a value that is
    not finite may reach rows of its own sequence that do not see it (0 * inf), and in float32 with ``dim`` up to 64 an
    infinity gives NaN where the formula may have an infinity. There a call also reads all rows of k and v, filled or
    not, and needs a workspace of one and a half times their bytes."""
    _lib.require_cuda(q, k, v, offsets, key_offsets, key_counts)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[2] != k.shape[2]:
        raise ValueError("q must be [rows, heads, dim] and k and v the same [keys, key_heads, dim], got "
                         f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    if q.dtype not in TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v must all be float32 or bfloat16, got {q.dtype}, {k.dtype} and {v.dtype}")
    heads, key_heads, dim = q.shape[1], k.shape[1], q.shape[2]
    if dim % 8 or not 8 <= dim <= 128:
        raise ValueError(f"the head size must be a multiple of 8 up to 128, got {dim}")
    if key_heads < 1 or heads < 1 or heads % key_heads or heads // key_heads > 64:
        raise ValueError(f"heads must be a multiple of key_heads, at most 64 of each, got {heads} and {key_heads}")
    if offsets.dim() != 1 or offsets.shape[0] < 1:
        raise ValueError(f"offsets must be int64 [sequences + 1], got {tuple(offsets.shape)}")
    batch = offsets.shape[0] - 1
    if batch == 0 and (q.shape[0] or k.shape[0]):
        raise ValueError("rows without a sequence: offsets holds one value")
    offsets = _check_offsets("offsets", offsets, (batch + 1,))
    if key_offsets is None:
        if k.shape[0] != q.shape[0]:
            raise ValueError("key_offsets are needed where there are other keys than rows")
        key_offsets = offsets
    else:
        key_offsets = _check_offsets("key_offsets", key_offsets, (batch + 1,))
    if key_counts is not None:
        key_counts = _check_offsets("key_counts", key_counts, (batch,))
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0.0 <= scale <= 1e38:
        raise ValueError(f"scale must be between 0 and 1e38, got {scale}")
    args = (_head_rows(q), _head_rows(k), _head_rows(v), offsets, key_offsets, key_counts, bool(causal), scale)
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) or has_tangent(q, k, v):
        out, lse = _PackedAttention.apply(*args)
    else:
        out, lse = _forward(*args, return_lse)
    return (out, lse) if return_lse else out


__all__ = ["packed_attention"]
