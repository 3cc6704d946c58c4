"""Linear attention over packed sequences with a decay for each head, its gradients and its form for single rows.

Where ``packed_attention`` reads all that a replica has logged, ``decay_attention`` carries it along as one matrix a head, so
that a log may go on for ever: a new row costs the same whatever came before. ``decay_attention`` takes whole sequences or
chunks that follow a state; ``decay_attention_step`` takes one new row of every sequence. No call reads a length on the
host, so every call can be captured in a CUDA graph. The kernels are ``fmd_decay_attention`` and ``_bwd``, ``_step``
(fastmd_b200/csrc/decay_attention*.cu). CUDA tensors only: there is no CPU path.
"""
from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import Function

from . import _lib
from ._first_order import first_order, has_tangent
from ._lib import FmdDecay, c_size_t, call, on_device, ptr, stream
from .head_rotary import TYPES, _aligned, _head_rows, _like


def _problem(q, k, v, log_decay, offsets, scale) -> FmdDecay:
    return FmdDecay(q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), ptr(offsets), q.shape[0], q.stride(0),
                    q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), scale, TYPES[q.dtype],
                    offsets.shape[0] - 1 if offsets is not None else 0, q.shape[1], q.shape[2])


def _workspace(problem: FmdDecay, backward: int, device) -> tuple[Tensor | None, int]:
    """Of the forward pass (0), of the backward pass (1), or of one that is handed the forward pass's (2)."""
    nbytes = c_size_t()
    call("fmd_decay_attention_workspace_bytes", problem, backward, nbytes)
    size = nbytes.value
    return (torch.empty(size, device=device, dtype=torch.uint8) if size else None), size


def _states(q: Tensor, offsets: Tensor) -> Tensor:
    return torch.empty(offsets.shape[0] - 1, q.shape[1], q.shape[2], q.shape[2], device=q.device, dtype=torch.float32)


def _forward(q, k, v, log_decay, offsets, state, scale, keep):
    device = q.device
    out, after = _like(q), _states(q, offsets) if keep else None
    problem = _problem(q, k, v, log_decay, offsets, scale)
    workspace, size = _workspace(problem, 0, device)
    call("fmd_decay_attention", problem, ptr(state), out.data_ptr(), ptr(after), ptr(workspace), size,
         _lib.flags_word(device).data_ptr(), stream(device))
    return out, after, workspace


class _DecayAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, offsets, state, scale, keep):
        out, after, workspace = _forward(q, k, v, log_decay, offsets, state, scale, keep)
        if q.dtype != torch.float32:
            workspace = None
        ctx.save_for_backward(q, k, v, log_decay, offsets, state, workspace)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, after

    @staticmethod
    def backward(ctx, g, gafter):
        q, k, v, log_decay, offsets, state, forward = ctx.saved_tensors
        if g is None and gafter is None:
            return (None,) * 8
        inputs = (g, gafter, q, k, v, state)
        # a hook may have moved what was saved to another start
        q, k, v, log_decay, offsets = _head_rows(q), _head_rows(k), _head_rows(v), log_decay.contiguous(), offsets.contiguous()
        state, forward = _aligned_state(state), _aligned_state(forward)
        g = torch.zeros_like(q, memory_format=torch.contiguous_format) if g is None else _head_rows(g)
        gafter = _aligned_state(gafter)
        need = ctx.needs_input_grad
        dq, dk, dv = (_like(t) if n else None for t, n in zip((q, k, v), need))
        dstate = torch.empty_like(state) if need[5] else None
        problem = _problem(q, k, v, log_decay, offsets, ctx.scale)
        workspace, size = _workspace(problem, 1 if forward is None else 2, q.device)
        call("fmd_decay_attention_bwd", problem, ptr(state), ptr(forward), g.data_ptr(), g.stride(0), g.stride(1),
             ptr(gafter), ptr(dq), ptr(dk), ptr(dv), ptr(dstate), ptr(workspace), size,
             _lib.flags_word(q.device).data_ptr(), stream(q.device))
        dq, dk, dv, dstate = first_order("decay_attention", (dq, dk, dv, dstate), inputs)
        return dq, dk, dv, None, None, dstate, None, None


def _aligned_state(state: Tensor | None) -> Tensor | None:
    return None if state is None else _aligned(state)


def _check(q, k, v, log_decay, scale, *others) -> float:
    shape, kind, index = q.shape, q.dtype, q.get_device()
    if index < 0 or k.get_device() != index or v.get_device() != index or log_decay.get_device() != index \
            or any(t is not None and t.get_device() != index for t in others):
        _lib.require_cuda(q, k, v, log_decay, *others)
        raise ValueError("all tensors must be on the device of q")
    if len(shape) != 3 or k.shape != shape or v.shape != shape:
        raise ValueError("q, k and v must all be [rows, heads, dim], got "
                         f"{tuple(shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    if kind not in TYPES or k.dtype != kind or v.dtype != kind:
        raise ValueError(f"q, k and v must all be float32 or bfloat16, got {kind}, {k.dtype} and {v.dtype}")
    _, heads, dim = shape
    if dim % 8 or not 8 <= dim <= 128:
        raise ValueError(f"the head size must be a multiple of 8 up to 128, got {dim}")
    if not 1 <= heads <= 1024:
        raise ValueError(f"between 1 and 1024 heads, got {heads}")
    if log_decay.shape != (heads,) or log_decay.dtype != torch.float32:
        raise ValueError(f"log_decay must be float32 [{heads}], got {log_decay.dtype} {tuple(log_decay.shape)}")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0.0 <= scale <= 1e38:
        raise ValueError(f"scale must be between 0 and 1e38, got {scale}")
    return scale


def _check_state(state, batch, q) -> None:
    _, heads, dim = q.shape
    if state.shape != (batch, heads, dim, dim) or state.dtype != torch.float32:
        raise ValueError(f"state must be float32 {[batch, heads, dim, dim]}, got {state.dtype} {list(state.shape)}")


def decay_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, offsets: Tensor, state: Tensor | None = None, *,
                    scale: float | None = None, return_state: bool = False) -> Tensor | tuple[Tensor, Tensor]:
    """``out_t = scale * q_t S_t`` with ``S_t = exp(log_decay) S_{t-1} + k_t v_t^T``: ``[rows, heads, dim]``.

    q, k and v ``[rows, heads, dim]``, float32 or bfloat16; ``dim`` is a multiple of 8 up to 128. Strides are free; tensors
    whose heads have no unit stride or do not start at multiples of 16 bytes are copied first. Sequence ``b`` has the rows
    ``offsets[b] .. offsets[b + 1] - 1`` (int64 on the device; offsets that do not start at 0, fall or end elsewhere than
    at the last row raise ``FMD_FLAG_INDEX_RANGE`` in the device's flags word). ``log_decay`` is float32 ``[heads]``, at
    most 0 (0: nothing is forgotten; values above count as 0, values below -10,000 as that); it is given, not learned:
    where it requires a gradient the call raises. ``scale`` (not negative) defaults to ``dim ** -0.5``.

    ``state``: float32 ``[sequences, heads, dim, dim]``, k's index first: the matrices before the first rows (default:
    zeros). ``return_state`` also returns those behind the last rows, from which a later call or
    ``decay_attention_step`` goes on; a sequence without rows keeps its own.

    Differentiable in q, k, v and ``state`` (first derivatives in reverse mode: others raise), with the same bits on every
    run. Sums and matrices are held in 32 bits, and states are exact to FP32 in both types; in bfloat16 the weights of the
    pairs of rows and the decayed rows are rounded once as operands, which costs an output about as much as its own rounding
    (1.4 of it in all). Row by row the decay is one FP32 number, so that n rows' is off by up to n / 2 of its last bits.
    Sequences do not see each other's values, finite or not; within a sequence a value that is not finite may reach earlier
    rows too (0 * inf), and an infinity may give NaN. A ``log_decay`` of NaN gives NaN. Sequences of a few rows are taken row
    by row, others in chunks and, where they are few and long, in segments that run side by side. Which of these goes by the
    average length alone: one long sequence among many short ones takes its rows one after the other (0.2 us a row, or 2 to 5
    a chunk of 128), however many there are; a call of its own is faster for it. For the backward pass a call in float32
    keeps the planes of q, k and v (6 bytes a value) and, with segments, their matrices (13 MB at most). As for any autograd
    function, a backward pass is captured in a CUDA graph only while no eager graph of the same leaves is alive."""
    scale = _check(q, k, v, log_decay, scale, offsets, state)
    if offsets.dim() != 1 or offsets.shape[0] < 1 or offsets.dtype != torch.int64:
        raise ValueError(f"offsets must be int64 [sequences + 1], got {offsets.dtype} {tuple(offsets.shape)}")
    if offsets.shape[0] == 1 and q.shape[0]:
        raise ValueError("rows without a sequence: offsets holds one value")
    if state is not None:
        _check_state(state, offsets.shape[0] - 1, q)
    if torch.is_grad_enabled() and log_decay.requires_grad:
        raise ValueError("log_decay has no gradient here: pass it detached")
    args = (_head_rows(q), _head_rows(k), _head_rows(v), log_decay.contiguous(), offsets.contiguous(), _aligned_state(state),
            scale, bool(return_state))
    trains = q.requires_grad or k.requires_grad or v.requires_grad or (state is not None and state.requires_grad)
    with on_device(q.device):
        if (torch.is_grad_enabled() and trains) or has_tangent(q, k, v, log_decay, state):
            out, after = _DecayAttention.apply(*args)
        else:
            out, after, _ = _forward(*args)
    return (out, after) if return_state else out


def decay_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, *,
                         scale: float | None = None) -> Tensor:
    """One new row of every sequence: ``state = exp(log_decay) state + k v^T`` in place, ``out = scale * q state``.

    q, k and v ``[sequences, heads, dim]`` and ``log_decay`` as for ``decay_attention``; any strides. ``state`` is
    contiguous float32 ``[sequences, heads, dim, dim]`` and is the caller's: it moves on by a row each call, by a decay that is
    one FP32 number (of a ``log_decay`` below some 10^-7 nothing is left of it). Not differentiable: where an argument requires a gradient the call raises (``decay_attention`` takes single rows too)."""
    scale = _check(q, k, v, log_decay, scale, state)
    _check_state(state, q.shape[0], q)
    if not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError("state must be contiguous and start at a multiple of 16 bytes: it is changed in place")
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad
                                     or state.requires_grad)) or has_tangent(q, k, v, log_decay, state):
        raise ValueError("decay_attention_step has no gradient: call it under torch.no_grad(), or decay_attention")
    if q.stride(2) != 1:
        q = q.contiguous()
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    device = q.device
    out = torch.empty(q.shape, device=device, dtype=q.dtype)
    with on_device(device):
        call("fmd_decay_attention_step", _problem(q, k, v, log_decay.contiguous(), None, scale), state.data_ptr(),
             out.data_ptr(), stream(device))
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)
    return out


__all__ = ["decay_attention", "decay_attention_step"]
