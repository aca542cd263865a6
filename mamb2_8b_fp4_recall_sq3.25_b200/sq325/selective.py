"""The mixer's selective scan in unquantised states (sq_selective_*): prompts, gradients, single tokens.

Per head, with s_t = softplus(dt_t + dt_bias),

    H_t = exp(A s_t) H_{t-1} + s_t x_t B_t^T,    y_t = H_t C_t + D x_t

H is fp32 [dim, 128]; B and C are shared by the heads of a group.  Where `codec.scan` and `state_codec.scan` carry
quantised states, this one carries them whole, and where `state_training.scan_training` freezes A, D and dt_bias, it has
gradients for everything, the states among them.  Nothing but the inputs is kept for the backward pass.  A is negative
(the largest decay is 1).  What depends on a NaN or an infinity is not finite, and other values of its chunk of 128 tokens and
of later ones may be NaN with it, in its head, or behind B and C in its group; a dt of minus infinity passes its token over.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib
from .activations import TYPES
from .conv import _ptr, checked_lengths, inner_packed, written

__all__ = ['selective_scan', 'selective_step']

N = 128
_HALF = (torch.float16, torch.bfloat16)


def checked_heads(A, D, dt_bias, heads, device):
    """Per-head parameters: A fp32, D and dt_bias fp16, bf16, fp32 or None."""
    if not isinstance(A, torch.Tensor) or A.shape != (heads,) or A.dtype != torch.float32 or A.get_device() != device.index:
        raise ValueError(f'A must be FP32 [{heads}] on {device}')
    for name, t in (('D', D), ('dt_bias', dt_bias)):
        if t is not None and (not isinstance(t, torch.Tensor) or t.shape != (heads,) or t.dtype not in TYPES
                              or t.get_device() != device.index):
            raise ValueError(f'{name} must be None or FP16, BF16 or FP32 [{heads}] on {device}')
    return A.contiguous(), None if D is None else D.contiguous(), None if dt_bias is None else dt_bias.contiguous()


def checked_state(state, shape, device, name='initial_state'):
    if state is None:
        return None
    if not isinstance(state, torch.Tensor) or state.shape != shape or state.dtype != torch.float32 \
            or state.get_device() != device.index:
        raise ValueError(f'{name} must be FP32 {list(shape)} on {device}')
    return state.contiguous()


def scan_args(x, dt, A, B, C_, D, dt_bias, state, lengths):
    """The arguments that forward and backward share, of checked tensors."""
    batch, length, heads, dim = x.shape
    sx, st, sb, sc = x.stride(), dt.stride(), B.stride(), C_.stride()
    return _lib.SelectiveArgs(batch, length, heads, dim, B.shape[2], TYPES[x.dtype], x.data_ptr(), sx[0], sx[1],
                              dt.data_ptr(), st[0], st[1], A.data_ptr(), B.data_ptr(), sb[0], sb[1], C_.data_ptr(), sc[0], sc[1],
                              _ptr(D), 0 if D is None else TYPES[D.dtype], _ptr(dt_bias), 0 if dt_bias is None else TYPES[dt_bias.dtype],
                              _ptr(state), _ptr(lengths))


@functools.lru_cache(maxsize=256)
def _workspace_bytes(batch, length, heads, dim, groups, backward):
    return int(_lib.load().sq_selective_workspace(batch, length, heads, dim, groups, backward))


def _workspace(a, backward, device):
    nbytes = _workspace_bytes(a.batch, a.length, a.heads, a.dim, a.groups, backward)
    work = torch.empty(nbytes, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = work.data_ptr(), nbytes
    return work                                              # alive until the launch


def scan_forward(x, dt, A, B, C_, D, dt_bias, state, lengths, want_state):
    """(y, final state or None) of checked tensors."""
    batch, length, heads, dim = x.shape
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    last = torch.empty(batch, heads, dim, N, dtype=torch.float32, device=x.device) if want_state else None
    a = scan_args(x, dt, A, B, C_, D, dt_bias, state, lengths)
    a.y, a.y_batch_stride, a.y_token_stride, a.state_out = y.data_ptr(), length * heads * dim, heads * dim, _ptr(last)
    work = _workspace(a, 0, x.device)
    _lib.launch('sq_selective_forward', x.device, C.byref(a))
    del work
    return y, last


def scan_backward(x, dt, A, B, C_, D, dt_bias, state, lengths, dy, dlast, dx, dB, dC, need):
    """Writes dx, dB, dC (dB and dC with the same strides) and returns (ddt, dA, dD, ddt_bias, dstate); need: which
    of A, D, dt_bias, state have a gradient."""
    device = x.device
    ddt = torch.empty_like(dt, memory_format=torch.contiguous_format)
    dA, dD, dbias, dstate = (torch.empty_like(t) if want else None for t, want in zip((A, D, dt_bias, state), need))
    a = scan_args(x, dt, A, B, C_, D, dt_bias, state, lengths)
    a.dy, a.dy_batch_stride, a.dy_token_stride, a.dstate_out = dy.data_ptr(), dy.stride(0), dy.stride(1), _ptr(dlast)
    a.dx, a.dx_batch_stride, a.dx_token_stride, a.ddt = dx.data_ptr(), dx.stride(0), dx.stride(1), ddt.data_ptr()
    a.dB, a.dC, a.dg_batch_stride, a.dg_token_stride = dB.data_ptr(), dC.data_ptr(), dB.stride(0), dB.stride(1)
    a.dA, a.dD, a.ddt_bias, a.dstate_in = _ptr(dA), _ptr(dD), _ptr(dbias), _ptr(dstate)
    work = _workspace(a, 1, device)
    _lib.launch('sq_selective_backward', device, C.byref(a))
    del work
    return ddt, dA, dD, dbias, dstate


def packed_like_forward(x, dt, B, C_):
    """Tensors whose last axes the kernels step through, also after hooks moved them."""
    return inner_packed(x, 2), inner_packed(dt, 1), inner_packed(B, 2), inner_packed(C_, 2)


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C_, D, dt_bias, state, lengths, want_state):
        y, last = scan_forward(x, dt, A, B, C_, D, dt_bias, state, lengths, want_state)
        ctx.save_for_backward(x, dt, A, B, C_, D, dt_bias, state, lengths)
        ctx.set_materialize_grads(False)
        return (y, last) if want_state else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast=None):
        x, dt, A, B, C_, D, dt_bias, state, lengths = ctx.saved_tensors
        # Hooks on saved tensors (offloading, recomputation) may have put them elsewhere, with other strides.
        x, dt, B, C_ = packed_like_forward(x, dt, B, C_)
        A, D, dt_bias, state, lengths = (None if t is None else t.contiguous() for t in (A, D, dt_bias, state, lengths))
        dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else inner_packed(dy, 2)
        dlast = None if dlast is None else dlast.contiguous()
        need = ctx.needs_input_grad
        dx, dB, dC = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (x, B, C_))
        ddt, dA, dD, dbias, dstate = scan_backward(x, dt, A, B, C_, D, dt_bias, state, lengths, dy, dlast, dx, dB, dC,
                                                   (need[2], need[5], need[6], need[7]))
        return dx, ddt, dA, dB, dC, dD, dbias, dstate, None, None


def selective_scan(x, dt, A, B, C_, D=None, dt_bias=None, initial_state=None, lengths=None, return_final_state=False):
    """The scan of x [batch, length, heads, dim] with dt [batch, length, heads] and B, C [batch, length, groups, 128], all
    fp16 or all bf16: y like x, or (y, final state) with return_final_state.

    A fp32 [heads], negative; D and dt_bias [heads] in fp16, bf16 or fp32, or None.
    initial_state fp32 [batch, heads, dim, 128]: the state before the first token (None: zero).
    lengths int32 [batch]: tokens of each sequence; those behind leave the state as it is, are not read, and are zero in
    y and in the gradients.  Differentiable in every tensor but lengths."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _HALF or not x.is_cuda or x.ndim != 4 or 0 in x.shape:
        raise ValueError('x must be CUDA FP16 or BF16 [batch,length,heads,dim]')
    batch, length, heads, dim = x.shape
    device = x.device
    if not isinstance(B, torch.Tensor) or B.ndim != 4 or B.shape[2] < 1 or heads % B.shape[2]:
        raise ValueError('heads must be divisible by B/C groups')
    groups = (batch, length, B.shape[2], N)
    for name, t, shape in (('dt', dt, (batch, length, heads)), ('B', B, groups), ('C', C_, groups)):
        if not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype != x.dtype or t.get_device() != device.index:
            raise ValueError(f"{name} must be {list(shape)} in x's dtype, on its device")
    A, D, dt_bias = checked_heads(A, D, dt_bias, heads, device)
    state = checked_state(initial_state, (batch, heads, dim, N), device)
    lengths = checked_lengths(lengths, batch, device)
    _lib.refuse_tangents('selective_scan', x, dt, A, B, C_, D, dt_bias, state)
    x, dt, B, C_ = packed_like_forward(x, dt, B, C_)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, dt, A, B, C_, D, dt_bias, state)):
        return _SelectiveScan.apply(x, dt, A, B, C_, D, dt_bias, state, lengths, bool(return_final_state))
    y, last = scan_forward(x, dt, A, B, C_, D, dt_bias, state, lengths, return_final_state)
    return (y, last) if return_final_state else y


@torch.no_grad()
def selective_step(x, dt, A, B, C_, state, D=None, dt_bias=None):
    """One token of each row: y [batch, heads, dim] of x [batch, heads, dim], dt [batch, heads], B and C
    [batch, groups, 128], all fp16 or all bf16; state fp32 [batch, heads, dim, 128], contiguous, moves on in place."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _HALF or not x.is_cuda or x.ndim != 3 or 0 in x.shape:
        raise ValueError('x must be CUDA FP16 or BF16 [batch,heads,dim]')
    batch, heads, dim = x.shape
    device = x.device
    if not isinstance(B, torch.Tensor) or B.ndim != 3 or B.shape[1] < 1 or heads % B.shape[1]:
        raise ValueError('heads must be divisible by B/C groups')
    groups = (batch, B.shape[1], N)
    for name, t, shape in (('dt', dt, (batch, heads)), ('B', B, groups), ('C', C_, groups)):
        if not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype != x.dtype or t.get_device() != device.index:
            raise ValueError(f"{name} must be {list(shape)} in x's dtype, on its device")
    A, D, dt_bias = checked_heads(A, D, dt_bias, heads, device)
    if checked_state(state, (batch, heads, dim, N), device, 'state') is not state:
        raise ValueError('state must be contiguous: it is updated in place')
    _lib.refuse_tangents('selective_step', x, dt, A, B, C_, D, dt_bias, state)
    x, dt, B, C_ = inner_packed(x, 2), inner_packed(dt, 1), inner_packed(B, 2), inner_packed(C_, 2)
    y = torch.empty(batch, heads, dim, dtype=x.dtype, device=device)
    a = _lib.SelectiveStepArgs(batch, heads, dim, groups[1], TYPES[x.dtype], x.data_ptr(), x.stride(0), dt.data_ptr(), dt.stride(0),
                               A.data_ptr(), B.data_ptr(), B.stride(0), C_.data_ptr(), C_.stride(0),
                               _ptr(D), 0 if D is None else TYPES[D.dtype], _ptr(dt_bias), 0 if dt_bias is None else TYPES[dt_bias.dtype],
                               state.data_ptr(), y.data_ptr())
    _lib.launch('sq_selective_step', device, C.byref(a))
    written(state)
    return y
