"""The mixer's short causal convolution (sq_causal_conv_*): prompts, gradients, single tokens.

    z[t,c] = bias[c] + sum_k weight[c,k] x[t - (taps-1) + k, c],    y = z sigmoid(z)  (activation='silu')  or  z

Inputs before the first token are those of a carried state [batch, taps-1, channels], or zero.  Sums are fp32, the
result is rounded once.  The backward pass computes z again from the input; with keep='int8' it does so from the input
in 8 bits, which is all that is kept: the output is that of the given input, the gradients are those at the kept values.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .activations import TYPES, PackedActivations, empty_packed

__all__ = ['causal_conv', 'causal_conv_step']


def inner_packed(t, axes):
    """t with its last `axes` axes contiguous (a copy only where they are not)."""
    if t.is_contiguous():
        return t
    step = 1
    for k in range(t.ndim - 1, t.ndim - 1 - axes, -1):
        if t.shape[k] != 1 and t.stride(k) != step:
            return t.contiguous()
        step *= t.shape[k]
    return t


def checked_lengths(lengths, batch, device):
    if lengths is None:
        return None
    if not isinstance(lengths, torch.Tensor) or lengths.shape != (batch,) or lengths.dtype != torch.int32 \
            or lengths.get_device() != device.index:
        raise ValueError(f'lengths must be an int32 tensor of shape ({batch},) on {device}')
    return lengths.contiguous()


def checked_weight(weight, bias, channels, dtype, device):
    if not isinstance(weight, torch.Tensor) or weight.ndim != 2 or weight.shape[0] != channels or not 2 <= weight.shape[1] <= 4:
        raise ValueError(f'weight must be [{channels}, taps] with 2 to 4 taps')
    if weight.dtype != dtype and weight.dtype != torch.float32 or weight.get_device() != device.index:
        raise ValueError("weight must have the input's dtype or FP32, on its device")
    if bias is not None and (not isinstance(bias, torch.Tensor) or bias.shape != (channels,) or bias.dtype != weight.dtype
                             or bias.get_device() != device.index):
        raise ValueError(f"bias must be [{channels}] in the weight's dtype, on its device")
    return weight.contiguous(), None if bias is None else bias.contiguous()


def checked_keep(keep):
    if keep not in (None, 'int8'):
        raise ValueError("keep must be None or 'int8'")
    return keep


def _silu(activation):
    if activation not in ('silu', None):
        raise ValueError("activation must be 'silu' or None")
    return int(activation == 'silu')


def _ptr(t):
    return None if t is None else t.data_ptr()


def written(*tensors):
    """Tells autograd that a kernel wrote tensors in place: a gradient that saved one of them raises."""
    for t in tensors:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def conv_args(shape, dtype, x, packed, weight, bias, state, lengths, silu):
    """The arguments that forward and backward share."""
    batch, length, channels = shape
    at = (None, 0, 0) if x is None else (x.data_ptr(), x.stride(0), x.stride(1))
    codes = (None, None) if packed is None else (packed.codes.data_ptr(), packed.scales.data_ptr())
    return _lib.CausalConvArgs(batch, length, channels, weight.shape[1], silu, TYPES[dtype], TYPES[weight.dtype], *at, *codes,
                               weight.data_ptr(), _ptr(bias), _ptr(state), _ptr(lengths))


def conv_forward(shape, dtype, x, packed, weight, bias, state, lengths, silu, want_state=False):
    """(y, last inputs or None) on checked arguments; x is kept in 8 bits in `packed`, where that is given."""
    device = weight.device
    y = torch.empty(shape, dtype=dtype, device=device)
    last = torch.empty(shape[0], weight.shape[1] - 1, shape[2], dtype=dtype, device=device) if want_state else None
    a = conv_args(shape, dtype, x, packed, weight, bias, state, lengths, silu)
    a.y, a.y_batch_stride, a.y_token_stride, a.state_out = y.data_ptr(), shape[1] * shape[2], shape[2], _ptr(last)
    _lib.launch('sq_causal_conv_forward', device, C.byref(a))
    return y, last


def conv_backward(shape, dtype, x, packed, weight, bias, state, lengths, silu, dy, dlast, want_weight, want_bias, want_state):
    """(dx, dweight, dbias, dstate) on checked arguments."""
    device = weight.device
    dx = torch.empty(shape, dtype=dtype, device=device)
    dweight = torch.empty_like(weight) if want_weight else None
    dbias = torch.empty_like(bias) if want_bias else None
    dstate = torch.empty_like(state) if want_state else None
    nbytes = int(_lib.load().sq_causal_conv_workspace(*shape))
    work = torch.empty(nbytes, dtype=torch.uint8, device=device)
    a = conv_args(shape, dtype, x, packed, weight, bias, state, lengths, silu)
    a.dy, a.dy_batch_stride, a.dy_token_stride, a.dstate_out = dy.data_ptr(), dy.stride(0), dy.stride(1), _ptr(dlast)
    a.dx, a.dstate_in, a.dweight, a.dbias = dx.data_ptr(), _ptr(dstate), _ptr(dweight), _ptr(dbias)
    a.workspace, a.workspace_bytes = work.data_ptr(), nbytes
    _lib.launch('sq_causal_conv_backward', device, C.byref(a))
    return dx, dweight, dbias, dstate


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu, want_state, keep):
        packed = empty_packed(x.shape, x.dtype, x.device) if keep else None
        y, last = conv_forward(x.shape, x.dtype, x, packed, weight, bias, state, lengths, silu, want_state)
        ctx.save_for_backward(weight, bias, state, lengths, *(packed[:2] if keep else (x,)))
        ctx.shape, ctx.dtype, ctx.silu = x.shape, x.dtype, silu
        ctx.set_materialize_grads(False)
        return (y, last) if want_state else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast=None):
        weight, bias, state, lengths, *kept = ctx.saved_tensors
        # Hooks on saved tensors (offloading, recomputation) may have put them elsewhere, with other strides.
        weight, bias, state, lengths = (None if t is None else t.contiguous() for t in (weight, bias, state, lengths))
        x = packed = None
        if len(kept) == 2:
            packed = PackedActivations(kept[0].contiguous(), kept[1].contiguous(), ctx.dtype)
        else:
            x = inner_packed(kept[0], 1)
        dy = torch.zeros(ctx.shape, dtype=ctx.dtype, device=weight.device) if dy is None else inner_packed(dy, 1)
        dlast = None if dlast is None else dlast.contiguous()
        need = ctx.needs_input_grad
        dx, dweight, dbias, dstate = conv_backward(ctx.shape, ctx.dtype, x, packed, weight, bias, state, lengths, ctx.silu, dy,
                                                   dlast, need[1], need[2], need[3])
        return dx, dweight, dbias, dstate, None, None, None, None


def causal_conv(x, weight, bias=None, initial_state=None, lengths=None, activation='silu', return_final_state=False, keep=None):
    """The convolution of x [batch, length, channels] (fp16, bf16 or fp32) with weight [channels, taps] and bias
    [channels], both in x's dtype or fp32: y [batch, length, channels], or (y, final state) with return_final_state.

    initial_state [batch, taps-1, channels] in x's dtype: the inputs before the first token, oldest first.
    lengths int32 [batch]: tokens of each sequence; those behind are not read, and zero in y and in the gradient.
    Differentiable in x, weight, bias and the states; keep='int8' keeps x in 8 bits for that."""
    if not isinstance(x, torch.Tensor) or x.dtype not in TYPES or not x.is_cuda or x.ndim != 3 or 0 in x.shape:
        raise ValueError('x must be CUDA FP16, BF16 or FP32 [batch,length,channels]')
    batch, _, channels = x.shape
    silu = _silu(activation)
    checked_keep(keep)
    weight, bias = checked_weight(weight, bias, channels, x.dtype, x.device)
    lengths = checked_lengths(lengths, batch, x.device)
    if initial_state is not None:
        if not isinstance(initial_state, torch.Tensor) or initial_state.shape != (batch, weight.shape[1] - 1, channels) \
                or initial_state.dtype != x.dtype or initial_state.device != x.device:
            raise ValueError(f"initial_state must be [{batch}, {weight.shape[1] - 1}, {channels}] in x's dtype, on its device")
        initial_state = initial_state.contiguous()
    _lib.refuse_tangents('causal_conv', x, weight, bias, initial_state)
    x = inner_packed(x, 1)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, initial_state)):
        return _CausalConv.apply(x, weight, bias, initial_state, lengths, silu, bool(return_final_state), keep)
    y, last = conv_forward(x.shape, x.dtype, x, None, weight, bias, initial_state, lengths, silu, return_final_state)
    return (y, last) if return_final_state else y


@torch.no_grad()
def causal_conv_step(x, state, weight, bias=None, activation='silu'):
    """One token x [batch, channels] of each row: y [batch, channels]; the row's state [batch, taps-1, channels] (the
    inputs before it, oldest first, contiguous, in x's dtype) moves on by it in place."""
    if not isinstance(x, torch.Tensor) or x.dtype not in TYPES or not x.is_cuda or x.ndim != 2 or 0 in x.shape:
        raise ValueError('x must be CUDA FP16, BF16 or FP32 [batch,channels]')
    batch, channels = x.shape
    silu = _silu(activation)
    weight, bias = checked_weight(weight, bias, channels, x.dtype, x.device)
    if not isinstance(state, torch.Tensor) or state.shape != (batch, weight.shape[1] - 1, channels) or state.dtype != x.dtype \
            or state.device != x.device or not state.is_contiguous():
        raise ValueError(f"state must be contiguous [{batch}, {weight.shape[1] - 1}, {channels}] in x's dtype, on its device")
    _lib.refuse_tangents('causal_conv_step', x, weight, bias, state)
    x = inner_packed(x, 1)
    y = torch.empty(batch, channels, dtype=x.dtype, device=x.device)
    _lib.launch('sq_causal_conv_step', x.device, x.data_ptr(), x.stride(0), state.data_ptr(), weight.data_ptr(), _ptr(bias),
                y.data_ptr(), batch, channels, weight.shape[1], silu, TYPES[x.dtype], TYPES[weight.dtype])
    written(state)
    return y
