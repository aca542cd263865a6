"""Convolution and selective scan of a mixer in one call: prompts and gradients (`conv_scan`), single tokens
(`conv_scan_step`).

Taken one after the other they keep for the backward pass the convolution's input and its output.  `conv_scan` keeps the
input alone and computes the output again; with keep='int8' it keeps the input in 8 bits, 1.03 bytes a channel and token
in place of four.  The output is then that of the given input, and the gradients are those at the kept values.
`conv_scan_step` has the convolution's output in fp32 on its way to the state.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .activations import TYPES, PackedActivations, empty_packed
from .conv import _ptr, checked_keep, checked_lengths, checked_weight, conv_backward, conv_forward, inner_packed
from .selective import _HALF, N, checked_heads, checked_state, scan_backward, scan_forward

__all__ = ['conv_scan', 'conv_scan_step']


def _split(z, heads, groups):
    """x, B and C of the convolution's channels, as views."""
    batch, length, width = z.shape
    inner = width - 2 * groups * N
    return (z[:, :, :inner].view(batch, length, heads, inner // heads), z[:, :, inner:inner + groups * N].view(batch, length, groups, N),
            z[:, :, inner + groups * N:].view(batch, length, groups, N))


class _ConvScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, xbc, dt, A, weight, bias, D, dt_bias, conv_state, state, lengths, heads, groups, want_state, keep):
        packed = empty_packed(xbc.shape, xbc.dtype, xbc.device) if keep else None
        z, conv_last = conv_forward(xbc.shape, xbc.dtype, xbc, packed, weight, bias, conv_state, lengths, 1, want_state)
        x, B, C_ = _split(z, heads, groups)
        y, last = scan_forward(x, dt, A, B, C_, D, dt_bias, state, lengths, want_state)
        ctx.save_for_backward(dt, A, weight, bias, D, dt_bias, conv_state, state, lengths, *(packed[:2] if keep else (xbc,)))
        ctx.shape, ctx.dtype, ctx.heads, ctx.groups = xbc.shape, xbc.dtype, heads, groups
        ctx.set_materialize_grads(False)
        return (y, conv_last, last) if want_state else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dconv_last=None, dlast=None):
        dt, A, weight, bias, D, dt_bias, conv_state, state, lengths, *kept = ctx.saved_tensors
        # Hooks on saved tensors (offloading, recomputation) may have put them elsewhere, with other strides.
        dt = inner_packed(dt, 1)
        A, weight, bias, D, dt_bias, conv_state, state, lengths = (
            None if t is None else t.contiguous() for t in (A, weight, bias, D, dt_bias, conv_state, state, lengths))
        xbc = packed = None
        if len(kept) == 2:
            packed = PackedActivations(kept[0].contiguous(), kept[1].contiguous(), ctx.dtype)
        else:
            xbc = inner_packed(kept[0], 1)
        conv = (ctx.shape, ctx.dtype, xbc, packed, weight, bias, conv_state, lengths, 1)
        x, B, C_ = _split(conv_forward(*conv)[0], ctx.heads, ctx.groups)
        dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else inner_packed(dy, 2)
        need = ctx.needs_input_grad
        dz = torch.empty(ctx.shape, dtype=ctx.dtype, device=x.device)
        ddt, dA, dD, ddt_bias, dstate = scan_backward(x, dt, A, B, C_, D, dt_bias, state, lengths, dy,
                                                      None if dlast is None else dlast.contiguous(), *_split(dz, ctx.heads, ctx.groups),
                                                      (need[2], need[5], need[6], need[8]))
        dxbc, dweight, dbias, dconv_state = conv_backward(*conv, dz, None if dconv_last is None else dconv_last.contiguous(),
                                                          need[3], need[4], need[7])
        return dxbc, ddt, dA, dweight, dbias, dD, ddt_bias, dconv_state, dstate, None, None, None, None, None


def _checked(xbc, dt, A, conv_weight, conv_bias, D, dt_bias, heads, groups, lead):
    """Checks that a prompt's and a token's call share; returns A, weight, bias, D, dt_bias and the rows of a head."""
    for name, v in (('heads', heads), ('groups', groups)):
        if isinstance(v, bool) or not isinstance(v, int) or v < 1:
            raise ValueError(f'{name} must be a positive integer')
    width, device = xbc.shape[-1], xbc.device
    inner = width - 2 * groups * N
    if heads % groups or inner < heads or inner % heads:
        raise ValueError('xbc must have heads*dim + 2*groups*128 channels, with heads divisible by groups')
    if not isinstance(dt, torch.Tensor) or dt.shape != (*lead, heads) or dt.dtype != xbc.dtype \
            or dt.get_device() != device.index:
        raise ValueError(f"dt must be {[*lead, heads]} in xbc's dtype, on its device")
    weight, bias = checked_weight(conv_weight, conv_bias, width, xbc.dtype, device)
    A, D, dt_bias = checked_heads(A, D, dt_bias, heads, device)
    return A, weight, bias, D, dt_bias, inner // heads


def _checked_conv_state(conv_state, batch, weight, xbc):
    if conv_state is None:
        return None
    shape = (batch, weight.shape[1] - 1, xbc.shape[-1])
    if not isinstance(conv_state, torch.Tensor) or conv_state.shape != shape or conv_state.dtype != xbc.dtype or conv_state.device != xbc.device:
        raise ValueError(f"conv_state must be {list(shape)} in xbc's dtype, on its device")
    return conv_state.contiguous()


def conv_scan(xbc, dt, A, conv_weight, conv_bias=None, D=None, dt_bias=None, *, heads, groups, conv_state=None, initial_state=None,
              lengths=None, return_final_state=False, keep=None):
    """selective_scan of the silu convolution of xbc [batch, length, heads*dim + 2*groups*128] (fp16 or bf16; x, B and C side
    by side as the model's in_proj gives them): y [batch, length, heads, dim], or (y, final conv_state, final state) with
    return_final_state.  dt [batch, length, heads] in xbc's dtype; the other arguments are those of `causal_conv` and
    `selective_scan`.  Differentiable in every tensor but lengths; keep='int8' keeps xbc in 8 bits for that."""
    if not isinstance(xbc, torch.Tensor) or xbc.dtype not in _HALF or not xbc.is_cuda or xbc.ndim != 3 or 0 in xbc.shape:
        raise ValueError('xbc must be CUDA FP16 or BF16 [batch,length,channels]')
    batch, length, _ = xbc.shape
    device = xbc.device
    checked_keep(keep)
    A, weight, bias, D, dt_bias, dim = _checked(xbc, dt, A, conv_weight, conv_bias, D, dt_bias, heads, groups, (batch, length))
    conv_state = _checked_conv_state(conv_state, batch, weight, xbc)
    state = checked_state(initial_state, (batch, heads, dim, N), device)
    lengths = checked_lengths(lengths, batch, device)
    xbc, dt = inner_packed(xbc, 1), inner_packed(dt, 1)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (xbc, dt, A, weight, bias, D, dt_bias, conv_state, state)):
        return _ConvScan.apply(xbc, dt, A, weight, bias, D, dt_bias, conv_state, state, lengths, heads, groups,
                               bool(return_final_state), keep)
    z, conv_last = conv_forward(xbc.shape, xbc.dtype, xbc, None, weight, bias, conv_state, lengths, 1, return_final_state)
    x, B, C_ = _split(z, heads, groups)
    y, last = scan_forward(x, dt, A, B, C_, D, dt_bias, state, lengths, return_final_state)
    return (y, conv_last, last) if return_final_state else y


@torch.no_grad()
def conv_scan_step(xbc, dt, A, conv_weight, conv_bias=None, D=None, dt_bias=None, *, heads, groups, conv_state, state):
    """One token of each row: y [batch, heads, dim] of xbc [batch, heads*dim + 2*groups*128] (fp16 or bf16) and dt
    [batch, heads]; conv_state [batch, taps-1, channels] and state fp32 [batch, heads, dim, 128], both contiguous, move on in
    place."""
    if not isinstance(xbc, torch.Tensor) or xbc.dtype not in _HALF or not xbc.is_cuda or xbc.ndim != 2 or 0 in xbc.shape:
        raise ValueError('xbc must be CUDA FP16 or BF16 [batch,channels]')
    batch, width = xbc.shape
    device = xbc.device
    A, weight, bias, D, dt_bias, dim = _checked(xbc, dt, A, conv_weight, conv_bias, D, dt_bias, heads, groups, (batch,))
    for name, given, held in (('conv_state', conv_state, _checked_conv_state(conv_state, batch, weight, xbc)),
                              ('state', state, checked_state(state, (batch, heads, dim, N), device, 'state'))):
        if given is None or held is not given:
            raise ValueError(f'{name} must be given, and contiguous: it is updated in place')
    xbc, dt = inner_packed(xbc, 1), inner_packed(dt, 1)
    y = torch.empty(batch, heads, dim, dtype=xbc.dtype, device=device)
    work = torch.empty(batch, width, dtype=torch.float32, device=device)
    a = _lib.ConvScanStepArgs(batch, heads, dim, groups, weight.shape[1], TYPES[xbc.dtype], TYPES[weight.dtype],
                              xbc.data_ptr(), xbc.stride(0), dt.data_ptr(), dt.stride(0), A.data_ptr(), weight.data_ptr(), _ptr(bias),
                              _ptr(D), 0 if D is None else TYPES[D.dtype], _ptr(dt_bias), 0 if dt_bias is None else TYPES[dt_bias.dtype],
                              conv_state.data_ptr(), state.data_ptr(), y.data_ptr(), work.data_ptr(), batch * width * 4)
    _lib.launch('sq_conv_scan_step', device, C.byref(a))
    return y
