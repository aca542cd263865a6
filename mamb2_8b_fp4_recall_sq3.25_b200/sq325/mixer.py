"""Convolution and selective scan of a mixer in one call: prompts and gradients (`conv_scan`), single tokens
(`conv_scan_step`).

Taken one after the other they keep for the backward pass the convolution's input and its output.  `conv_scan` keeps the
input alone and computes the output again; with keep='int8' it keeps the input in 8 bits, 1.03 bytes a channel and token
in place of four.  The output is then that of the given input, and the gradients are those at the kept values.  A call's
workspace, which it gives back, is larger than what is kept (2 x 2,048 tokens at 128 heads: 233 MB forward, 619 MB backward).  Between
the two the convolution's output is scaled fp16 (11 bits, down to 2^-28 of a tile's largest value, also where the input is
bf16), its gradient fp32; in `conv_scan_step` the output is fp32.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib
from .activations import TYPES, PackedActivations, pack_activations
from .conv import _ptr, checked_keep, checked_lengths, checked_weight, conv_args, inner_packed, written
from .selective import _HALF, N, checked_heads, checked_state

__all__ = ['conv_scan', 'conv_scan_step']


@functools.lru_cache(maxsize=256)
def _workspace_bytes(batch, length, heads, dim, groups, backward):
    return int(_lib.load().sq_conv_scan_workspace(batch, length, heads, dim, groups, backward))


def _args(shape, dtype, xbc, packed, dt, A, weight, bias, D, dt_bias, conv_state, state, lengths, heads, groups, backward):
    """The arguments of convolution and scan that forward and backward share, and the workspace."""
    batch, length, width = shape
    dim = (width - 2 * groups * N) // heads
    conv = conv_args(shape, dtype, xbc, packed, weight, bias, conv_state, lengths, 1)
    scan = _lib.SelectiveArgs(batch, length, heads, dim, groups, TYPES[dtype])
    scan.dt, scan.dt_batch_stride, scan.dt_token_stride, scan.A = dt.data_ptr(), dt.stride(0), dt.stride(1), A.data_ptr()
    if D is not None:
        scan.D, scan.d_type = D.data_ptr(), TYPES[D.dtype]
    if dt_bias is not None:
        scan.dt_bias, scan.bias_type = dt_bias.data_ptr(), TYPES[dt_bias.dtype]
    scan.state_in, scan.lengths = _ptr(state), _ptr(lengths)
    nbytes = _workspace_bytes(batch, length, heads, dim, groups, backward)
    work = torch.empty(nbytes, dtype=torch.uint8, device=dt.device)
    scan.workspace, scan.workspace_bytes = work.data_ptr(), nbytes
    return conv, scan, work


def _forward(xbc, dt, A, weight, bias, D, dt_bias, conv_state, state, lengths, heads, groups, want_state):
    """(y, last inputs or None, state or None) of checked tensors."""
    batch, length, width = xbc.shape
    dim = (width - 2 * groups * N) // heads
    device = xbc.device
    conv, scan, work = _args(xbc.shape, xbc.dtype, xbc, None, dt, A, weight, bias, D, dt_bias, conv_state, state, lengths, heads, groups, 0)
    y = torch.empty(batch, length, heads, dim, dtype=xbc.dtype, device=device)
    conv_last = torch.empty(batch, weight.shape[1] - 1, width, dtype=xbc.dtype, device=device) if want_state else None
    last = torch.empty(batch, heads, dim, N, dtype=torch.float32, device=device) if want_state else None
    conv.state_out, scan.state_out = _ptr(conv_last), _ptr(last)
    scan.y, scan.y_batch_stride, scan.y_token_stride = y.data_ptr(), length * heads * dim, heads * dim
    _lib.launch('sq_conv_scan_forward', device, C.byref(conv), C.byref(scan))
    del work                                                 # alive until the launch
    return y, conv_last, last


class _ConvScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, xbc, dt, A, weight, bias, D, dt_bias, conv_state, state, lengths, heads, groups, want_state, keep):
        y, conv_last, last = _forward(xbc, dt, A, weight, bias, D, dt_bias, conv_state, state, lengths, heads, groups, want_state)
        kept = pack_activations(xbc)[:2] if keep else (xbc,)
        ctx.save_for_backward(dt, A, weight, bias, D, dt_bias, conv_state, state, lengths, *kept)
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
        batch, length, width = ctx.shape
        device, heads, need = dt.device, ctx.heads, ctx.needs_input_grad
        if dy is None:
            dy = torch.zeros(batch, length, heads, (width - 2 * ctx.groups * N) // heads, dtype=ctx.dtype, device=device)
        else:
            dy = inner_packed(dy, 2)
        dconv_last, dlast = (None if t is None else t.contiguous() for t in (dconv_last, dlast))
        conv, scan, work = _args(ctx.shape, ctx.dtype, xbc, packed, dt, A, weight, bias, D, dt_bias, conv_state, state, lengths, heads,
                                 ctx.groups, 1)
        dxbc = torch.empty(ctx.shape, dtype=ctx.dtype, device=device)
        ddt = torch.empty(dt.shape, dtype=dt.dtype, device=device)
        dA, dweight, dbias, dD, ddt_bias, dconv_state, dstate = (
            torch.empty_like(t) if need[i] else None for i, t in ((2, A), (3, weight), (4, bias), (5, D), (6, dt_bias), (7, conv_state), (8, state)))
        conv.dx, conv.dweight, conv.dbias, conv.dstate_in, conv.dstate_out = dxbc.data_ptr(), _ptr(dweight), _ptr(dbias), _ptr(dconv_state), _ptr(dconv_last)
        scan.dy, scan.dy_batch_stride, scan.dy_token_stride, scan.dstate_out = dy.data_ptr(), dy.stride(0), dy.stride(1), _ptr(dlast)
        scan.ddt, scan.dA, scan.dD, scan.ddt_bias, scan.dstate_in = ddt.data_ptr(), _ptr(dA), _ptr(dD), _ptr(ddt_bias), _ptr(dstate)
        _lib.launch('sq_conv_scan_backward', device, C.byref(conv), C.byref(scan))
        del work                                             # alive until the launch
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
    _lib.refuse_tangents('conv_scan', xbc, dt, A, weight, bias, D, dt_bias, conv_state, state)
    xbc, dt = inner_packed(xbc, 1), inner_packed(dt, 1)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (xbc, dt, A, weight, bias, D, dt_bias, conv_state, state)):
        return _ConvScan.apply(xbc, dt, A, weight, bias, D, dt_bias, conv_state, state, lengths, heads, groups,
                               bool(return_final_state), keep)
    y, conv_last, last = _forward(xbc, dt, A, weight, bias, D, dt_bias, conv_state, state, lengths, heads, groups, bool(return_final_state))
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
    _lib.refuse_tangents('conv_scan_step', xbc, dt, A, weight, bias, D, dt_bias, conv_state, state)
    xbc, dt = inner_packed(xbc, 1), inner_packed(dt, 1)
    y = torch.empty(batch, heads, dim, dtype=xbc.dtype, device=device)
    work = torch.empty(batch, width, dtype=torch.float32, device=device)
    a = _lib.ConvScanStepArgs(batch, heads, dim, groups, weight.shape[1], TYPES[xbc.dtype], TYPES[weight.dtype],
                              xbc.data_ptr(), xbc.stride(0), dt.data_ptr(), dt.stride(0), A.data_ptr(), weight.data_ptr(), _ptr(bias),
                              _ptr(D), 0 if D is None else TYPES[D.dtype], _ptr(dt_bias), 0 if dt_bias is None else TYPES[dt_bias.dtype],
                              conv_state.data_ptr(), state.data_ptr(), y.data_ptr(), work.data_ptr(), batch * width * 4)
    _lib.launch('sq_conv_scan_step', device, C.byref(a))
    written(conv_state, state)
    return y
