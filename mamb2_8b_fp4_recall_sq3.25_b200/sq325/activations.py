"""Activations in 8 bits (sq_pack_activations, sq_unpack_activations), for what a backward pass keeps.

In the last axis each 128 neighbouring values (the last block may have fewer) share scale = max|x| (1 / 127) in fp32 and
are kept as codes rint(x / scale): 1.03 bytes a value, off by at most half a scale.  A block with a NaN or an infinity
comes back as NaN.  `causal_conv(..., keep='int8')` and `conv_scan(..., keep='int8')` keep their input in this form.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

__all__ = ['PackedActivations', 'pack_activations', 'unpack_activations']

BLOCK = 128
TYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


class PackedActivations(NamedTuple):
    """codes int8 [..., width], scales fp32 [..., ceil(width / 128)], and the type that was packed."""
    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype


def empty_packed(shape, dtype, device):
    """An unwritten record for activations of `shape`."""
    return PackedActivations(torch.empty(shape, dtype=torch.int8, device=device),
                             torch.empty(*shape[:-1], -(-shape[-1] // BLOCK), dtype=torch.float32, device=device), dtype)


def pack_activations(x):
    """Activations [..., width] (fp16, bf16 or fp32 on the GPU) in 8 bits.  Receives no gradient."""
    if not isinstance(x, torch.Tensor) or x.dtype not in TYPES or not x.is_cuda:
        raise ValueError('Activations must be a CUDA FP16, BF16 or FP32 tensor')
    shape = x.shape
    if not shape or shape[-1] < 1:
        raise ValueError('Activations must be [..., width] with a positive width')
    x = x.detach()
    rows = x if x.ndim == 2 else x.reshape(-1, shape[-1])
    if rows.stride(1) != 1 and shape[-1] > 1:
        rows = rows.contiguous()
    out = empty_packed(shape, x.dtype, x.device)
    _lib.launch('sq_pack_activations', x.device, rows.data_ptr(), rows.stride(0), rows.shape[0], shape[-1], TYPES[x.dtype],
                out.codes.data_ptr(), out.scales.data_ptr())
    return out


def unpack_activations(packed, dtype=None):
    """The values that a record holds, code * scale rounded to `dtype` (None: the type that was packed)."""
    if not isinstance(packed, tuple) or len(packed) != 3:
        raise ValueError('unpack_activations takes what pack_activations returned')
    codes, scales, was = packed
    dtype = was if dtype is None else dtype
    if dtype not in TYPES:
        raise ValueError('dtype must be FP16, BF16 or FP32')
    if not isinstance(codes, torch.Tensor) or not isinstance(scales, torch.Tensor) or codes.dtype != torch.int8 \
            or scales.dtype != torch.float32 or not codes.is_cuda or scales.device != codes.device or not codes.shape \
            or codes.shape[-1] < 1 or scales.shape != (*codes.shape[:-1], -(-codes.shape[-1] // BLOCK)):
        raise ValueError('Codes must be CUDA int8 [..., width] with a positive width, scales fp32 [..., ceil(width / 128)] on the same device')
    codes, scales = codes.contiguous(), scales.contiguous()
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    rows = codes.numel() // codes.shape[-1]
    _lib.launch('sq_unpack_activations', codes.device, codes.data_ptr(), scales.data_ptr(), rows, codes.shape[-1], TYPES[dtype],
                out.data_ptr())
    return out
