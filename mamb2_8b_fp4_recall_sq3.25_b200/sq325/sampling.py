"""Drawing tokens from rows of logits (sq_sample): temperature, top-k, top-p and min-p, from
uniform numbers the caller gives.

With m the row's largest logit, y_j = 2^((x_j - m) log2(e) / temperature) and the whole weight
w_j = rint(y_j 2^31).  Tokens are ordered by logit, equal ones by index.  The settings apply in
this order: top-k keeps the first k tokens, top-p those whose predecessors hold less than
top_p of the kept weight (the first always), min-p those with y_j >= min_p.  The token drawn is
the first in index order at which the running weight passes floor(uniform * total), the product
in 64-bit floating point.  Weights and sums are integers, so the same inputs give the same token
whatever the launch shape.  Uniform numbers are fp32: on a grid of 2^-24, a token whose share of the
weight is smaller than that is drawn only where a grid point falls on it.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

__all__ = ['sample']

MAX_VOCAB = 1 << 18
_TYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


def logits_rows(logits):
    """Checks a tensor of logits [..., vocab] and returns it as rows [n, vocab] whose last
    dimension is contiguous (a copy only where its layout has no single row stride)."""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _TYPES or not logits.is_cuda:
        raise ValueError('Logits must be a CUDA FP16, BF16 or FP32 tensor')
    shape = logits.shape
    if not shape or not 1 <= shape[-1] <= MAX_VOCAB:
        raise ValueError(f'Logits must be [..., vocab] with vocab in [1, {MAX_VOCAB}]')
    x = logits if len(shape) == 2 else logits.reshape(-1, shape[-1])
    return x if x.stride(1) == 1 or shape[-1] == 1 else x.contiguous()


def row_numbers(x, lead):
    """An empty fp32 tensor with a number a row of x, of shape `lead`."""
    out = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    return out if len(lead) == 1 else out.view(lead)


def logits_fields(x):
    """The fields of an sq_logits for rows that logits_rows() returned."""
    rows, vocab = x.shape
    return x.data_ptr(), x.stride(0), rows, vocab, _TYPES[x.dtype]


def _per_row(name, value, x, lead, dtype):
    """A tensor with one setting a row."""
    if value.shape != lead or value.dtype != dtype or value.get_device() != x.get_device():
        raise ValueError(f'{name} must be a number or a {dtype} tensor of shape {tuple(lead)} on {x.device}')
    return value.contiguous()


def _number(name, value, kinds, low, high):
    if isinstance(value, bool) or not isinstance(value, kinds) or not low <= value <= high:
        raise ValueError(f'{name} is out of range: {value!r}')


def sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Draws one token per row of logits [..., vocab]: int64 [...].

    logits: fp16, bf16 or fp32 on the GPU; NaN counts as masked (-inf).
    uniform: fp32 [...] numbers in [0, 1), one a row.
    temperature >= 0 (0: the largest logit, lowest index), top_k >= 0 (0: off), top_p in (0, 1]
    (1: off), min_p in [0, 1] (0: off): a number for all rows, or a tensor [...] on the device
    (fp32, top_k int32) with a setting per row, whose values are the caller's to check.
    A row with nothing above -inf gives -1.
    """
    x = logits_rows(logits)
    lead = logits.shape[:-1]
    if not isinstance(uniform, torch.Tensor) or uniform.shape != lead or uniform.dtype != torch.float32 \
            or uniform.get_device() != x.get_device():
        raise ValueError(f'uniform must be a float32 tensor of shape {tuple(lead)} on {x.device}')
    uniform = uniform.contiguous()
    t = k = p = q = None                         # addresses of per-row settings
    kept = []                                    # alive until the launch
    if isinstance(temperature, torch.Tensor):
        kept.append(_per_row('temperature', temperature, x, lead, torch.float32))
        t, temperature = kept[-1].data_ptr(), 0.0
    elif type(temperature) is not float or not 0 <= temperature <= 3.4e38:
        _number('temperature', temperature, (int, float), 0, 3.4e38)
    if isinstance(top_k, torch.Tensor):
        kept.append(_per_row('top_k', top_k, x, lead, torch.int32))
        k, top_k = kept[-1].data_ptr(), 0
    elif type(top_k) is not int or not 0 <= top_k < 2 ** 31:
        _number('top_k', top_k, int, 0, 2 ** 31 - 1)
    if isinstance(top_p, torch.Tensor):
        kept.append(_per_row('top_p', top_p, x, lead, torch.float32))
        p, top_p = kept[-1].data_ptr(), 0.0
    elif type(top_p) is not float or not 0 < top_p <= 1:
        _number('top_p', top_p, (int, float), 5e-324, 1)
    if isinstance(min_p, torch.Tensor):
        kept.append(_per_row('min_p', min_p, x, lead, torch.float32))
        q, min_p = kept[-1].data_ptr(), 0.0
    elif type(min_p) is not float or not 0 <= min_p <= 1:
        _number('min_p', min_p, (int, float), 0, 1)
    tokens = torch.empty_like(uniform, dtype=torch.long)
    a = _lib.SampleArgs(*logits_fields(x), uniform.data_ptr(), t, k, p, q, temperature, top_k, top_p, min_p, tokens.data_ptr())
    _lib.launch('sq_sample', x.device, C.byref(a))
    return tokens
