"""Distillation from a teacher's largest logits (sq_top_logits, sq_distill_*).

The teacher's record of a token is its k largest logits and their indices (`top_logits`).  With
q the softmax of the recorded logits / T over the record and p the student's softmax of its
logits / T over the whole vocabulary,

    loss = T^2 sum_k q_k (log q_k - log p_jk),    d loss / d s_j = T (p_j - q_j)

(q_j = 0 outside the record).  `distillation_loss` is differentiable in the student's logits: its
backward reads the logits again and recomputes p from the row's maximum and sum.
`distillation_loss_grad` gives loss and gradient in one call, for steps that know each row's
weight beforehand.  Sums are fp32, the gradient is rounded once to the logits' type.  Any
positive finite temperature is computed; a loss past fp32's range (temperatures of about 1e19) is infinite.  Places of
the record with an index outside the vocabulary or a value of -inf or NaN are unused; a row
without used places has loss 0 and gradient 0.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .sampling import _TYPES, logits_fields, logits_rows, row_numbers

__all__ = ['top_logits', 'distillation_loss', 'distillation_loss_grad']

MAX_RECORD = 1024


def top_logits(logits, k):
    """The k largest of each row of logits [..., vocab], largest first and equal ones by index:
    (values [..., k] in the logits' dtype, indices int32 [..., k]).  k in [1, min(1024, vocab)].
    NaN and -inf are not taken; places left over hold -inf and -1."""
    x = logits_rows(logits)
    if isinstance(k, bool) or not isinstance(k, int) or not 1 <= k <= min(MAX_RECORD, x.shape[1]):
        raise ValueError(f'k must be an integer in [1, min({MAX_RECORD}, vocab)]')
    values = torch.empty(*logits.shape[:-1], k, dtype=x.dtype, device=x.device)
    indices = torch.empty_like(values, dtype=torch.int32)
    _lib.launch('sq_top_logits', x.device, C.byref(_lib.Logits(*logits_fields(x))), k, values.data_ptr(), indices.data_ptr())
    return values, indices


def _checked(logits, values, indices, temperature):
    x = logits_rows(logits)
    if not isinstance(values, torch.Tensor) or not isinstance(indices, torch.Tensor):
        raise ValueError('The record must be two tensors, values and indices')
    shape, lead = values.shape, logits.shape[:-1]
    if shape != indices.shape or not shape or shape[:-1] != lead:
        raise ValueError('The record must be values and indices [..., k] with the leading shape of the logits')
    if not 1 <= shape[-1] <= MAX_RECORD:
        raise ValueError(f'The record must have 1 to {MAX_RECORD} entries a row')
    device = x.get_device()
    if values.dtype not in _TYPES or indices.dtype != torch.int32 or values.get_device() != device \
            or indices.get_device() != device:
        raise ValueError('The record must be FP16, BF16 or FP32 values and int32 indices on the device of the logits')
    if values.requires_grad:
        raise ValueError("The teacher's record receives no gradient: detach it")
    if isinstance(temperature, bool) or not isinstance(temperature, (int, float)) or not 0 < temperature <= 3e38:
        raise ValueError('temperature must be a positive finite number')
    return x, values.contiguous(), indices.contiguous(), lead


def _args(x, values, indices, temperature, loss=None, weight=None, stats=None, grad=None):
    return _lib.DistillArgs(*logits_fields(x), values.data_ptr(), indices.data_ptr(), values.shape[-1], _TYPES[values.dtype],
                            temperature, None if weight is None else weight.data_ptr(),
                            0 if weight is None else weight.stride(0), None if loss is None else loss.data_ptr(),
                            None if stats is None else stats.data_ptr(), None if grad is None else grad.data_ptr(),
                            x.shape[1])


def _row_weights(weight):
    """Per-row factors as a vector the kernels step through: a broadcast one keeps its stride of 0."""
    return weight if weight.ndim == 1 else weight.reshape(-1)


class _DistillationLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, values, indices, temperature):
        x, values, indices, lead = _checked(logits, values, indices, temperature)
        loss = row_numbers(x, lead)
        stats = torch.empty(x.shape[0], 4, dtype=torch.float32, device=x.device)
        ctx.save_for_backward(x, values, indices, stats)
        ctx.shape, ctx.temperature = logits.shape, temperature
        _lib.launch('sq_distill_forward', x.device, C.byref(_args(x, values, indices, temperature, loss=loss, stats=stats)))
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        x, values, indices, stats = ctx.saved_tensors       # raises if one of them was changed in place
        # Hooks on saved tensors (offloading, recomputation) may have put them elsewhere, with other strides.
        x, values, indices, stats = logits_rows(x), values.contiguous(), indices.contiguous(), stats.contiguous()
        weight = _row_weights(grad_loss)
        grad = torch.empty(*ctx.shape, dtype=x.dtype, device=x.device)
        _lib.launch('sq_distill_backward', x.device,
                    C.byref(_args(x, values, indices, ctx.temperature, weight=weight, stats=stats, grad=grad)))
        return grad, None, None, None


def distillation_loss(logits, values, indices, temperature=1.0):
    """Per-row distillation loss, fp32 [...], of the student's logits [..., vocab] against the
    teacher's record (values [..., k], int32 indices [..., k], k <= 1024).  Differentiable in the
    logits; the record receives no gradient."""
    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        return _DistillationLoss.apply(logits, values, indices, temperature)
    x, values, indices, lead = _checked(logits, values, indices, temperature)
    loss = row_numbers(x, lead)
    _lib.launch('sq_distill_forward', x.device, C.byref(_args(x, values, indices, temperature, loss=loss)))
    return loss


def distillation_loss_grad(logits, values, indices, temperature=1.0, weight=None):
    """(loss fp32 [...], gradient [..., vocab] in the logits' dtype) in one call.  weight: fp32
    [...] factor of each row's gradient (None: 1), as the upstream gradient of the loss would be;
    the loss itself is not weighted."""
    x, values, indices, lead = _checked(logits, values, indices, temperature)
    if weight is not None:
        if not isinstance(weight, torch.Tensor) or weight.shape != lead or weight.dtype != torch.float32 \
                or weight.get_device() != x.get_device():
            raise ValueError(f'weight must be a float32 tensor of shape {tuple(lead)} on {x.device}')
        weight = _row_weights(weight)
    loss = row_numbers(x, lead)
    grad = torch.empty(*logits.shape, dtype=x.dtype, device=x.device)
    _lib.launch('sq_distill_loss_grad', x.device,
                C.byref(_args(x, values, indices, temperature, weight=weight, loss=loss, grad=grad)))
    return loss, grad
