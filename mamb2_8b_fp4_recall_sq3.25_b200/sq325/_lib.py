"""ctypes binding of the C ABI in include/sq325.h (libsq325.so, built in-tree for sm_100a).

There is no fallback: if the shared library is missing or a GPU call fails, the
error surfaces as an exception with the library's own message.  Status codes map to
the exception classes the reference raises for the same conditions
(ValueError / RuntimeError / FloatingPointError).
"""
from __future__ import annotations

import ctypes as C
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / 'libsq325.so'

SQ_OK, SQ_EINVAL, SQ_ESTATE, SQ_ENONFINITE, SQ_ECUDA, SQ_ETIMEOUT, SQ_ENOMEM = range(7)
ABI_VERSION = 1


class DeviceTimeout(RuntimeError):
    """A bounded device-side wait expired (SQ_ETIMEOUT); the CUDA context stays usable."""


_EXC = {SQ_EINVAL: ValueError, SQ_ESTATE: RuntimeError, SQ_ENONFINITE: FloatingPointError,
        SQ_ECUDA: RuntimeError, SQ_ETIMEOUT: DeviceTimeout, SQ_ENOMEM: MemoryError}

p = C.c_void_p
i32 = C.c_int32
i64 = C.c_int64


class ScanArgs(C.Structure):
    _fields_ = [('batch', i32), ('length', i32), ('heads', i32), ('dim', i32), ('groups', i32), ('layout', i32),
                ('x', p), ('x_batch_stride', i64), ('x_token_stride', i64),
                ('dt', p), ('dt_batch_stride', i64), ('dt_token_stride', i64),
                ('A', p),
                ('B', p), ('b_batch_stride', i64), ('b_token_stride', i64),
                ('C', p), ('c_batch_stride', i64), ('c_token_stride', i64),
                ('D', p), ('d_is_f32', i32), ('dt_bias', p), ('dt_bias_is_f32', i32),
                ('permutation', p), ('basis', p), ('latent_scale', p), ('predictor', p),
                ('lo', p), ('hi', p), ('q4', p), ('latent', p), ('s8', p), ('s4', p),
                ('y', p), ('y_batch_stride', i64), ('y_token_stride', i64),
                ('workspace', p), ('workspace_bytes', i64)]


class S16Args(C.Structure):
    _fields_ = [('batch', i32), ('length', i32), ('heads', i32), ('dim', i32), ('groups', i32),
                ('x', p), ('x_batch_stride', i64), ('x_token_stride', i64),
                ('dt', p), ('dt_batch_stride', i64), ('dt_token_stride', i64),
                ('A', p),
                ('B', p), ('b_batch_stride', i64), ('b_token_stride', i64),
                ('C', p), ('c_batch_stride', i64), ('c_token_stride', i64),
                ('D', p), ('d_is_f32', i32), ('dt_bias', p), ('dt_bias_is_f32', i32),
                ('state', p), ('y', p), ('y_batch_stride', i64), ('y_token_stride', i64), ('stats', p)]


class Sq3p25Args(C.Structure):
    _fields_ = [('batch', i32), ('length', i32), ('heads', i32), ('dim', i32), ('groups', i32),
                ('x', p), ('x_batch_stride', i64), ('x_token_stride', i64),
                ('dt', p), ('dt_batch_stride', i64), ('dt_token_stride', i64),
                ('A', p),
                ('B', p), ('b_batch_stride', i64), ('b_token_stride', i64),
                ('C', p), ('c_batch_stride', i64), ('c_token_stride', i64),
                ('D', p), ('d_is_f32', i32), ('dt_bias', p), ('dt_bias_is_f32', i32),
                ('permutation', p),
                ('lo', p), ('hi', p), ('q4', p), ('s8', p), ('s4', p),
                ('y', p), ('y_batch_stride', i64), ('y_token_stride', i64)]


class ConvArgs(C.Structure):
    _fields_ = [('weight', p), ('bias', p), ('ring', p), ('ring_batch_stride', i64), ('position', i32)]


class ModelConfig(C.Structure):
    _fields_ = [('n_layer', i32), ('vocab', i32), ('eps', C.c_float)]


class Fp4Matrix(C.Structure):
    _fields_ = [('codes', p), ('block_scales', p), ('global_scale', p), ('rows', i32), ('cols', i32)]


class LayerDesc(C.Structure):
    _fields_ = [('in_proj', Fp4Matrix), ('out_proj', Fp4Matrix), ('norm_weight', p), ('conv_weight', p),
                ('conv_bias', p), ('A', p), ('D', p), ('dt_bias', p), ('gated_norm_weight', p), ('layout', i32),
                ('permutation', p), ('basis', p), ('latent_scale', p), ('predictor', p)]


F16, BF16, F32 = range(3)


class Logits(C.Structure):
    _fields_ = [('data', p), ('row_stride', i64), ('rows', i32), ('vocab', i32), ('type', i32)]


# sq_sample_args and sq_distill_args begin with an sq_logits; its fields stand for themselves here (the same
# layout, one structure less to build per call)
class SampleArgs(C.Structure):
    _fields_ = [*Logits._fields_, ('uniform', p), ('temperature', p), ('top_k', p), ('top_p', p), ('min_p', p),
                ('temperature_all', C.c_float), ('top_k_all', i32), ('top_p_all', C.c_float), ('min_p_all', C.c_float),
                ('tokens', p)]


class DistillArgs(C.Structure):
    _fields_ = [*Logits._fields_, ('values', p), ('indices', p), ('k', i32), ('value_type', i32),
                ('temperature', C.c_float), ('weight', p), ('weight_stride', i64), ('loss', p), ('stats', p),
                ('grad', p), ('grad_stride', i64)]


class SelectiveArgs(C.Structure):
    _fields_ = [('batch', i32), ('length', i32), ('heads', i32), ('dim', i32), ('groups', i32), ('type', i32),
                ('x', p), ('x_batch_stride', i64), ('x_token_stride', i64),
                ('dt', p), ('dt_batch_stride', i64), ('dt_token_stride', i64),
                ('A', p),
                ('B', p), ('b_batch_stride', i64), ('b_token_stride', i64),
                ('C', p), ('c_batch_stride', i64), ('c_token_stride', i64),
                ('D', p), ('d_type', i32), ('dt_bias', p), ('bias_type', i32), ('state_in', p), ('lengths', p),
                ('y', p), ('y_batch_stride', i64), ('y_token_stride', i64), ('state_out', p),
                ('dy', p), ('dy_batch_stride', i64), ('dy_token_stride', i64), ('dstate_out', p),
                ('dx', p), ('dx_batch_stride', i64), ('dx_token_stride', i64), ('ddt', p),
                ('dB', p), ('dC', p), ('dg_batch_stride', i64), ('dg_token_stride', i64),
                ('dA', p), ('dD', p), ('ddt_bias', p), ('dstate_in', p),
                ('workspace', p), ('workspace_bytes', i64)]


class SelectiveStepArgs(C.Structure):
    _fields_ = [('batch', i32), ('heads', i32), ('dim', i32), ('groups', i32), ('type', i32),
                ('x', p), ('x_batch_stride', i64), ('dt', p), ('dt_batch_stride', i64), ('A', p),
                ('B', p), ('b_batch_stride', i64), ('C', p), ('c_batch_stride', i64),
                ('D', p), ('d_type', i32), ('dt_bias', p), ('bias_type', i32), ('state', p), ('y', p)]


class ConvScanStepArgs(C.Structure):
    _fields_ = [('batch', i32), ('heads', i32), ('dim', i32), ('groups', i32), ('taps', i32), ('type', i32), ('weight_type', i32),
                ('xbc', p), ('xbc_batch_stride', i64), ('dt', p), ('dt_batch_stride', i64), ('A', p), ('weight', p), ('bias', p),
                ('D', p), ('d_type', i32), ('dt_bias', p), ('bias_type', i32), ('conv_state', p), ('state', p), ('y', p),
                ('workspace', p), ('workspace_bytes', i64)]


class CausalConvArgs(C.Structure):
    _fields_ = [('batch', i32), ('length', i32), ('channels', i32), ('taps', i32), ('silu', i32), ('type', i32),
                ('weight_type', i32),
                ('x', p), ('x_batch_stride', i64), ('x_token_stride', i64), ('codes', p), ('scales', p),
                ('weight', p), ('bias', p), ('state_in', p), ('lengths', p),
                ('y', p), ('y_batch_stride', i64), ('y_token_stride', i64), ('state_out', p),
                ('dy', p), ('dy_batch_stride', i64), ('dy_token_stride', i64), ('dstate_out', p),
                ('dx', p), ('dstate_in', p), ('dweight', p), ('dbias', p),
                ('workspace', p), ('workspace_bytes', i64)]


# name -> (restype, argtypes)
_PROTOS = {
    'sq_abi_version': (C.c_int, []),
    'sq_last_error': (C.c_char_p, []),
    'sq_layout_index': (C.c_int, [C.c_char_p]),
    'sq_layout_counts': (C.c_int, [C.c_int, C.POINTER(C.c_int), C.POINTER(C.c_int), C.POINTER(C.c_int)]),
    'sq_state_bytes': (i64, [C.c_int, C.c_int, C.c_int]),
    'sq_scan': (C.c_int, [C.POINTER(ScanArgs), p]),
    'sq_scan_conv': (C.c_int, [C.POINTER(ScanArgs), C.POINTER(ConvArgs), p]),
    'sq_s16_scan': (C.c_int, [C.POINTER(S16Args), p]),
    'sq_sq3p25_scan': (C.c_int, [C.POINTER(Sq3p25Args), p]),
    'sq_ste_workspace': (i64, [C.c_int, C.c_int, C.c_int, C.c_int, C.c_int]),
    'sq_ste_backward': (C.c_int, [C.POINTER(Sq3p25Args), C.c_int, p, p, p, p, p, p, i64, p]),
    'sq_state_decode': (C.c_int, [C.c_int] * 5 + [p] * 9 + [p]),
    'sq_state_encode': (C.c_int, [C.c_int] * 6 + [p] * 9 + [p]),
    'sq_fp4_decode': (C.c_int, [p, p, p, C.c_int, C.c_int, p, i64, p]),
    'sq_fp4_validate': (C.c_int, [p, p, p, C.c_int, C.c_int, p]),
    'sq_scan_workspace': (i64, [C.c_int, C.c_int, C.c_int, C.c_int, C.c_int]),
    'sq_model_set_exact_skinny': (C.c_int, [p, C.c_int]),
    'sq_model_time_gemm': (C.c_int, [p, C.c_int]),
    'sq_model_gemm_time': (C.c_int, [p, C.POINTER(C.c_double), C.POINTER(i64)]),
    'sq_model_set_capture': (C.c_int, [p, p, i64]),
    'sq_model_decode': (C.c_int, [p, p, C.c_int, C.c_int, p, p]),
    'sq_fp4_linear_workspace': (i64, [C.c_int, C.c_int, C.c_int]),
    'sq_fp4_linear': (C.c_int, [p, p, p, C.c_int, C.c_int, p, i64, C.c_int, p, i64, p, i64, p]),
    'sq_fp4_linear_static_max_k': (i64, []),
    'sq_fp4_linear_static': (C.c_int, [p, p, p, C.c_int, C.c_int, p, i64, C.c_int, p, i64, p]),
    'sq_gemm_f16': (C.c_int, [p, i64, p, i64, p, i64, C.c_int, C.c_int, C.c_int, p]),
    'sq_device_check': (C.c_int, [p]),
    'sq_set_wait_limit_ns': (C.c_int, [C.c_uint64]),
    'sq_model_create': (C.c_int, [C.POINTER(ModelConfig), C.POINTER(p)]),
    'sq_model_destroy': (C.c_int, [p]),
    'sq_model_set_layer': (C.c_int, [p, C.c_int, C.POINTER(LayerDesc)]),
    'sq_model_set_globals': (C.c_int, [p, C.POINTER(Fp4Matrix), C.POINTER(Fp4Matrix), p]),
    'sq_model_set_adapter': (C.c_int, [p, C.c_int, p, p, p, p, C.c_int]),
    'sq_model_bind_state': (C.c_int, [p, C.c_int, C.c_int, p, p, p, p, p, p, p]),
    'sq_model_reserve': (C.c_int, [p, C.c_int]),
    'sq_model_forward': (C.c_int, [p, p, C.c_int, C.c_int, C.c_int, p, p]),
    'sq_model_mixer_forward': (C.c_int, [p, C.c_int, p, C.c_int, C.c_int, C.c_int, p, p]),
    'sq_model_score': (C.c_int, [p, p, C.c_int, p, p, p]),
    'sq_model_logits': (C.c_int, [p, p, C.c_int, p, p, i64, p]),
    'sq_model_greedy': (C.c_int, [p, p, C.c_int, p, p, p]),
    'sq_model_check': (C.c_int, [p, p]),
    'sq_sample': (C.c_int, [C.POINTER(SampleArgs), p]),
    'sq_top_logits': (C.c_int, [C.POINTER(Logits), C.c_int, p, p, p]),
    'sq_distill_forward': (C.c_int, [C.POINTER(DistillArgs), p]),
    'sq_distill_backward': (C.c_int, [C.POINTER(DistillArgs), p]),
    'sq_distill_loss_grad': (C.c_int, [C.POINTER(DistillArgs), p]),
    'sq_selective_workspace': (i64, [C.c_int] * 6),
    'sq_selective_forward': (C.c_int, [C.POINTER(SelectiveArgs), p]),
    'sq_selective_backward': (C.c_int, [C.POINTER(SelectiveArgs), p]),
    'sq_selective_step': (C.c_int, [C.POINTER(SelectiveStepArgs), p]),
    'sq_conv_scan_workspace': (i64, [C.c_int] * 6),
    'sq_conv_scan_forward': (C.c_int, [C.POINTER(CausalConvArgs), C.POINTER(SelectiveArgs), p]),
    'sq_conv_scan_backward': (C.c_int, [C.POINTER(CausalConvArgs), C.POINTER(SelectiveArgs), p]),
    'sq_conv_scan_step': (C.c_int, [C.POINTER(ConvScanStepArgs), p]),
    'sq_causal_conv_workspace': (i64, [C.c_int] * 3),
    'sq_causal_conv_forward': (C.c_int, [C.POINTER(CausalConvArgs), p]),
    'sq_causal_conv_backward': (C.c_int, [C.POINTER(CausalConvArgs), p]),
    'sq_causal_conv_step': (C.c_int, [p, i64, p, p, p, p] + [C.c_int] * 6 + [p]),
    'sq_pack_activations': (C.c_int, [p, i64, i64, C.c_int, C.c_int, p, p, p]),
    'sq_unpack_activations': (C.c_int, [p, p, i64, C.c_int, C.c_int, p, p]),
}

_lib = None


def load():
    """Load libsq325.so once; raise ImportError if it is absent (no fallback path exists)."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise ImportError(f'{LIB_PATH} is missing: build it with '
                          f'`python mamb2_8b_fp4_recall_sq3.25_b200/build.py` (nvcc, sm_100a)')
    lib = C.CDLL(str(LIB_PATH))
    for name, (res, args) in _PROTOS.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    if lib.sq_abi_version() != ABI_VERSION:
        raise ImportError('libsq325.so ABI version differs from the Python binding')
    _lib = lib
    return lib


def exported_symbols():
    return tuple(_PROTOS)


def call(name, *args):
    """Call an entry point; map a non-zero status to the reference's exception class."""
    lib = load()
    status = getattr(lib, name)(*args)
    if status != SQ_OK:
        msg = lib.sq_last_error().decode(errors='replace')
        raise _EXC.get(status, RuntimeError)(f'{name}: {msg}')
    return status


def stream_ptr(stream=None):
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


def launch(name, device, *args):
    """call() with the current stream of `device` appended, for short kernels: the device is
    switched only where another one is current, and the stream handle is read without building
    a Stream object."""
    import torch
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    return call(name, *args, torch._C._cuda_getCurrentRawStream(index))


def refuse_tangents(what, *tensors):
    """There are no forward-mode derivatives here: a tensor's tangent is refused, where a kernel would drop it."""
    from torch.autograd import forward_ad
    if forward_ad._current_level < 0:                        # outside every dual_level
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f'{what} has no forward-mode derivative')


def ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else C.c_void_p(0)
