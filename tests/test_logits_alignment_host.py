"""The operators on rows of logits refuse arrays that are not aligned to their type: a kernel's access to one would
fault the GPU.  Nothing is read or launched: the pointers are not valid ones."""
import ctypes as C

import pytest


def _logits(_lib):
    return 4096, 10, 2, 10, _lib.F32


@pytest.mark.parametrize('field', ['uniform', 'temperature', 'top_k', 'top_p', 'min_p', 'tokens'])
def test_sample_refuses_misaligned_arrays(field):
    from sq325 import _lib
    lib = _lib.load()
    a = _lib.SampleArgs(*_logits(_lib), 4096, 4096, 4096, 4096, 4096, 1.0, 0, 1.0, 0.0, 4096)
    setattr(a, field, 4100 if field == 'tokens' else 4098)
    assert lib.sq_sample(C.byref(a), None) == _lib.SQ_EINVAL
    assert b'sample: misaligned' in lib.sq_last_error()


@pytest.mark.parametrize('type_name,values,indices', [('F32', 4098, 4096), ('F16', 4097, 4096), ('BF16', 4097, 4096), ('F32', 4096, 4098)])
def test_top_logits_refuses_misaligned_outputs(type_name, values, indices):
    from sq325 import _lib
    lib = _lib.load()
    rows = _lib.Logits(4096, 10, 2, 10, getattr(_lib, type_name))
    assert lib.sq_top_logits(C.byref(rows), 2, values, indices, None) == _lib.SQ_EINVAL
    assert b'top_logits: misaligned' in lib.sq_last_error()


@pytest.mark.parametrize('name,field', [('sq_distill_forward', 'loss'), ('sq_distill_loss_grad', 'loss'),
                                        ('sq_distill_loss_grad', 'weight'), ('sq_distill_backward', 'weight')])
def test_distillation_refuses_misaligned_arrays(name, field):
    from sq325 import _lib
    lib = _lib.load()
    d = _lib.DistillArgs(*_logits(_lib), 4096, 4096, 2, _lib.F32, 1.0, 4096, 1, 4096, 4096, 4096, 10)
    setattr(d, field, 4098)
    assert getattr(lib, name)(C.byref(d), None) == _lib.SQ_EINVAL
    assert b'misaligned' in lib.sq_last_error()
