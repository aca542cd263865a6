"""Refusals of the mixer's operators that need no GPU: nothing is read or launched, the pointers are not valid ones."""
import ctypes as C

import pytest
import torch


def _lib():
    from sq325 import _lib
    return _lib


def _scan(lib, backward=False):
    a = lib.SelectiveArgs(1, 10, 4, 64, 2, lib.F16, 4096, 2560, 256, 4096, 40, 4, 4096, 4096, 2560, 256, 4096, 2560, 256)
    a.y, a.y_batch_stride, a.y_token_stride = 4096, 2560, 256
    a.dy = a.dx = a.ddt = a.dB = a.dC = 4096
    a.workspace, a.workspace_bytes = 4096, lib.load().sq_selective_workspace(1, 10, 4, 64, 2, int(backward))
    return a


SCAN_BAD = [('type', 2), ('type', 7), ('batch', 0), ('length', 0), ('length', 1 << 25), ('heads', 3), ('groups', 0), ('dim', 0), ('dim', 2048),
            ('batch', 70000), ('x', 0), ('x', 4097), ('dt', 0), ('A', 4098), ('B', 0), ('C', 4097), ('state_in', 4098), ('lengths', 4098),
            ('workspace', 0), ('workspace', 4100), ('workspace_bytes', 16)]


@pytest.mark.parametrize('field,value', SCAN_BAD)
@pytest.mark.parametrize('name', ['sq_selective_forward', 'sq_selective_backward'])
def test_scan_refuses(name, field, value):
    lib = _lib()
    a = _scan(lib, name.endswith('backward'))
    setattr(a, field, value)
    assert getattr(lib.load(), name)(C.byref(a), None) == lib.SQ_EINVAL
    assert name[3:].encode() in lib.load().sq_last_error()


@pytest.mark.parametrize('field,value', [('D', 4097), ('dt_bias', 4097)])
def test_scan_refuses_misaligned_parameters(field, value):
    lib = _lib()
    a = _scan(lib)
    setattr(a, field, value)
    assert lib.load().sq_selective_forward(C.byref(a), None) == lib.SQ_EINVAL
    a = _scan(lib)
    a.D, a.d_type = 4096, 9
    assert lib.load().sq_selective_forward(C.byref(a), None) == lib.SQ_EINVAL


def test_scan_workspace():
    f = _lib().load().sq_selective_workspace
    assert f(0, 10, 4, 64, 2, 0) == -1 and f(1, 10, 3, 64, 2, 0) == -1
    assert 0 < f(1, 10, 4, 64, 2, 0) < f(1, 10, 4, 64, 2, 1) < f(2, 300, 4, 64, 2, 1)
    g = _lib().load().sq_conv_scan_workspace
    assert g(1, 10, 4, 64, 0, 0) == -1 and g(1, 10, 4, 64, 2, 1) > f(1, 10, 4, 64, 2, 1)


def _conv(lib):
    a = lib.CausalConvArgs(1, 10, 512, 4, 1, lib.F16, lib.F16, 4096, 5120, 512, None, None, 4096, 4096)
    a.y, a.y_batch_stride, a.y_token_stride = 4096, 5120, 512
    a.dy = a.dx = 4096
    a.workspace, a.workspace_bytes = 4096, lib.load().sq_causal_conv_workspace(1, 10, 512)
    return a


@pytest.mark.parametrize('field,value', [('type', 3), ('weight_type', 1), ('taps', 1), ('taps', 5), ('channels', 0), ('batch', 70000), ('length', 0),
                                         ('weight', 0), ('weight', 4097), ('bias', 4097), ('x', 0), ('x', 4097), ('codes', 4096), ('state_in', 4097),
                                         ('lengths', 4098)])
@pytest.mark.parametrize('name', ['sq_causal_conv_forward', 'sq_causal_conv_backward'])
def test_conv_refuses(name, field, value):
    lib = _lib()
    a = _conv(lib)
    setattr(a, field, value)
    assert getattr(lib.load(), name)(C.byref(a), None) == lib.SQ_EINVAL
    assert name[3:].encode() in lib.load().sq_last_error()


@pytest.mark.parametrize('name,field,value', [('sq_causal_conv_forward', 'y', 0), ('sq_causal_conv_forward', 'y', 4097), ('sq_causal_conv_backward', 'dx', 0),
                                              ('sq_causal_conv_backward', 'dweight', 4097), ('sq_causal_conv_backward', 'workspace_bytes', 8),
                                              ('sq_causal_conv_backward', 'workspace', 4100)])
def test_conv_refuses_outputs(name, field, value):
    lib = _lib()
    a = _conv(lib)
    setattr(a, field, value)
    assert getattr(lib.load(), name)(C.byref(a), None) == lib.SQ_EINVAL


def test_conv_state_is_not_its_own_successor():
    lib = _lib()
    a = _conv(lib)
    a.state_in = a.state_out = 8192
    assert lib.load().sq_causal_conv_forward(C.byref(a), None) == lib.SQ_EINVAL


@pytest.mark.parametrize('change', [dict(channels=511), dict(length=9), dict(batch=2), dict(silu=0), dict(type=1, weight_type=1), dict(lengths=8192)])
def test_conv_scan_refuses_a_convolution_of_another_geometry(change):
    lib = _lib()
    conv, scan = _conv(lib), lib.SelectiveArgs(1, 10, 4, 64, 1, lib.F16)
    scan.dt, scan.A, scan.y, scan.workspace, scan.workspace_bytes = 4096, 4096, 4096, 4096, 1 << 30
    for k, v in change.items():
        setattr(conv, k, v)
    assert lib.load().sq_conv_scan_forward(C.byref(conv), C.byref(scan), None) == lib.SQ_EINVAL
    assert lib.load().sq_conv_scan_backward(C.byref(conv), C.byref(scan), None) == lib.SQ_EINVAL


def test_steps_refuse():
    lib = _lib()
    good = dict(batch=2, heads=4, dim=64, groups=2, type=0, x=4096, dt=4096, A=4096, B=4096, C=4096, state=4096, y=4096)
    for bad in (dict(type=2), dict(batch=0), dict(heads=3), dict(x=0), dict(dt=4097), dict(state=4100), dict(state=0), dict(y=4097), dict(B=0), dict(D=4097)):
        a = lib.SelectiveStepArgs(**{**good, **bad})
        assert lib.load().sq_selective_step(C.byref(a), None) == lib.SQ_EINVAL, bad
    good = dict(batch=2, heads=4, dim=64, groups=2, taps=4, type=0, weight_type=0, xbc=4096, dt=4096, A=4096, weight=4096, conv_state=4096, state=4096, y=4096,
                workspace=4096, workspace_bytes=1 << 20)
    for bad in (dict(taps=5), dict(weight=0), dict(conv_state=4097), dict(workspace=0), dict(workspace_bytes=64), dict(xbc=0), dict(weight_type=1)):
        a = lib.ConvScanStepArgs(**{**good, **bad})
        assert lib.load().sq_conv_scan_step(C.byref(a), None) == lib.SQ_EINVAL, bad
    f = lib.load().sq_causal_conv_step
    assert f(4096, 8, None, 4096, None, 4096, 1, 8, 4, 1, 0, 0, None) == lib.SQ_EINVAL
    assert f(4096, 8, 4096, 4096, None, 4096, 1, 8, 1, 1, 0, 0, None) == lib.SQ_EINVAL
    assert f(4096, 8, 4097, 4096, None, 4096, 1, 8, 4, 1, 0, 0, None) == lib.SQ_EINVAL


def test_pack_refuses():
    lib = _lib()
    pack, unpack = lib.load().sq_pack_activations, lib.load().sq_unpack_activations
    for args in ((4096, 8, 2, 8, 3, 4096, 4096), (4096, 8, -1, 8, 0, 4096, 4096), (4096, 8, 2, 0, 0, 4096, 4096), (4097, 8, 2, 8, 0, 4096, 4096),
                 (None, 8, 2, 8, 0, 4096, 4096), (4096, 8, 2, 8, 0, None, 4096), (4096, 8, 2, 8, 0, 4096, 4098)):
        assert pack(*args, None) == lib.SQ_EINVAL, args
    assert unpack(4096, 4096, 2, 8, 2, 4098, None) == lib.SQ_EINVAL
    assert pack(None, 8, 0, 8, 0, None, None, None) == lib.SQ_OK


def test_tensors_on_the_host_are_refused():
    import sq325
    x = torch.zeros(1, 2, 8)
    for call in (lambda: sq325.causal_conv(x, torch.zeros(8, 4)), lambda: sq325.causal_conv_step(x[0], x[:, :1], torch.zeros(8, 4)),
                 lambda: sq325.pack_activations(x), lambda: sq325.selective_scan(x.half()[..., None], x[..., :2], x, x, x),
                 lambda: sq325.selective_step(x.half(), x[0], x, x, x, x), lambda: sq325.conv_scan(x.half(), x, x, x, heads=1, groups=1),
                 lambda: sq325.conv_scan_step(x.half()[0], x, x, x, heads=1, groups=1, conv_state=x, state=x)):
        with pytest.raises(ValueError, match='CUDA'):
            call()


def test_a_grid_has_room_for_every_tile():
    lib = _lib()
    for name in ('sq_selective_forward', 'sq_selective_backward'):
        a = _scan(lib, name.endswith('backward'))
        a.heads = a.groups = 30001                       # a grid's second dimension would hold two tiles a group and more
        assert getattr(lib.load(), name)(C.byref(a), None) == lib.SQ_EINVAL
        assert b'heads is too large' in lib.load().sq_last_error()


def test_a_convolution_keeps_what_it_is_given():
    lib = _lib()
    a = _conv(lib)
    a.x, a.codes, a.scales = 0, 4096, 4096
    assert lib.load().sq_causal_conv_forward(C.byref(a), None) == lib.SQ_EINVAL
    assert b'null x' in lib.load().sq_last_error()
