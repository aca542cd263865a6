"""conv_scan's limit of groups: its tiles of x, B and C are one grid's second dimension.  Nothing is launched."""
import ctypes as C

import pytest


@pytest.mark.parametrize('heads,groups,dim', [(26300, 26300, 1), (30000, 30000, 64), (29000, 29000, 8)])
@pytest.mark.parametrize('name', ['sq_conv_scan_forward', 'sq_conv_scan_backward'])
def test_a_grid_has_room_for_every_tile(name, heads, groups, dim):
    from sq325 import _lib
    lib = _lib.load()
    width = heads * dim + 256 * groups
    conv = _lib.CausalConvArgs(1, 10, width, 4, 1, _lib.F16, _lib.F16, 4096, 10 * width, width, None, None, 4096, 4096)
    conv.dx = 4096
    scan = _lib.SelectiveArgs(1, 10, heads, dim, groups, _lib.F16)
    scan.dt = scan.A = scan.y = scan.dy = scan.ddt = 4096
    scan.workspace, scan.workspace_bytes = 4096, lib.sq_conv_scan_workspace(1, 10, heads, dim, groups, int(name.endswith('backward')))
    assert getattr(lib, name)(C.byref(conv), C.byref(scan), None) == _lib.SQ_EINVAL
    assert b'too large' in lib.sq_last_error()
