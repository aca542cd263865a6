"""A process whose first call comes while a stream is captured."""
import subprocess
import sys

import pytest

from conftest import PKG_ROOT

pytestmark = pytest.mark.gpu

FIRST = """
import ctypes, sys
sys.path.insert(0, {path!r})
import torch, sq325
from sq325 import _lib
gen = torch.Generator(device='cuda').manual_seed(0)
rnd = lambda *s: torch.randn(s, generator=gen, device='cuda').half()
x, dt, A, B, C = rnd(1, 200, 2, 64), rnd(1, 200, 2) - 3, -torch.ones(2, device='cuda'), rnd(1, 200, 1, 128), rnd(1, 200, 1, 128)
y = torch.zeros_like(x)
lib = _lib.load()
a = sq325.selective.scan_args(x, dt, A, B, C, None, None, None, None)
a.y, a.y_batch_stride, a.y_token_stride = y.data_ptr(), y.stride(0), y.stride(1)
work = torch.empty(lib.sq_selective_workspace(1, 200, 2, 64, 1, 0), dtype=torch.uint8, device='cuda')
a.workspace, a.workspace_bytes = work.data_ptr(), work.numel()
torch.cuda.synchronize()
rt = ctypes.CDLL('libcudart.so.12')
stream, graph, ready = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
ok = lambda e: e and sys.exit('CUDA error %d' % e)
ok(rt.cudaStreamCreateWithFlags(ctypes.byref(stream), {flags}))
ok(rt.cudaStreamBeginCapture(stream, {mode}))
status = lib.sq_selective_forward(ctypes.byref(a), stream)
end = rt.cudaStreamEndCapture(stream, ctypes.byref(graph))
if status or end:
    sys.exit('status %d (%s), end of capture %d' % (status, lib.sq_last_error().decode(), end))
ok(rt.cudaGraphInstantiate(ctypes.byref(ready), graph, ctypes.c_ulonglong(0)))
assert not y.any()
ok(rt.cudaGraphLaunch(ready, stream))
ok(rt.cudaStreamSynchronize(stream))
ok(rt.cudaGraphExecDestroy(ready))
ok(rt.cudaGraphDestroy(graph))
assert torch.equal(y, sq325.selective_scan(x, dt, A, B, C)) and y.any()
_lib.call('sq_device_check', _lib.stream_ptr())
print('captured')
"""


@pytest.mark.parametrize('flags', [0, 1], ids=['blocking', 'non-blocking'])
@pytest.mark.parametrize('mode', [0, 1, 2], ids=['global', 'thread', 'relaxed'])
def test_a_process_may_begin_with_a_capture(flags, mode):
    """The first call sets up the device's error word, which a capture on any kind of stream is no part of."""
    r = subprocess.run([sys.executable, '-c', FIRST.format(path=str(PKG_ROOT), flags=flags, mode=mode)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and 'captured' in r.stdout, r.stdout + r.stderr
