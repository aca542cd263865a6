"""fp4.linear above 256 rows decodes the weights into a staging buffer: every call has its own, so that calls on
different streams do not overwrite weights another one still reads."""
import contextlib

import pytest
import torch


class _OnDevice(torch.Tensor):
    """A host tensor that passes for a device tensor."""
    is_cuda = True


def test_every_call_stages_in_its_own_buffer(monkeypatch):
    """Without a GPU: nothing is launched, the buffers that two calls hand over are compared.  On the device
    the allocator orders a buffer's reuse by the stream it was allocated on, so it must be allocated in the call."""
    from sq325 import _lib, fp4
    w = fp4.Fp4Tensor(torch.zeros(16, 64, dtype=torch.uint8), torch.zeros(16, 8, dtype=torch.uint8), torch.ones(1), (16, 128))
    x = torch.zeros(300, 128, dtype=torch.float16).as_subclass(_OnDevice)
    allocated, handed = [], []
    empty = torch.empty

    def recorded(*args, **kw):
        allocated.append(empty(*args, **kw))         # kept: two live buffers have two addresses
        return allocated[-1]

    monkeypatch.setattr(torch, 'empty', recorded)
    monkeypatch.setattr(torch.cuda, 'device', lambda device: contextlib.nullcontext())
    monkeypatch.setattr(_lib, 'stream_ptr', lambda: None)
    monkeypatch.setattr(_lib, 'call', lambda name, *args: handed.append((args[10].value, args[11])))
    for _ in range(2):
        assert fp4.linear(w, x).shape == (300, 16)
    (first, size), (second, again) = handed
    assert size == again == _lib.load().sq_fp4_linear_workspace(300, 16, 128)
    assert first != second
    mine = {t.data_ptr(): t.numel() for t in allocated}
    assert mine[first] == mine[second] == size


@pytest.mark.gpu
def test_two_heads_on_two_streams():
    """Two heads, 300 rows each, on two streams at once: the same bits as one after the other."""
    from sq325 import fp4
    g = torch.Generator(device='cuda').manual_seed(5)
    heads = [fp4.synthetic(8192, 4096, g) for _ in range(2)]
    inputs = [torch.randn(300, 4096, generator=g, device='cuda').half() for _ in range(2)]
    want = [fp4.linear(w, x) for w, x in zip(heads, inputs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(fp4.linear(heads[n], inputs[n]))
    torch.cuda.synchronize()
    for n in range(2):
        assert want[n].isfinite().all() and all(torch.equal(want[n], y) for y in got[n])
