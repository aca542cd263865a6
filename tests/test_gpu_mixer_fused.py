"""conv_scan's values and gradients by norm, group of channels by group of channels, and its forms that only the C interface has.

Tolerance.  A result is made of terms that were rounded, each on its own: x, B and C behind the convolution to fp16, the pairs'
weights and the states, the operands of dB and dC, the gradient of the convolution's output, and the result itself: at most eight
roundings of at most half a step u, whose root mean square is u / sqrt(3).  Independent terms with errors of that size make a
sum whose error is at most sqrt(8 / 3) u < 1.7 u of the sum's root mean square.  Twice that and a little for sums that cancel: 4 u of the norm, where
u is 2^-11 (fp16) or 2^-8 (bf16).  The norms are taken over at least 16 numbers, so that cancelling in one of them does not count."""
import ctypes as C

import pytest
import torch

import _mixer64 as ref
from test_gpu_mixer import HALF, sq, u  # noqa: F401

pytestmark = pytest.mark.gpu


def inputs(batch, length, heads, groups, dim, taps, dtype, param=None, carried=False, seed=0):
    width, param = heads * dim + 256 * groups, param or dtype
    gen = torch.Generator(device='cuda').manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    a = dict(xbc=rnd(batch, length, width).to(dtype), dt=(0.5 * rnd(batch, length, heads) - 3).to(dtype), A=-(0.2 + 6 * rnd(heads).abs()),
             w=(0.5 * rnd(width, taps)).to(param), b=(0.3 * rnd(width)).to(param), D=rnd(heads).to(param), bias=(0.3 * rnd(heads)).to(param),
             conv_state=rnd(batch, taps - 1, width).to(dtype) if carried else None, state=rnd(batch, heads, dim, 128) if carried else None)
    dy, dlast, dconv = rnd(batch, length, heads, dim).to(dtype), rnd(batch, heads, dim, 128), rnd(batch, taps - 1, width).to(dtype)
    return a, dy, dlast, dconv


def definition(a, heads, groups, dim, n, dy, dlast, dconv, names, xbc=None):
    d = {k: a[k].detach().double().requires_grad_() for k in names}
    if xbc is not None:
        d['xbc'] = xbc.double().requires_grad_()
    z, cl = ref.conv(d['xbc'], d['w'], d['b'], d.get('conv_state'), n)
    x, B, C_ = z.split([heads * dim, groups * 128, groups * 128], -1)
    y, last = ref.scan(x.unflatten(2, (heads, dim)), d['dt'], d['A'], B.unflatten(2, (groups, 128)), C_.unflatten(2, (groups, 128)), d['D'], d['bias'], d.get('state'), n)
    up = dy.double()
    if n is not None:
        up = torch.where(ref.present(n, *dy.shape[:2], 'cuda')[..., None, None], up, torch.zeros_like(up))
    loss = (y * up).sum() + (0 if dlast is None else (last * dlast.double()).sum()) + (0 if dconv is None else (cl * dconv.double()).sum())
    return y.detach(), last.detach(), dict(zip(names, torch.autograd.grad(loss, [d[k] for k in names])))


def close(got, want, c, what):
    got, want = got.detach().double(), want.double()
    assert want.numel() >= 16 and want.norm() > 0
    off = float((got - want).norm() / want.norm())
    assert off <= c, f'{what}: off by {off:.2e} of its norm, {off / c:.2f} bounds'


def check(got, want, heads, groups, dim, c):
    """By x's, B's and C's channels where there are such."""
    at = dict(x=slice(0, heads * dim), B=slice(heads * dim, heads * dim + 128 * groups), C=slice(heads * dim + 128 * groups, None))
    for k, g in got.items():
        for part, s in at.items() if k in ('xbc', 'w', 'b', 'conv_state') else (('', None),):
            cut = lambda t: t if s is None else t[s] if k in ('w', 'b') else t[..., s]
            close(cut(g), cut(want[k]), c, f'd{k} {part}')


CASES = [(2, 200, 16, 2, 64, None, True, 4), (3, 131, 17, 1, 9, [131, 0, 64], False, 3), (2, 260, 16, 4, 72, [257, 260], True, 2), (1, 600, 16, 1, 64, None, False, 4)]


@pytest.mark.parametrize('keep', [None, 'int8'])
@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('case', CASES, ids=str)
def test_values_and_gradients(sq, case, dtype, keep):  # noqa: F811
    batch, length, heads, groups, dim, lengths, carried, taps = case
    a, dy, dlast, dconv = inputs(batch, length, heads, groups, dim, taps, dtype, carried=carried, seed=length)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device='cuda')
    names = [k for k, v in a.items() if v is not None]
    leaves = {k: a[k].detach().requires_grad_() for k in names}
    y, conv_last, last = sq.conv_scan(leaves['xbc'], leaves['dt'], leaves['A'], leaves['w'], leaves['b'], leaves['D'], leaves['bias'], heads=heads, groups=groups,
                                      conv_state=leaves.get('conv_state'), initial_state=leaves.get('state'), lengths=n, return_final_state=True, keep=keep)
    grads = dict(zip(names, torch.autograd.grad([y, conv_last, last], list(leaves.values()), [dy, dconv, dlast])))
    vy, vl, want = definition(a, heads, groups, dim, n, dy, dlast, dconv, names)
    if keep:
        _, _, want = definition(a, heads, groups, dim, n, dy, dlast, dconv, names, ref.pack(a['xbc'])[2])
    c = 4 * u(dtype)
    close(y, vy, c, 'y')
    close(last, vl, 4 * 2 ** -11, 'last')              # x and B in fp16, sums in fp32
    check(grads, want, heads, groups, dim, c)


@pytest.mark.parametrize('dtype,size', [(torch.float16, 2.0 ** -6), (torch.float16, 16.0), (torch.bfloat16, 1e-12), (torch.bfloat16, 1e12)])
def test_gradients_of_other_sizes(sq, dtype, size):  # noqa: F811
    """Within what the gradient of the convolution's output, in the input's type, has room for; weights in 32 bits."""
    heads, groups, dim = 16, 1, 64
    a, dy, _, _ = inputs(2, 200, heads, groups, dim, 4, dtype, param=torch.float32, seed=6)
    dy = (dy.float() * size).to(dtype)
    names = [k for k, v in a.items() if v is not None]
    leaves = {k: a[k].detach().requires_grad_() for k in names}
    y = sq.conv_scan(leaves['xbc'], leaves['dt'], leaves['A'], leaves['w'], leaves['b'], leaves['D'], leaves['bias'], heads=heads, groups=groups)
    grads = dict(zip(names, torch.autograd.grad(y, list(leaves.values()), dy)))
    _, _, want = definition(a, heads, groups, dim, None, dy, None, None, names)
    check(grads, want, heads, groups, dim, 4 * u(dtype))


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('lengths,carried', [([140, 2, 0, 1], True), ([3, 140, 0, 1], False), (None, True)], ids=str)
def test_a_prompt_from_its_codes(sq, dtype, lengths, carried):  # noqa: F811
    """The C interface takes an input in 8 bits: the outputs and the last inputs of the values that the codes stand for."""
    from sq325 import mixer
    from sq325.activations import PackedActivations
    batch, length, heads, groups, dim, taps = 4, 140, 4, 1, 40, 4
    a, _, _, _ = inputs(batch, length, heads, groups, dim, taps, dtype, carried=carried, seed=9)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device='cuda')
    packed = sq.pack_activations(a['xbc'])
    width = a['xbc'].shape[2]
    conv, scan, work = mixer._args(a['xbc'].shape, dtype, None, PackedActivations(*packed), a['dt'], a['A'], a['w'], a['b'], a['D'], a['bias'], a['conv_state'],
                                   a['state'], n, heads, groups, 0)
    y = torch.empty(batch, length, heads, dim, dtype=dtype, device='cuda')
    conv_last, last = torch.empty(batch, taps - 1, width, dtype=dtype, device='cuda'), torch.empty(batch, heads, dim, 128, device='cuda')
    conv.state_out, scan.state_out = conv_last.data_ptr(), last.data_ptr()
    scan.y, scan.y_batch_stride, scan.y_token_stride = y.data_ptr(), length * heads * dim, heads * dim
    sq._lib.launch('sq_conv_scan_forward', y.device, C.byref(conv), C.byref(scan))
    del work
    held = ref.pack(a['xbc'])[2]
    z, cl = ref.conv(held.double(), a['w'].double(), a['b'].double(), None if a['conv_state'] is None else a['conv_state'].double(), n)
    x, B, C_ = z.split([heads * dim, 128, 128], -1)
    vy, vl = ref.scan(x.unflatten(2, (heads, dim)), a['dt'].double(), a['A'].double(), B.unflatten(2, (1, 128)), C_.unflatten(2, (1, 128)), a['D'].double(),
                      a['bias'].double(), None if a['state'] is None else a['state'].double(), n)
    close(y, vy, 4 * u(dtype), 'y')
    close(last, vl, 4 * 2 ** -11, 'last')
    assert torch.equal(conv_last, cl.to(torch.float32).to(dtype))
