"""Infinities and NaN inside a sequence: no result is finite and wrong.

What depends on such a token is not finite; the rest of its chunk of 128 tokens is right or not finite; chunks before it (behind
it, for gradients), the other heads and, behind B or C, the other groups have the bits that they have without it.  Bounds of
what is finite are those of test_gpu_mixer."""
import pytest
import torch

import _mixer64 as ref
from test_gpu_mixer import HALF, least, scan_inputs, sq, u  # noqa: F401

pytestmark = pytest.mark.gpu
INF, NAN = float('inf'), float('nan')
T0 = 170                                          # the token, in the second chunk of three


def right_or_not_finite(got, value, bound, what):
    bound = bound + least(got.dtype)
    got, value, finite = got.double(), value.double(), got.isfinite()
    assert not finite[~value.isfinite()].any(), f'{what}: finite where the definition is not'
    both = finite & value.isfinite()
    off = (got - value).abs()[both]
    assert (off <= 1.5 * bound[both]).all(), f'{what}: finite and wrong'


def inputs(dtype):
    a = scan_inputs(1, 384, 4, 2, 64, dtype, seed=12, param=torch.float32)
    a.pop('lengths'), a.pop('state')
    return a


def forward(sq, a):
    with torch.no_grad():
        return sq.selective_scan(a['x'], a['dt'], a['A'], a['B'], a['C'], a['D'], a['dt_bias'], return_final_state=True)


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('name,place,value', [('x', (0, T0, 1, 5), INF), ('x', (0, T0, 1, 5), -INF), ('x', (0, T0, 1, 5), NAN), ('dt', (0, T0, 1), INF), ('dt', (0, T0, 1), NAN),
                                              ('B', (0, T0, 0, 7), INF), ('B', (0, T0, 0, 7), NAN), ('C', (0, T0, 0, 7), -INF), ('C', (0, T0, 0, 7), NAN)])
def test_scan(sq, dtype, name, place, value):  # noqa: F811
    a = inputs(dtype)
    clean, clean_last = forward(sq, a)
    a[name][place] = value
    y, last = forward(sq, a)
    heads = [1] if name in ('x', 'dt') else [0, 1]         # that the token has a say in
    others = [h for h in range(4) if h not in heads]
    assert torch.equal(y[:, :128], clean[:, :128]) and torch.equal(y[:, :, others], clean[:, :, others])
    assert torch.equal(last[:, others], clean_last[:, others])
    d = [a[k].double() for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias')]
    vy, vl = ref.scan(*d)
    b = inputs(dtype)                                      # magnitudes, of the clean inputs
    sy, sl = ref.scan(*(b[k].double() if k in ('dt', 'A', 'dt_bias') else b[k].double().abs() for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias')))
    right_or_not_finite(y, vy, u(dtype) * vy.abs() + (u(dtype) + 2 ** -11) * sy, 'y')
    right_or_not_finite(last, vl, 2 ** -17 * sl, 'last')


@pytest.mark.parametrize('dtype', HALF)
def test_a_step_of_minus_infinity_passes_its_token_over(sq, dtype):  # noqa: F811
    a = inputs(dtype)
    a['dt'][0, T0:T0 + 20, 1] = -INF
    y, last = forward(sq, a)
    d = [a[k].double() for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias')]
    vy, vl = ref.scan(*d)
    sy, sl = ref.scan(*(t if k in ('dt', 'A', 'dt_bias') else t.abs() for k, t in zip(('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias'), d)))
    assert y.isfinite().all() and last.isfinite().all()
    right_or_not_finite(y, vy, u(dtype) * vy.abs() + (u(dtype) + 2 ** -11) * sy, 'y')
    right_or_not_finite(last, vl, 2 ** -17 * sl, 'last')


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('value', [INF, NAN])
def test_gradients(sq, dtype, value):  # noqa: F811
    """One infinite value of dy: later chunks, other heads and other groups as without it."""
    a = inputs(dtype)
    names = ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias')
    leaves = [a[k].requires_grad_() for k in names]
    dy = torch.randn(1, 384, 4, 64, generator=torch.Generator(device='cuda').manual_seed(3), device='cuda').to(dtype)
    run = lambda: dict(zip(names, torch.autograd.grad(sq.selective_scan(*leaves), leaves, dy)))
    clean = run()
    _, sums = ref.scan_with_grads(*(a[k] for k in names), None, None, dy)
    dy[0, T0, 1, 5] = value
    got = run()
    values, _ = ref.scan_with_grads(*(a[k] for k in names), None, None, dy)
    others = [0, 2, 3]
    for k in ('x', 'dt'):
        assert torch.equal(got[k][:, 256:], clean[k][:, 256:]) and torch.equal(got[k][:, :, others], clean[k][:, :, others]), k
    for k in ('B', 'C'):
        assert torch.equal(got[k][:, 256:], clean[k][:, 256:]) and torch.equal(got[k][:, :, 1], clean[k][:, :, 1]), k
    for k in ('A', 'D', 'dt_bias'):
        assert torch.equal(got[k][others], clean[k][others]), k
    t = u(dtype)
    for k in names:
        wide = {'x': t + 2 ** -11, 'B': 2 ** -10, 'C': 2 ** -10}.get(k, 2 ** -17)
        right_or_not_finite(got[k], values['d' + k], u(got[k].dtype) * values['d' + k].abs() + wide * sums['d' + k], 'd' + k)


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('channel', [70, 256 + 7, 512 + 9], ids=['x', 'B', 'C'])
@pytest.mark.parametrize('value', [INF, NAN])
def test_conv_scan(sq, dtype, channel, value):  # noqa: F811
    """The same behind a convolution, which takes the token to the three behind it."""
    heads, groups, width = 4, 2, 256 + 512
    gen = torch.Generator(device='cuda').manual_seed(4)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    xbc, dt = rnd(1, 384, width).to(dtype), (0.5 * rnd(1, 384, heads) - 3).to(dtype)
    A, w, b, D = -(0.2 + 3 * rnd(heads).abs()), (0.5 * rnd(width, 4)).to(dtype), (0.3 * rnd(width)).to(dtype), rnd(heads).to(dtype)
    run = lambda: sq.conv_scan(xbc, dt, A, w, b, D, heads=heads, groups=groups, return_final_state=True)

    def definition(f, x):
        z, _ = ref.conv(f(x.double()), f(w.double()), f(b.double()))
        xx, B, C = z.split([256, 256, 256], -1)
        return ref.scan(xx.unflatten(2, (heads, 64)), dt.double(), A.double(), B.unflatten(2, (2, 128)), C.unflatten(2, (2, 128)), f(D.double()))
    clean, _, clean_last = run()
    sy, sl = definition(torch.abs, xbc)
    xbc[0, T0, channel] = value
    y, _, last = run()
    hit = [1] if channel < 256 else [0, 1]
    others = [h for h in range(heads) if h not in hit]
    assert torch.equal(y[:, :128], clean[:, :128]) and torch.equal(y[:, :, others], clean[:, :, others]) and torch.equal(last[:, others], clean_last[:, others])
    vy, vl = definition(lambda t: t, xbc)
    # x, B and C once each in fp16 (2^-11 of a value), weights and states once each
    right_or_not_finite(y, vy, u(dtype) * vy.abs() + (3 * 2 ** -11 + 2 ** -10) * sy, 'y')
    right_or_not_finite(last, vl, 3 * 2 ** -11 * sl, 'last')
