"""The mixer's operators in unquantised states against their definitions in 64 bits.

Tolerances.  A rounding to a type is off by at most half a step, u = eps / 2 of the value: 2^-11 (fp16), 2^-8 (bf16),
2^-24 (fp32); below the type's smallest normal number steps stay as they are there (fp16: 2^-24 below 2^-14), so that half of
one is added.  What is made of many terms is bounded by the sum of their magnitudes S (tests/_mixer64.py):
  y, dx       the result's own rounding u |v|, the pairs' weights once in the operands' type (u S), the states once in
              fp16 (2^-11 S)
  dB, dC      own rounding u |v|, operands once in fp16 and the pairs' sum once in fp16 (2 * 2^-11 S)
  ddt         own rounding, and 32-bit sums
  32-bit sums (ddt, dD, ddt_bias, dA, states): products of 128 terms and chunks behind one another, fp32 accumulation
              128 * 2^-24 S = 2^-17 S, operands of 22 bits (2^-22 S, within that)
B and C lose nothing on their way to scaled fp16 but what is 2^-28 of a tile's largest value.  Each bound is taken one
and a half times for products of roundings."""
import math

import pytest
import torch

import _mixer64 as ref

pytestmark = pytest.mark.gpu
HALF = [torch.float16, torch.bfloat16]


def u(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half a step among the type's smallest numbers."""
    return torch.finfo(dtype).smallest_normal * u(dtype)


@pytest.fixture(autouse=True)
def same_inputs():
    torch.manual_seed(0)


@pytest.fixture(scope='module')
def sq():
    import sq325
    return sq325


def near(got, value, bound, what):
    bound = bound + least(got.dtype)
    got, off = got.detach().double(), (got.detach().double() - value).abs()
    bad = ~(off <= bound * 1.5 + 1e-30)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / (bound + 1e-30)).max()):.2f} bounds, first at {bad.nonzero()[0].tolist()}'


def scan_inputs(batch, length, heads, groups, dim, dtype, seed=0, pad=0, carried=False, lengths=None, param=None, junk=False):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    part = lambda *s: rnd(s[0], s[1], math.prod(s[2:]) + pad).to(dtype)[:, :, :math.prod(s[2:])].unflatten(2, s[2:])
    param = param or dtype
    a = dict(x=part(batch, length, heads, dim), dt=(0.5 * rnd(batch, length, heads) - 3).to(dtype), A=-(0.2 + 6 * rnd(heads).abs()),
             B=part(batch, length, groups, 128) * 0.5, C=part(batch, length, groups, 128) * 0.5, D=rnd(heads).to(param),
             dt_bias=(0.3 * rnd(heads)).to(param), state=rnd(batch, heads, dim, 128) if carried else None,
             lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device='cuda'))
    if pad:                                        # keep the strides of a part of a wider buffer
        a['B'], a['C'] = part(batch, length, groups, 128), part(batch, length, groups, 128)
    if junk and lengths is not None:               # behind the sequences' ends
        for k in ('x', 'dt', 'B', 'C'):
            for b, n in enumerate(lengths):
                a[k][b, n:] = float('nan') if b % 2 else float('inf')
    return a


def check_scan(a, got, names, values, sums, dtype):
    t = u(dtype)
    bounds = {'y': t * values['y'].abs() + (t + 2 ** -11) * sums['y'], 'last': 2 ** -17 * sums['last']}
    for k in names:
        v, s = values['d' + k].abs(), sums['d' + k]
        own = u(a[k].dtype) * v
        bounds['d' + k] = own + {'x': (t + 2 ** -11) * s, 'B': 2 ** -10 * s, 'C': 2 ** -10 * s}.get(k, 2 ** -17 * s)
    for k, g in got.items():
        near(g, values[k], bounds[k], k)


CASES = [
    # batch, length, heads, groups, dim, lengths, carried, pad
    (1, 1, 1, 1, 64, None, False, 0), (2, 1, 3, 1, 9, [0, 1], True, 0), (1, 2, 2, 2, 1, None, True, 0),
    (1, 127, 2, 1, 64, None, False, 0), (1, 128, 4, 2, 64, None, True, 8), (2, 129, 2, 1, 65, None, True, 0),
    (3, 300, 6, 3, 40, [300, 0, 131], True, 0), (2, 260, 4, 1, 128, [256, 257], False, 3), (1, 513, 16, 1, 64, None, False, 64),
    (2, 140, 5, 5, 72, [12, 140], False, 1),
]


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('case', CASES, ids=str)
def test_scan_and_gradients(sq, case, dtype):
    batch, length, heads, groups, dim, lengths, carried, pad = case
    a = scan_inputs(batch, length, heads, groups, dim, dtype, seed=length, pad=pad, carried=carried, lengths=lengths, junk=True)
    gen = torch.Generator(device='cuda').manual_seed(7)
    dy = torch.randn(batch, length, heads, dim, generator=gen, device='cuda').to(dtype)
    dlast = torch.randn(batch, heads, dim, 128, generator=gen, device='cuda')
    names = [k for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias', 'state') if a[k] is not None]
    for k in names:
        a[k].requires_grad_()
    y, last = sq.selective_scan(a['x'], a['dt'], a['A'], a['B'], a['C'], a['D'], a['dt_bias'], a['state'], a['lengths'], True)
    grads = torch.autograd.grad([y, last], [a[k] for k in names], [dy, dlast])
    values, sums = ref.scan_with_grads(a['x'], a['dt'], a['A'], a['B'], a['C'], a['D'], a['dt_bias'], a['state'], a['lengths'], dy, dlast)
    check_scan(a, dict(y=y, last=last, **{'d' + k: g for k, g in zip(names, grads)}), names, values, sums, dtype)
    if lengths is not None:
        for b, n in enumerate(lengths):
            assert not y[b, n:].any() and not any(grads[names.index(k)][b, n:].any() for k in ('x', 'dt', 'B', 'C'))
    # without gradients the same kernels give the same bits, and so does a second call
    with torch.no_grad():
        again, last2 = sq.selective_scan(a['x'], a['dt'], a['A'], a['B'], a['C'], a['D'], a['dt_bias'], a['state'], a['lengths'], True)
    assert torch.equal(again, y) and torch.equal(last2, last)


@pytest.mark.parametrize('dtype', HALF)
def test_scan_without_optional_terms_and_with_32_bit_parameters(sq, dtype):
    a = scan_inputs(2, 150, 4, 2, 64, dtype, seed=3, param=torch.float32)
    dy = torch.randn(2, 150, 4, 64, device='cuda').to(dtype)
    for D, bias in ((None, None), (a['D'], None), (None, a['dt_bias']), (a['D'], a['dt_bias'])):
        a2 = dict(a, D=D, dt_bias=bias)
        names = [k for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias') if a2[k] is not None]
        leaves = [a2[k].detach().requires_grad_() for k in names]
        full = dict(zip(names, leaves))
        y = sq.selective_scan(*(full.get(k) for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias')))
        grads = torch.autograd.grad(y, leaves, dy)
        values, sums = ref.scan_with_grads(a2['x'], a2['dt'], a2['A'], a2['B'], a2['C'], D, bias, None, None, dy)
        check_scan(a2, dict(y=y, **{'d' + k: g for k, g in zip(names, grads)}), names, values, sums, dtype)


@pytest.mark.parametrize('scale_b,scale_x,scale_dy', [(1e-6, 1.0, 1.0), (300.0, 1e-4, 1e-5), (1.0, 2000.0, 1e-3), (0.0, 1.0, 1.0)])
@pytest.mark.parametrize('dtype', HALF)
def test_scan_over_a_wide_range_of_values(sq, dtype, scale_b, scale_x, scale_dy):
    """Scaled fp16 operands hold small and large tensors alike."""
    a = scan_inputs(1, 200, 2, 1, 64, torch.float32, seed=9)
    a = {k: (v * {'B': scale_b, 'C': 1.0, 'x': scale_x}.get(k, 1.0)).to(dtype) if v is not None and k != 'A' else v for k, v in a.items() if k != 'lengths'}
    a['lengths'] = None
    dy = (torch.randn(1, 200, 2, 64, device='cuda') * scale_dy).to(dtype)
    names = ['x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias']
    leaves = [a[k].requires_grad_() for k in names]
    y = sq.selective_scan(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    values, sums = ref.scan_with_grads(*(a[k] for k in names), None, None, dy)
    got = dict(y=y, **{'d' + k: g for k, g in zip(names, grads)})
    t = u(dtype)
    for k in list(got):
        s = sums[k]
        wide = {'y': t + 2 ** -11, 'dx': t + 2 ** -11, 'dB': 2 ** -10, 'dC': 2 ** -10}.get(k, 2 ** -17)
        near(got[k], values[k], u(got[k].dtype) * values[k].abs() + wide * s, k)


def test_decays_of_any_speed(sq):
    """Steps that forget everything, steps that forget nothing, and both in one chunk; A of zero."""
    a = scan_inputs(1, 260, 3, 1, 64, torch.float16, seed=4)
    a['A'] = torch.tensor([0.0, -16.0, -1e-3], device='cuda')
    a['dt'][0, 60:64] = 40.0
    a['dt'][0, 100:140] = -15.0
    dy = torch.randn(1, 260, 3, 64, device='cuda').half()
    names = ['x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias']
    leaves = [a[k].requires_grad_() for k in names]
    y = sq.selective_scan(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    values, sums = ref.scan_with_grads(*(a[k] for k in names), None, None, dy)
    check_scan(a, dict(y=y, **{'d' + k: g for k, g in zip(names, grads)}), names, values, sums, torch.float16)


def test_gradients_against_differences(sq):
    """A step along a direction changes the loss by the gradient's product with it: both by the kernels' forward, in
    states, whose sums are 32-bit."""
    a = scan_inputs(1, 200, 2, 1, 64, torch.float16, seed=11, param=torch.float32, carried=True)
    gen = torch.Generator(device='cuda').manual_seed(5)
    dlast = torch.randn(1, 2, 64, 128, generator=gen, device='cuda')
    for k in ('A', 'dt_bias', 'state'):
        leaf = a[k].clone().requires_grad_()
        run = lambda v: sq.selective_scan(*(v if n == k else a[n] for n in ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias', 'state')),
                                          return_final_state=True)[1]
        g, = torch.autograd.grad(run(leaf), leaf, dlast)
        way = torch.randn(leaf.shape, generator=gen, device='cuda')
        h = 1e-2
        with torch.no_grad():
            loss = [(run(leaf + s * h * way).double() * dlast.double()).sum() for s in (1, -1)]
        # second differences' error h^2 of smooth functions of size about one in h; forward sums 2^-17 of a loss's terms, over h
        terms = float((run(leaf.detach()).double() * dlast.double()).abs().sum())
        want, got = float(loss[0] - loss[1]) / (2 * h), float((g.double() * way.double()).sum())
        size = float((g.double() * way.double()).abs().sum())
        assert abs(want - got) <= 2 ** -17 * terms / h + 10 * h * h * size, (k, want, got)


@pytest.mark.parametrize('weights', ['same', 'float32'])
@pytest.mark.parametrize('dtype', [*HALF, torch.float32])
@pytest.mark.parametrize('case', [(1, 1, 4, 4, None, False, 0, 'silu'), (2, 37, 129, 3, [0, 37], True, 0, 'silu'),
                                  (3, 70, 1280, 4, [70, 2, 33], True, 4, 'silu'), (1, 300, 64, 2, None, True, 3, None),
                                  (2, 130, 516, 4, [1, 129], False, 0, 'silu'), (1, 2, 7, 4, None, True, 1, 'silu')], ids=str)
def test_causal_conv_and_gradients(sq, case, dtype, weights):
    batch, length, channels, taps, lengths, carried, pad, activation = case
    gen = torch.Generator(device='cuda').manual_seed(length)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    wt = dtype if weights == 'same' else torch.float32
    x = rnd(batch, length, channels + pad).to(dtype)[:, :, :channels]
    w, b = (rnd(channels, taps) * 0.5).to(wt), rnd(channels).to(wt)
    state = rnd(batch, taps - 1, channels).to(dtype) if carried else None
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device='cuda')
    dy, dlast = rnd(batch, length, channels).to(dtype), rnd(batch, taps - 1, channels).to(dtype)
    clean = x.clone()
    if lengths is not None:
        for i, e in enumerate(lengths):
            x[i, e:], clean[i, e:] = float('nan'), 0
    names = ['x', 'w', 'b'] + (['state'] if carried else [])
    leaves = [t.requires_grad_() for t in (x, w, b, state) if t is not None]
    y, last = sq.causal_conv(x, w, b, state, n, activation, True)
    grads = torch.autograd.grad([y, last], leaves, [dy, dlast])

    def run(f):
        d = {k: f(t.detach().double()).requires_grad_() for k, t in (('x', clean), ('w', w), ('b', b), ('state', state)) if t is not None}
        yy, ll = ref.conv(d['x'], d['w'], d['b'], d.get('state'), n, activation == 'silu')
        up = f(dy.double()) if n is None else torch.where(ref.present(n, batch, length, 'cuda')[..., None], f(dy.double()), torch.zeros_like(dy, dtype=torch.double))
        return yy.detach(), ll.detach(), torch.autograd.grad((yy * up).sum() + (ll * f(dlast.double())).sum(), list(d.values()))
    vy, vl, vg = run(lambda t: t)
    sy, sl, sg = run(torch.abs)
    # z is a sum of five products, its activation and slope a few fp32 steps more (16-bit types: __expf and a reciprocal);
    # sums over tokens fp32.  |slope| < 1.2 and |slope'| < 0.6 bound what an error of z does.
    f32 = 2 ** -19
    near(y, vy, u(dtype) * vy.abs() + f32 * (sy + 1), 'y')
    assert torch.equal(last.double(), vl)
    tokens = batch * length
    for k, leaf, g, v, s in zip(names, leaves, grads, vg, sg):
        near(g, v, u(leaf.dtype) * v.abs() + f32 * (s + (s.max() if k in ('w', 'b') else 4) + 4 * (tokens ** 0.5 if k in ('w', 'b') else 1)), 'd' + k)
    with torch.no_grad():
        assert torch.equal(sq.causal_conv(x, w, b, state, n, activation), y)


@pytest.mark.parametrize('dtype', [*HALF, torch.float32])
@pytest.mark.parametrize('shape,pad', [((1,), 0), ((3, 128), 0), ((7, 11, 1001), 0), ((5, 256), 3), ((2, 3, 4, 130), 0), ((4, 2560), 64), ((0, 16), 0)], ids=str)
def test_pack_and_unpack(sq, shape, pad, dtype):
    gen = torch.Generator(device='cuda').manual_seed(len(shape))
    x = torch.randn((*shape[:-1], shape[-1] + pad), generator=gen, device='cuda')
    x = (x * torch.exp(3 * torch.randn((*shape[:-1], 1), generator=gen, device='cuda'))).to(dtype)[..., :shape[-1]]
    if x.numel() > 200:
        x.view(-1) if pad == 0 else None
        x[..., :min(128, shape[-1])][..., 0] = 0
        x[0, ..., :128] = 0                                   # a block of zeros
    packed = sq.pack_activations(x)
    codes, scales, values = ref.pack(x)
    assert packed.dtype == dtype and torch.equal(packed.codes, codes) and torch.equal(packed.scales, scales)
    assert torch.equal(sq.unpack_activations(packed), values.to(dtype))
    assert torch.equal(sq.unpack_activations(packed, torch.float32), values)


def test_pack_of_extreme_blocks(sq):
    x = torch.zeros(9, 128, device='cuda')
    x[1, 5], x[1, 6] = 1e-42, 3e-43                            # among the smallest numbers
    x[2, 0], x[2, 1] = 3e38, -3e38
    x[3, 7] = float('inf')
    x[4, 7] = float('nan')
    x[5] = -1.0
    x[6, 3] = 1e-25
    x[7, :3] = torch.tensor([127.0, 0.5, 1.5])                 # halves go to the even code
    got = sq.unpack_activations(sq.pack_activations(x))
    _, _, want = ref.pack(x)
    fine = [0, 1, 2, 5, 6, 7, 8]
    assert torch.equal(got[fine], want[fine])
    assert got[3].isnan().all() and got[4].isnan().all()
    assert sq.pack_activations(x).codes[7, :3].tolist() == ref.pack(x)[0][7, :3].tolist()


@pytest.mark.parametrize('dtype', [*HALF, torch.float32])
@pytest.mark.parametrize('channels,taps', [(1280, 4), (131, 3)])
def test_conv_kept_in_8_bits(sq, channels, taps, dtype):
    """The output is the given input's, the gradients are those at the kept values."""
    gen = torch.Generator(device='cuda').manual_seed(2)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    x, w, b, dy = rnd(2, 90, channels).to(dtype), rnd(channels, taps).to(dtype), rnd(channels).to(dtype), rnd(2, 90, channels).to(dtype)
    n = torch.tensor([90, 41], dtype=torch.int32, device='cuda')
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = sq.causal_conv(*leaves, lengths=n, keep='int8')
    grads = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(y, sq.causal_conv(x, w, b, lengths=n).detach())
    held = torch.where(ref.present(n, 2, 90, 'cuda')[..., None], ref.pack(x.detach())[2], torch.zeros((), device='cuda')).double().requires_grad_()
    wd, bd = w.detach().double().requires_grad_(), b.detach().double().requires_grad_()
    want = torch.autograd.grad(ref.conv(held, wd, bd, None, n)[0], [held, wd, bd], torch.where(ref.present(n, 2, 90, 'cuda')[..., None], dy.double(), torch.zeros((), device='cuda', dtype=torch.double)))
    for g, v, leaf in zip(grads, want, leaves):
        near(g, v, u(leaf.dtype) * v.abs() + 2 ** -19 * (v.abs().max() + 8 * 90 ** 0.5), 'gradient')


@pytest.mark.parametrize('keep', [None, 'int8'])
@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('case', [(2, 200, 4, 2, 64, None, True, 4), (3, 131, 3, 1, 9, [131, 0, 64], False, 3), (1, 1, 2, 1, 40, None, True, 4)], ids=str)
def test_conv_scan_and_gradients(sq, case, dtype, keep):
    batch, length, heads, groups, dim, lengths, carried, taps = case
    width = heads * dim + 256 * groups
    gen = torch.Generator(device='cuda').manual_seed(length)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    a = dict(xbc=rnd(batch, length, width).to(dtype), dt=(0.5 * rnd(batch, length, heads) - 3).to(dtype), A=-(0.2 + 6 * rnd(heads).abs()),
             w=(0.5 * rnd(width, taps)).to(dtype), b=(0.3 * rnd(width)).to(dtype), D=rnd(heads).to(dtype), bias=(0.3 * rnd(heads)).to(dtype),
             conv_state=rnd(batch, taps - 1, width).to(dtype) if carried else None, state=rnd(batch, heads, dim, 128) if carried else None)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device='cuda')
    names = [k for k, v in a.items() if v is not None]
    for k in names:
        a[k].requires_grad_()
    dy, dlast = rnd(batch, length, heads, dim).to(dtype), rnd(batch, heads, dim, 128)
    dconv = rnd(batch, taps - 1, width).to(dtype)
    y, conv_last, last = sq.conv_scan(a['xbc'], a['dt'], a['A'], a['w'], a['b'], a['D'], a['bias'], heads=heads, groups=groups,
                                      conv_state=a['conv_state'], initial_state=a['state'], lengths=n, return_final_state=True, keep=keep)
    grads = torch.autograd.grad([y, conv_last, last], [a[k] for k in names], [dy, dconv, dlast])

    def run(f, xbc):
        d = {k: (f(a[k].detach().double()) if k not in ('dt', 'A', 'bias') else a[k].detach().double()).requires_grad_() for k in names}
        if xbc is not None:
            d['xbc'] = f(xbc.double()).requires_grad_()
        z, cl = ref.conv(d['xbc'], d['w'], d['b'], d.get('conv_state'), n)
        x, B, C = z.split([heads * dim, groups * 128, groups * 128], -1)
        yy, ll = ref.scan(x.unflatten(2, (heads, dim)), d['dt'], d['A'], B.unflatten(2, (groups, 128)), C.unflatten(2, (groups, 128)), d['D'], d['bias'],
                          d.get('state'), n)
        up = f(dy.double())
        if n is not None:
            up = torch.where(ref.present(n, batch, length, 'cuda')[..., None, None], up, torch.zeros_like(up))
        loss = (yy * up).sum() + (cl * f(dconv.double())).sum() + (ll * f(dlast.double())).sum()
        return yy.detach(), cl.detach(), ll.detach(), torch.autograd.grad(loss, [d[k] for k in names])
    plain = lambda t: t
    vy, vc, vl, _ = run(plain, None)
    sy, _, sl, _ = run(torch.abs, None)
    kept = ref.pack(a['xbc'].detach())[2] if keep else None
    _, _, _, vg = run(plain, kept)
    _, _, _, sg = run(torch.abs, kept)
    # the convolution's output three times in 11 bits of its tile's largest value (x, B, C; 8 stands for the largest over a usual
    # one), the pairs' weights, states and operands once each in fp16: 6 roundings; its gradient once in the type
    z11 = 3 * 8 * 2 ** -11
    near(y, vy, u(dtype) * vy.abs() + (z11 + 2 ** -10) * sy, 'y')
    near(last, vl, z11 * sl, 'last')
    assert torch.equal(conv_last.double(), vc)
    for k, g, v, s in zip(names, grads, vg, sg):
        s = s.abs().amax() if k in ('dt', 'A', 'bias', 'w', 'b', 'D') else s.abs() + 0.05 * s.abs().amax()
        near(g, v, u(a[k].dtype) * v.abs() + (z11 + 2 ** -10 + 2 * u(dtype)) * s, 'd' + k)


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('batch,heads,groups,dim', [(1, 1, 1, 1), (3, 4, 2, 40), (2, 8, 1, 64), (5, 3, 3, 100)])
def test_steps_follow_a_prompt(sq, dtype, batch, heads, groups, dim):
    """A prompt by conv_scan, then tokens by conv_scan_step, against the whole sequence's definition; the two-call form
    gives the same states within the convolution's rounding."""
    width, prompt, tokens = heads * dim + 256 * groups, 140, 5
    gen = torch.Generator(device='cuda').manual_seed(dim)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    xbc, dt = rnd(batch, prompt + tokens, width).to(dtype), (0.5 * rnd(batch, prompt + tokens, heads) - 3).to(dtype)
    A, w, b, D, bias = -(0.2 + 3 * rnd(heads).abs()), (0.5 * rnd(width, 4)).to(dtype), (0.3 * rnd(width)).to(dtype), rnd(heads).to(dtype), rnd(heads).to(dtype)
    _, conv_state, state = sq.conv_scan(xbc[:, :prompt], dt[:, :prompt], A, w, b, D, bias, heads=heads, groups=groups, return_final_state=True)

    def definition(f):
        z, _ = ref.conv(f(xbc.double()), f(w.double()), f(b.double()))
        x, B, C = z.split([heads * dim, groups * 128, groups * 128], -1)
        return ref.scan(x.unflatten(2, (heads, dim)), dt.double(), A.double(), B.unflatten(2, (groups, 128)), C.unflatten(2, (groups, 128)), f(D.double()), bias.double())
    (y, last), (sy, sl) = definition(lambda t: t), definition(torch.abs)
    z11 = 3 * 8 * 2 ** -11
    conv2, state2 = conv_state.clone(), state.clone()
    for t in range(prompt, prompt + tokens):
        got = sq.conv_scan_step(xbc[:, t], dt[:, t], A, w, b, D, bias, heads=heads, groups=groups, conv_state=conv_state, state=state)
        near(got, y[:, t], u(dtype) * y[:, t].abs() + z11 * sy[:, t], 'y of a step')
        z = sq.causal_conv_step(xbc[:, t], conv2, w, b)
        x, B, C = z.split([heads * dim, groups * 128, groups * 128], -1)
        two = sq.selective_step(x.unflatten(1, (heads, dim)), dt[:, t], A, B.unflatten(1, (groups, 128)), C.unflatten(1, (groups, 128)), state2, D, bias)
        near(two, y[:, t], u(dtype) * y[:, t].abs() + (z11 + 3 * u(dtype)) * sy[:, t], 'y of two calls')
    near(state, last, z11 * sl, 'state')
    near(state2, last, (z11 + 2 * u(dtype)) * sl, 'state of two calls')
    assert torch.equal(conv_state, xbc[:, -3:]) and torch.equal(conv2, conv_state)


def test_a_state_is_carried_over_calls(sq):
    """Parts of a sequence behind one another end where the whole does; rows of their own lengths."""
    a = scan_inputs(2, 300, 4, 2, 64, torch.float16, seed=6)
    whole, last = sq.selective_scan(a['x'], a['dt'], a['A'], a['B'], a['C'], a['D'], a['dt_bias'], return_final_state=True)
    state, at = None, 0
    for n in (1, 128, 71, 100):
        cut = [a[k][:, at:at + n] for k in ('x', 'dt')], [a[k][:, at:at + n] for k in ('B', 'C')]
        y, state = sq.selective_scan(cut[0][0], cut[0][1], a['A'], cut[1][0], cut[1][1], a['D'], a['dt_bias'], state, return_final_state=True)
        values, sums = ref.scan_with_grads(a['x'], a['dt'], a['A'], a['B'], a['C'], a['D'], a['dt_bias'], None, None, torch.zeros_like(a['x']))
        part = slice(at, at + n)
        near(y, values['y'][:, part], 2 ** -11 * values['y'][:, part].abs() + 2 ** -10 * sums['y'][:, part], 'y')
        at += n
    near(state, last.double(), 2 * 2 ** -17 * sums['last'], 'state')


def test_graphs_of_steps_and_of_training(sq):
    """Captured and replayed on other inputs, twice, beside eager calls of the same leaves."""
    heads, groups, dim, width = 4, 2, 64, 4 * 64 + 512
    gen = torch.Generator(device='cuda').manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    w, b, A, D, bias = (0.5 * rnd(width, 4)).half(), rnd(width).half(), -rnd(heads).abs(), rnd(heads).half(), rnd(heads).half()
    xbc, dt, dy = rnd(2, 150, width).half(), (rnd(2, 150, heads) - 3).half(), rnd(2, 150, heads, dim).half()
    conv_state, state = torch.zeros(2, 3, width, device='cuda').half(), torch.zeros(2, heads, dim, 128, device='cuda')
    token, tdt = xbc[:, 0].clone(), dt[:, 0].clone()

    def train(leaves):
        y = sq.conv_scan(leaves[0], leaves[1], A, leaves[2], leaves[3], D, bias, heads=heads, groups=groups, keep='int8')
        return y, *torch.autograd.grad(y, leaves, dy)

    def step():
        return sq.conv_scan_step(token, tdt, A, w, b, D, bias, heads=heads, groups=groups, conv_state=conv_state, state=state)
    static = [t.clone().requires_grad_() for t in (xbc, dt, w, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train([t.detach().clone().requires_grad_() for t in static])
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, steps = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = train(static)
    conv_state.zero_(), state.zero_()
    with torch.cuda.graph(steps):
        y_step = step()
    for seed in (3, 4):
        fresh = torch.randn(xbc.shape, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda').half()
        with torch.no_grad():
            static[0].copy_(fresh)
        graph.replay()
        eager = train([t.detach().clone().requires_grad_() for t in static])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(captured, eager))
    conv_state.zero_(), state.zero_()
    ys = []
    for t in range(4):
        token.copy_(xbc[:, t]), tdt.copy_(dt[:, t])
        steps.replay()
        ys.append(y_step.clone())
    states = conv_state.clone(), state.clone()
    conv_state.zero_(), state.zero_()
    for t in range(4):
        token.copy_(xbc[:, t]), tdt.copy_(dt[:, t])
        assert torch.equal(step(), ys[t])
    assert torch.equal(states[0], conv_state) and torch.equal(states[1], state)
    sq._lib.call('sq_device_check', sq._lib.stream_ptr())


def test_two_streams_at_once(sq):
    """Calls on two streams share nothing."""
    a, b = (scan_inputs(2, 700, 8, 2, 64, torch.bfloat16, seed=s) for s in (21, 22))
    run = lambda i: sq.selective_scan(*(i[k] for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias')), return_final_state=True)
    want = run(a), run(b)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(6):
        for s, i in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(run(i))
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(g, want[k % 2]))


def test_gradients_are_whole_in_any_call(sq):
    """Broadcast inputs, a retained graph, an unused output, saved tensors moved by hooks."""
    a = scan_inputs(3, 140, 4, 1, 64, torch.float16, seed=8)
    state = torch.randn(1, 4, 64, 128, device='cuda', requires_grad=True)
    x = a['x'][:1].clone().requires_grad_()
    args = lambda xx, ss: (xx, a['dt'], a['A'], a['B'], a['C'], a['D'], a['dt_bias'], ss)
    dy = torch.randn(3, 140, 4, 64, device='cuda').half()
    y = sq.selective_scan(*args(x.expand(3, -1, -1, -1), state.expand(3, -1, -1, -1)))
    first = torch.autograd.grad(y, (x, state), dy, retain_graph=True)
    second = torch.autograd.grad(y, (x, state), dy)
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    parts = [torch.autograd.grad(sq.selective_scan(*(t[i:i + 1] if t.ndim > 1 else t for t in args(x.expand(3, -1, -1, -1), state.expand(3, -1, -1, -1)))),
                                 (x, state), dy[i:i + 1]) for i in range(3)]
    near(first[1], sum(p[1].double() for p in parts), 2 ** -16 * sum(p[1].double().abs() for p in parts), 'shared state')
    near(first[0], sum(p[0].double() for p in parts), 4 * 2 ** -11 * sum(p[0].double().abs() for p in parts), 'shared x')
    y2, last = sq.selective_scan(*args(x.expand(3, -1, -1, -1), state.expand(3, -1, -1, -1)), return_final_state=True)
    only_last, = torch.autograd.grad(last.sum(), (state,))
    assert torch.isfinite(only_last).all() and only_last.any()
    with torch.autograd.graph.save_on_cpu():
        y3 = sq.selective_scan(*args(x.expand(3, -1, -1, -1), state.expand(3, -1, -1, -1)))
    assert all(torch.equal(p, q) for p, q in zip(first, torch.autograd.grad(y3, (x, state), dy)))


def test_offsets_past_32_bits(sq):
    """A token stride that puts the last tokens more than 2^31 elements behind the first."""
    stride, length = (1 << 31) // 200, 260
    buf = torch.empty(stride * length + 4096, dtype=torch.float16, device='cuda')
    width = 2 * 64 + 256
    xbc = buf.as_strided((1, length, width), (stride * length, stride, 1))
    xbc.copy_(torch.randn(1, length, width, device='cuda'))
    w, b = torch.randn(width, 4, device='cuda').half(), torch.randn(width, device='cuda').half()
    assert torch.equal(sq.causal_conv(xbc, w, b), sq.causal_conv(xbc.contiguous(), w, b))
    x, B, C = (t.unflatten(2, s) for t, s in zip(xbc.split([128, 128, 128], -1), ((2, 64), (1, 128), (1, 128))))
    dt, A = torch.randn(1, length, 2, device='cuda').half() - 3, -torch.rand(2, device='cuda')
    got = sq.selective_scan(x, dt, A, B, C, return_final_state=True)
    want = sq.selective_scan(x.contiguous(), dt, A, B.contiguous(), C.contiguous(), return_final_state=True)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_refusals(sq):
    a = scan_inputs(2, 5, 4, 2, 64, torch.float16)
    good = [a[k] for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias')]

    def refused(match, i, value, **more):
        with pytest.raises(ValueError, match=match):
            sq.selective_scan(*(value if k == i else v for k, v in enumerate(good)), **more)
    refused('x must be', 0, a['x'].float())
    refused('x must be', 0, a['x'].cpu())
    refused('dt must be', 1, a['dt'].bfloat16())
    refused('dt must be', 1, a['dt'][:, :4])
    refused('A must be', 2, a['A'].half())
    refused('groups', 3, a['B'].expand(2, 5, 2, 128).repeat(1, 1, 2, 1)[:, :, :3])
    refused('C must be', 4, a['C'][..., :64])
    refused('D must be', 5, a['D'][:3])
    refused('initial_state', 7, None, initial_state=torch.zeros(2, 4, 64, 128, device='cuda').half())
    refused('lengths', 7, None, lengths=torch.zeros(2, device='cuda'))
    with pytest.raises(ValueError, match='contiguous'):
        sq.selective_step(a['x'][:, 0], a['dt'][:, 0], a['A'], a['B'][:, 0], a['C'][:, 0], torch.zeros(2, 4, 128, 64, device='cuda').transpose(2, 3))
    x = torch.zeros(1, 3, 8, device='cuda')
    w = torch.zeros(8, 4, device='cuda')
    for bad in (dict(weight=w[:, :1]), dict(weight=torch.zeros(8, 5, device='cuda')), dict(weight=w.half()), dict(bias=w[:, 0].half()),
                dict(activation='gelu'), dict(keep='int4'), dict(initial_state=torch.zeros(1, 2, 8, device='cuda')), dict(x=x[0]), dict(x=x[:, :0])):
        with pytest.raises(ValueError):
            sq.causal_conv(**dict(dict(x=x, weight=w), **bad))
    xbc = torch.zeros(1, 3, 2 * 64 + 256, device='cuda').half()
    dt, A, w2 = torch.zeros(1, 3, 2, device='cuda').half(), torch.zeros(2, device='cuda'), torch.zeros(384, 4, device='cuda').half()
    for bad in (dict(heads=3), dict(groups=2), dict(heads=0), dict(heads=True), dict(xbc=xbc.float()), dict(keep=8)):
        with pytest.raises(ValueError):
            sq.conv_scan(**dict(dict(xbc=xbc, dt=dt, A=A, conv_weight=w2, heads=2, groups=1), **bad))
    with pytest.raises(ValueError, match='state must be given'):
        sq.conv_scan_step(xbc[:, 0], dt[:, 0], A, w2, heads=2, groups=1, conv_state=torch.zeros(1, 3, 384, device='cuda').half(), state=None)
    with pytest.raises(ValueError):
        sq.pack_activations(torch.zeros(3, device='cuda', dtype=torch.int32))
    with pytest.raises(ValueError):
        sq.unpack_activations((torch.zeros(2, 130, dtype=torch.int8, device='cuda'), torch.zeros(2, 1, device='cuda'), torch.float16))
