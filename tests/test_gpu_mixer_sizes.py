"""The mixer's operators at sizes where a CTA has several units, long strips and second turns of its loops, and at strides
whose offsets pass 32 bits.  Bounds are those of test_gpu_mixer."""
import ctypes as C

import pytest
import torch

import _mixer64 as ref
from test_gpu_mixer import HALF, check_scan, near, scan_inputs, sq, u  # noqa: F401

pytestmark = pytest.mark.gpu
NAMES = ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias', 'state')


def units_of_a_cta(sq, batch, length, heads, groups, dim):  # noqa: F811
    """(forward, backward): the rule by which CTAs share a group's units (64 rows of a head); the backward's is checked
    against the sums by CTA that its workspace has room for."""
    nc, tiles_of_a_head = -(-length // 128), -(-dim // 64)
    units, bc = heads * tiles_of_a_head, batch * nc
    mine = units // groups

    def best(places, once):
        costs = []
        for s in range(1, mine + 1):
            per = -(-mine // s)
            if -(-mine // per) == s:
                costs.append((-(-bc * groups * s // places) * (per + once * (1.5 if s > 1 else 1.0)), s))
        least = min(c for c, _ in costs)
        return next(s for c, s in costs if c <= least * 1.001)
    fwd, bwd = best(296, 0.5), best(148, 1.0)
    room = sq._lib.load().sq_selective_workspace
    up = lambda n: -(-n // 256) * 256
    more = up(bc * units * 32768) + 2 * up(bc * units * 8) + up(batch * units * nc * 128 * 8) + up(bc * heads * 16)
    sums = room(batch, length, heads, dim, groups, 1) - room(batch, length, heads, dim, groups, 0) - more
    assert sums == (2 * up(bc * 128 * groups * 128 * 4 * bwd) if bwd > 1 else 0)
    return -(-mine // fwd), -(-mine // bwd)


def grads_of(call, leaves, up):
    outs = call()
    return outs, torch.autograd.grad(outs, leaves, up)


# batch, length, heads, groups, dim, lengths
MANY = [(16, 260, 64, 8, 64, None), (16, 260, 40, 8, 72, [260, 0, 1, 128, 129, 200, 257, 260, 3, 256, 255, 260, 130, 90, 260, 17]),
        (37, 90, 24, 8, 40, None), (25, 300, 40, 8, 64, None)]


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('case', MANY, ids=lambda c: str(c[:5]))
def test_several_units_a_cta(sq, case, dtype):  # noqa: F811
    """One group against the definition, all of it against calls of one sequence and one group, whose CTAs have one unit."""
    batch, length, heads, groups, dim, lengths = case
    per = units_of_a_cta(sq, batch, length, heads, groups, dim)
    assert min(per) > 1 and units_of_a_cta(sq, 1, length, heads // groups, 1, dim) == (1, 1)
    a = scan_inputs(batch, length, heads, groups, dim, dtype, seed=length, carried=True, lengths=lengths, junk=True)
    gen = torch.Generator(device='cuda').manual_seed(7)
    dy = torch.randn(batch, length, heads, dim, generator=gen, device='cuda').to(dtype)
    dlast = torch.randn(batch, heads, dim, 128, generator=gen, device='cuda')

    def call(t, up):
        leaves = [t[k].detach().requires_grad_() for k in NAMES]
        (y, last), grads = grads_of(lambda: sq.selective_scan(*leaves, t['lengths'], True), leaves, up)
        return dict(y=y, last=last, **{'d' + k: g for k, g in zip(NAMES, grads)})
    got = call(a, [dy, dlast])

    def cut(t, k, b, g):
        """The part of tensor k that sequences b and group g have."""
        n = heads // groups
        h = slice(g * n, (g + 1) * n)
        return t[b] if k == 'lengths' else t[h] if k in ('A', 'D', 'dt_bias') else t[b, h] if k in ('state', 'last') else t[b, :, g:g + 1] if k in ('B', 'C') else t[b, :, h]
    part = lambda b, g: {k: None if v is None else cut(v, k, b, g) for k, v in a.items()}
    # the definition, of the last group
    whole, g = slice(None), groups - 1
    p = part(whole, g)
    values, sums = ref.scan_with_grads(*(p[k] for k in NAMES), p['lengths'], cut(dy, 'x', whole, g), cut(dlast, 'state', whole, g))
    mine = {k: cut(v, k.removeprefix('d') if k not in ('dt_bias', 'dt') else k, whole, g) for k, v in got.items()}
    check_scan(p, mine, NAMES, values, sums, dtype)
    # one sequence and one group: the same bits, but for dB and dC, whose sums have a scale and an order by CTA
    for b, g in ((0, 0), (1, groups - 1), (batch - 1, groups // 2), (batch // 2, 1)):
        b = slice(b, b + 1)
        one = call(part(b, g), [cut(dy, 'x', b, g), cut(dlast, 'state', b, g)])
        for k in ('y', 'last', 'dx', 'ddt', 'dstate'):
            assert torch.equal(one[k], cut(got[k], 'x' if k == 'y' else k.removeprefix('d') if k != 'ddt' else 'dt', b, g)), (k, b, g)
    # a second time, on two streams at once
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    again = []
    for s in streams * 2:
        with torch.cuda.stream(s):
            again.append(call(a, [dy, dlast]))
    torch.cuda.synchronize()
    for other in again:
        assert all(torch.equal(other[k], got[k]) for k in got)


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('case,keep', [(MANY[1], None), (MANY[3], None), (MANY[0], 'int8')], ids=str)
def test_several_units_a_cta_behind_a_convolution(sq, case, keep, dtype):  # noqa: F811
    """The same bits as calls of one sequence and one group, but for what comes through dB and dC; a second time too."""
    batch, length, heads, groups, dim, lengths = case
    width, n = heads * dim + 256 * groups, heads // groups
    assert keep is None or n * dim % 128 == 0         # a group's channels are whole blocks that share a scale
    gen = torch.Generator(device='cuda').manual_seed(3)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    xbc, dt, dy = rnd(batch, length, width).to(dtype), (0.5 * rnd(batch, length, heads) - 3).to(dtype), rnd(batch, length, heads, dim).to(dtype)
    A, w, bias, D = -(0.2 + 6 * rnd(heads).abs()), (0.5 * rnd(width, 4)).to(dtype), (0.3 * rnd(width)).to(dtype), rnd(heads).to(dtype)
    count = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device='cuda')

    def call(xbc, dt, A, w, bias, D, count, dy, groups):
        leaves = [t.detach().requires_grad_() for t in (xbc, dt, A, w, bias, D)]
        y = sq.conv_scan(*leaves[:5], leaves[5], heads=leaves[1].shape[2], groups=groups, lengths=count, keep=keep)
        return y, *torch.autograd.grad(y, leaves, dy)
    got = call(xbc, dt, A, w, bias, D, count, dy, groups)
    for b, g in ((0, 0), (1, groups - 1), (batch // 2, 1)):
        h, b = slice(g * n, (g + 1) * n), slice(b, b + 1)
        at = [slice(h.start * dim, h.stop * dim), *(slice(heads * dim + k * groups * 128 + g * 128, heads * dim + k * groups * 128 + (g + 1) * 128) for k in (0, 1))]
        cols = torch.cat([torch.arange(s.start, s.stop, device='cuda') for s in at])
        one = call(xbc[b][..., cols], dt[b, :, h], A[h], w[cols], bias[cols], D[h], None if count is None else count[b], dy[b, :, h], 1)
        assert torch.equal(one[0], got[0][b, :, h]) and torch.equal(one[2], got[2][b, :, h])
        mine = got[1][b][..., cols]
        assert torch.equal(one[1][..., :n * dim], mine[..., :n * dim])
        # dB and dC through the convolution: operands, sums and result once each in the type or fp16, of the largest
        size = mine[..., n * dim:].double().abs().amax()
        assert (one[1][..., n * dim:].double() - mine[..., n * dim:].double()).abs().max() <= 6 * u(dtype) * size
    again = call(xbc, dt, A, w, bias, D, count, dy, groups)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize('dtype', [*HALF, torch.float32])
@pytest.mark.parametrize('channels,taps,activation', [(10240, 4, 'silu'), (10239, 3, None)])
def test_long_strips(sq, channels, taps, activation, dtype):  # noqa: F811
    """4 x 2,048 tokens at the model's width: strips of 64 and 128 tokens; some channels against the definition."""
    gen = torch.Generator(device='cuda').manual_seed(5)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    x, dy = rnd(4, 2048, channels).to(dtype), rnd(4, 2048, channels).to(dtype)
    w, b, state, dlast = (0.5 * rnd(channels, taps)).to(dtype), rnd(channels).to(dtype), rnd(4, taps - 1, channels).to(dtype), rnd(4, taps - 1, channels).to(dtype)
    n = torch.tensor([2048, 2, 1337, 128], dtype=torch.int32, device='cuda')
    for keep in (None, 'int8'):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, state)]
        y, last = sq.causal_conv(*leaves, n, activation, True, keep=keep)
        grads = torch.autograd.grad([y, last], leaves, [dy, dlast])
        for at in (slice(0, 12), slice(508, 520), slice(5117, 5131), slice(channels - 9, channels)):
            block = slice(at.start // 128 * 128, min(channels, -(-at.stop // 128) * 128))
            held = ref.pack(x[..., block])[2][..., at.start - block.start:at.stop - block.start] if keep else x[..., at]

            def run(f):
                d = [f(t.double()).requires_grad_() for t in (held, w[at], b[at], state[..., at])]
                vy, vl = ref.conv(*d, n, activation == 'silu')
                up = torch.where(ref.present(n, 4, 2048, 'cuda')[..., None], f(dy[..., at].double()), 0.0)
                return vy.detach(), vl.detach(), torch.autograd.grad([vy, vl], d, [up, f(dlast[..., at].double())])
            (vy, vl, want), (sy, _, sums) = run(lambda t: t), run(torch.abs)
            # bounds as those of test_causal_conv_and_gradients: a few fp32 steps of the sums of magnitudes
            if keep is None:
                near(y[..., at], vy, u(dtype) * vy.abs() + 2 ** -19 * (sy + 1), 'y')
                assert torch.equal(last[..., at].double(), vl)
            for k, g, v, m in zip(('dx', 'dw', 'db', 'dstate'), (grads[0][..., at], grads[1][at], grads[2][at], grads[3][..., at]), want, sums):
                many = k in ('dw', 'db')
                near(g, v, u(dtype) * v.abs() + 2 ** -19 * (m + (m.max() if many else 4) + 4 * (8192 ** 0.5 if many else 1)), k)


@pytest.mark.parametrize('dtype', [*HALF, torch.float32])
@pytest.mark.parametrize('rows,width', [(20000, 100), (3000, 10240), (9600, 1001)])
def test_packing_of_many_rows(sq, rows, width, dtype):  # noqa: F811
    x = (torch.randn(rows, width, device='cuda', generator=torch.Generator(device='cuda').manual_seed(rows)) * 3).to(dtype)
    packed = sq.pack_activations(x)
    codes, scales, values = ref.pack(x)
    assert torch.equal(packed.codes, codes) and torch.equal(packed.scales, scales)
    assert torch.equal(sq.unpack_activations(packed), values.to(dtype)) and torch.equal(sq.unpack_activations(packed, torch.float32), values)


@pytest.mark.parametrize('dtype', [*HALF, torch.float32])
@pytest.mark.parametrize('weights', ['same', 'float32'])
@pytest.mark.parametrize('taps,activation,batch,channels', [(2, None, 1, 1), (3, 'silu', 3, 131), (4, None, 2, 520), (2, 'silu', 5, 1280), (3, None, 2, 64)])
def test_conv_step_in_every_form(sq, dtype, weights, taps, activation, batch, channels):  # noqa: F811
    gen = torch.Generator(device='cuda').manual_seed(channels)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    wt = dtype if weights == 'same' else torch.float32
    w, b, state = rnd(channels, taps).to(wt), rnd(channels).to(wt), rnd(batch, taps - 1, channels).to(dtype)
    tokens = rnd(batch, 6, channels + 3).to(dtype)[..., :channels]
    vy, vl = ref.conv(tokens.double(), w.double(), b.double(), state.double(), None, activation == 'silu')
    sy, _ = ref.conv(tokens.double().abs(), w.double().abs(), b.double().abs(), state.double().abs(), None, activation == 'silu')
    for t in range(6):
        y = sq.causal_conv_step(tokens[:, t], state, w, b, activation)
        near(y, vy[:, t], u(dtype) * vy[:, t].abs() + 2 ** -19 * (sy[:, t] + 1), 'y')
    assert torch.equal(state.double(), vl)
    # without a bias
    state0 = rnd(batch, taps - 1, channels).to(dtype)
    vy, _ = ref.conv(tokens[:, :1].double(), w.double(), None, state0.double(), None, activation == 'silu')
    near(sq.causal_conv_step(tokens[:, 0], state0, w, None, activation), vy[:, 0], u(dtype) * vy[:, 0].abs() + 2 ** -19 * (vy.abs().amax() + 8), 'y without bias')


@pytest.mark.parametrize('stride', [10737416, 10737418], ids=['aligned', 'odd'])
def test_offsets_past_32_bits_with_gradients(sq, stride):  # noqa: F811
    """Inputs, gradients coming in and gradients going out with a token stride that puts the last ones behind 2^31 elements."""
    length, width = 260, 384
    buf = torch.empty(stride * length + 4096, dtype=torch.float16, device='cuda')
    far = lambda at, w: buf.as_strided((1, length, w), (stride * length, stride, 1), at)
    xbc, dyc = far(0, width), far(512, width)
    gen = torch.Generator(device='cuda').manual_seed(2)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    xbc.copy_(rnd(1, length, width)), dyc.copy_(rnd(1, length, width))
    w, b = rnd(width, 4).half(), rnd(width).half()

    def conv(x, dy):
        leaves = [x.detach().requires_grad_(), w.detach().requires_grad_(), b.detach().requires_grad_()]
        y = sq.causal_conv(*leaves)
        return y, *torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(conv(xbc, dyc), conv(xbc.contiguous(), dyc.contiguous())))
    parts = lambda t: [p.unflatten(2, s) for p, s in zip(t.split([128, 128, 128], -1), ((2, 64), (1, 128), (1, 128)))]
    dt, A = (rnd(1, length, 2) - 3).half(), -torch.rand(2, device='cuda')
    x, B, C_ = parts(xbc)
    dy = parts(dyc)[0]
    outs = [torch.empty(1, length, *s, dtype=torch.float16, device='cuda') for s in ((2, 64), (1, 128), (1, 128))]
    from sq325 import selective
    args = lambda *t: (t[0], dt, A, t[1], t[2], None, None, None, None)
    want = selective.scan_backward(*args(x.contiguous(), B.contiguous(), C_.contiguous()), dy.contiguous(), None, *outs, (True, False, False, False))
    there = parts(far(1024, width))
    got = selective.scan_backward(*args(x, B, C_), dy, None, *there, (True, False, False, False))
    assert all(torch.equal(p, q) for p, q in zip(outs, there)) and torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    # y as well
    y = parts(far(1536, width))[0]
    a = selective.scan_args(*args(x, B, C_))
    a.y, a.y_batch_stride, a.y_token_stride = y.data_ptr(), y.stride(0), y.stride(1)
    work = selective._workspace(a, 0, x.device)
    sq._lib.launch('sq_selective_forward', x.device, C.byref(a))
    del work
    assert torch.equal(y, sq.selective_scan(x.contiguous(), dt, A, B.contiguous(), C_.contiguous()))


def test_nothing_is_read_that_the_call_did_not_write(sq):  # noqa: F811
    """The same bits whatever the memory that outputs and workspaces come from held before."""
    a = scan_inputs(3, 300, 6, 3, 72, torch.bfloat16, seed=5, carried=True, lengths=[300, 0, 131])
    width = 6 * 72 + 768
    xbc, w = torch.randn(3, 300, width, device='cuda').bfloat16(), torch.randn(width, 4, device='cuda').bfloat16()
    dy = torch.randn(3, 300, 6, 72, device='cuda').bfloat16()

    def call():
        leaves = [a[k].detach().requires_grad_() for k in NAMES]
        y, last = sq.selective_scan(*leaves, a['lengths'], True)
        grads = torch.autograd.grad(y, leaves, dy)
        more = [t.detach().requires_grad_() for t in (xbc, a['dt'], a['A'], w)]
        z = sq.conv_scan(*more, heads=6, groups=3, lengths=a['lengths'], keep='int8')
        return [t.clone() for t in (y, last, *grads, z, *torch.autograd.grad(z, more, dy))]
    want = call()
    for fill in (0x7f, 0xff, 0x00):               # NaN in some types, and zeros
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        held = [torch.empty(n << 20, dtype=torch.uint8, device='cuda').fill_(fill) for n in (1, 1, 1, 1, 2, 4, 8, 20, 20, 40, 100, 200)]
        small = [torch.empty(n, dtype=torch.uint8, device='cuda').fill_(fill) for n in (512, 4096, 65536, 262144) for _ in range(12)]
        torch.cuda.synchronize()
        del held, small
        assert all(torch.equal(p, q) for p, q in zip(want, call())), fill
