"""Cases of the operators that a Mamba-2 mixer learns and answers with in unquantised states: the short
causal convolution (`sq325.causal_conv`), the selective scan over prompts and its gradients
(`sq325.selective_scan`), both for one token (`sq325.conv_scan_step`),
activations kept in 8 bits (`sq325.pack_activations`, `sq325.unpack_activations`), and convolution and
scan in one step of training that keeps its input in 8 bits (`sq325.conv_scan`).

`own = False` computes the plain form in elementary torch operations, `own = True` makes the
library's calls.  A case is a dict of plain values:

  op       'conv' | 'conv_train' | 'pack' | 'token' | 'scan' | 'train' | 'mix'
  batch, length, dtype ('float16' | 'bfloat16' | 'float32')
  channels                  (conv, conv_train, pack)
  heads, groups, dim        (the others; the state has 128 columns a row)
  taps     of the convolution
  pad      columns of the input's buffer beyond the used ones (a token stride that is not the width)
  ragged   sequences of lengths of their own, from zero to `length`
  carried  a state from earlier tokens is carried in
  keep     the input is kept for the backward pass in 8 bits
"""
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parent.parent
N = 128                          # columns of a state's row
BLOCK = 128                      # values that share a scale in 8 bits
CHUNK = 128                      # tokens of a chunk in the plain scan


def _package():
    path = str(ROOT / 'mamb2_8b_fp4_recall_sq3.25_b200')
    if path not in sys.path:
        sys.path.insert(0, path)
    import sq325
    return sq325


def _channels(name, op, batch, length, channels, dtype, taps=4, pad=0, ragged=False, carried=False, keep=False):
    return dict(name=name, op=op, batch=batch, length=length, channels=channels, dtype=dtype, taps=taps, pad=pad,
                ragged=ragged, carried=carried, keep=keep)


def _heads(name, op, batch, length, heads, groups, dim, dtype, taps=4, pad=0, ragged=False, carried=False, keep=False):
    return dict(name=name, op=op, batch=batch, length=length, heads=heads, groups=groups, dim=dim, dtype=dtype,
                taps=taps, pad=pad, ragged=ragged, carried=carried, keep=keep)


def listed():
    return [
        # the convolution of one prompt at the model's width, its last inputs carried on
        _channels('conv_1x1024', 'conv', 1, 1024, 10240, 'float16'),
        # a step of training of the convolution: rows of lengths of their own, parts of a wider buffer
        _channels('conv_train_4x2048', 'conv_train', 4, 2048, 10240, 'bfloat16', pad=128, ragged=True),
        # activations of a small odd layer, and of a window of 8,192 tokens at the model's width
        _channels('pack_77x1001_odd', 'pack', 7, 11, 1001, 'float32'),
        _channels('pack_8192x10240', 'pack', 4, 2048, 10240, 'bfloat16'),
        # one token of one request through convolution and state, and one of a served batch of 64
        _heads('token_1', 'token', 1, 1, 128, 8, 64, 'float16', carried=True),
        _heads('token_64', 'token', 64, 1, 128, 8, 64, 'bfloat16', carried=True),
        # a prompt of one request; a batch of prompts of lengths of their own that goes on from a state
        _heads('scan_1x1024', 'scan', 1, 1024, 128, 8, 64, 'float16'),
        _heads('scan_4x4096_ragged', 'scan', 4, 4096, 128, 8, 64, 'bfloat16', pad=2048, ragged=True, carried=True),
        # a step of training of the scan: a small odd geometry, and the model's
        _heads('train_3x333_odd', 'train', 3, 333, 6, 2, 40, 'bfloat16', ragged=True, carried=True),
        _heads('train_2x2048', 'train', 2, 2048, 128, 8, 64, 'float16'),
        # convolution and scan in a step of training with the input kept in 8 bits
        _heads('mix_2x511_odd', 'mix', 2, 511, 24, 2, 64, 'float16', keep=True),
        _heads('mix_2x2048', 'mix', 2, 2048, 128, 8, 64, 'bfloat16', keep=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(('conv', 'conv_train', 'pack', 'token', 'scan', 'scan', 'train', 'train', 'mix'))
    batch = rng.choice((1, 1, 2, 3, 4, _log_uniform(rng, 1, 16)))
    if op in ('conv', 'conv_train', 'pack'):
        dtype = rng.choice(('float16', 'bfloat16', 'float32'))
        channels = rng.choice((10240, _log_uniform(rng, 16, 12000), 8 * _log_uniform(rng, 4, 1500)))
        most = 4 * 2048 * 10240 // (2 if dtype == 'float32' else 1) // (batch * channels)
        length = _log_uniform(rng, 1, max(1, min(8192, most)))
        return dict(op=op, batch=batch, length=length, channels=channels, dtype=dtype, taps=rng.choice((4, 4, 3, 2)),
                    pad=rng.choice((0, 0, 3, 64)), ragged=op != 'pack' and rng.random() < 0.3,
                    carried=op == 'conv' and rng.random() < 0.5, keep=op == 'conv_train' and rng.random() < 0.5)
    dtype = rng.choice(('float16', 'bfloat16'))
    groups = rng.choice((8, 1, 2, 3))
    heads, dim = groups * rng.choice((16, 16, 1, 2, 4, 5)), rng.choice((64, 64, 64, 128, 32, 40, 9))
    if op == 'token':
        batch, length = _log_uniform(rng, 1, 64), 1
    else:
        most = (4 * 4096 if op == 'scan' else 2 * 2048) * 8192 // (batch * heads * dim)
        length = _log_uniform(rng, 1, max(1, min(16384 if op == 'scan' else 4096, most)))
    return dict(op=op, batch=batch, length=length, heads=heads, groups=groups, dim=dim, dtype=dtype, taps=4,
                pad=rng.choice((0, 0, 3, 64)), ragged=op not in ('token', 'mix') and rng.random() < 0.4,
                carried=op == 'token' or op != 'mix' and rng.random() < 0.5, keep=op == 'mix' and rng.random() < 0.7)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device='cuda')


def _rand(gen, *shape):
    return torch.rand(shape, generator=gen, device='cuda')


def _part(gen, case, width, scale=1.0):
    """[batch, length, width] of a buffer that is `pad` columns wider."""
    buf = torch.empty((case['batch'], case['length'], width + case['pad']), device='cuda', dtype=getattr(torch, case['dtype']))
    for row in buf:
        row.copy_(_randn(gen, *row.shape) * scale)
    return buf[:, :, :width]


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    op, batch, length = case['op'], case['batch'], case['length']
    dtype = getattr(torch, case['dtype'])
    s = dict(case=case, lengths=None, carried=None)
    if case['ragged']:
        s['lengths'] = (_rand(gen, batch) * (length + 1)).to(torch.int32)
        s['lengths'][0] = length
    if op in ('conv', 'conv_train', 'pack', 'mix', 'token'):
        if op in ('mix', 'token'):
            width = case['heads'] * case['dim'] + 2 * case['groups'] * N
        else:
            width = case['channels']
        s['x'] = _part(gen, case, width)
        if op == 'token':
            s['x'] = s['x'][:, 0]
        s['weight'] = (_rand(gen, width, case['taps']) - 0.5).to(dtype)
        s['bias'] = (0.2 * _randn(gen, width)).to(dtype)
        if case['carried']:
            s['carried'] = _randn(gen, batch, case['taps'] - 1, width).to(dtype)
        if op == 'conv_train':
            s['dy'] = _randn(gen, batch, length, width).to(dtype)
            s['leaves'] = [s[k].requires_grad_() for k in ('x', 'weight', 'bias')]
    if op in ('token', 'scan', 'train', 'mix'):
        heads, groups, dim = case['heads'], case['groups'], case['dim']
        # steps of 0.001 to 0.1 and decays of 1 to 16, as the mixers of this model family start with
        step = torch.exp(_rand(gen, heads) * 4.6 - 6.9)
        s['dt_bias'] = (step + torch.log(-torch.expm1(-step))).to(dtype)
        s['dt'] = (0.5 * _randn(gen, batch, length, heads)).to(dtype)
        s['A'] = -(1 + 15 * _rand(gen, heads))
        s['D'] = (1 + 0.1 * _randn(gen, heads)).to(dtype)
        if op == 'token':
            s['dt'] = s['dt'][:, 0]
        if op in ('scan', 'train'):
            s['x'] = _part(gen, case, heads * dim, 0.7).unflatten(2, (heads, dim))
            s['B'] = _part(gen, case, groups * N, 0.5).unflatten(2, (groups, N))
            s['C'] = _part(gen, case, groups * N, 0.5).unflatten(2, (groups, N))
        if case['carried']:
            s['state'] = 0.3 * _randn(gen, batch, heads, dim, N)
        if op in ('train', 'mix'):
            s['dy'] = _randn(gen, batch, length, heads, dim).to(dtype)
            names = (('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias') + (('state',) if case['carried'] else ()) if op == 'train'
                     else ('x', 'dt', 'weight', 'bias', 'D', 'dt_bias'))
            s['leaves'] = [s[k].requires_grad_() for k in names]
    return s


def _present(s, like):
    """1 where a token belongs to its sequence, [batch, length]."""
    if s['lengths'] is None:
        return None
    return torch.arange(s['case']['length'], device='cuda') < s['lengths'][:, None]


# ---------------------------------------------------------------- plain forms

def _plain_conv(s, x):
    """(silu of the convolution, the last taps - 1 inputs) of x [batch, length, width], in 32 bits."""
    taps, length = s['case']['taps'], x.shape[1]
    w, b, x = s['weight'].float(), s['bias'].float(), x.float()
    before = x.new_zeros(x.shape[0], taps - 1, x.shape[2]) if s['carried'] is None else s['carried'].float()
    there = _present(s, x)
    if there is not None:
        x = torch.where(there[..., None], x, 0.0)
    whole = torch.cat([before, x], 1)
    z = sum(whole[:, k:k + length] * w[:, k] for k in range(taps)) + b
    y = z * torch.sigmoid(z)
    if there is not None:
        y = torch.where(there[..., None], y, 0.0)
    ends = torch.full((x.shape[0],), length, device='cuda') if s['lengths'] is None else s['lengths'].long()
    at = ends[:, None] + torch.arange(taps - 1, device='cuda')
    return y, whole.gather(1, at[..., None].expand(-1, -1, x.shape[2]))


def _softplus(v):
    return torch.clamp_min(v, 0.0) + torch.log1p(torch.exp(-v.abs()))


def _plain_scan(s, x, dt, B, C):
    """(y, state after the last token) in 32 bits, chunk by chunk: within a chunk every pair of tokens, between
    chunks the states.  x [b, l, h, p], dt [b, l, h], B and C [b, l, g, n]."""
    b, length, h, p = x.shape
    g = B.shape[2]
    x, B, C, A, D = x.float(), B.float(), C.float(), s['A'].float(), s['D'].float()
    dt = _softplus(dt.float() + s['dt_bias'].float())
    there = _present(s, x)
    if there is not None:
        dt = torch.where(there[..., None], dt, 0.0)
        x = torch.where(there[..., None, None], x, 0.0)
    skip = D[:, None] * x
    nc = -(-length // CHUNK)
    fill = lambda v: torch.cat([v, v.new_zeros(b, nc * CHUNK - length, *v.shape[2:])], 1).unflatten(1, (nc, CHUNK))
    x, B, C = fill(x).unflatten(3, (g, h // g)), fill(B), fill(C)        # [b, c, t, g, k, p], [b, c, t, g, n]
    dt = fill(dt)
    l = torch.cumsum((dt * A).double(), 2)                               # [b, c, t, h]: logarithms of the decays
    at = l.unflatten(3, (g, h // g))
    u = x * dt.unflatten(3, (g, h // g))[..., None]
    gap = (at[:, :, :, None] - at[:, :, None]).float()                   # [b, c, t, s, g, k]
    low = torch.ones(CHUNK, CHUNK, device='cuda', dtype=torch.bool).tril()[..., None, None]
    mix = torch.exp(torch.where(low, gap, float('-inf'))) * torch.einsum('bctgn,bcsgn->bctsg', C, B)[..., None]
    y = torch.einsum('bctsgk,bcsgkp->bctgkp', mix, u)
    add = torch.einsum('bcsgn,bcsgkp->bcgkpn', B, u * torch.exp((at[:, :, -1:] - at).float())[..., None])
    first = s['state'].float().unflatten(1, (g, h // g))[:, None] if s.get('state') is not None else torch.zeros_like(add[:, :1])
    add = torch.cat([first, add], 1)                                     # what each chunk adds, the state carried in first
    ends = torch.cumsum(torch.cat([at.new_zeros(b, 1, g, h // g), at[:, :, -1]], 1), 1)
    gap = (ends[:, :, None] - ends[:, None]).float()
    low = torch.ones(nc + 1, nc + 1, device='cuda', dtype=torch.bool).tril()[..., None, None]
    pass_on = torch.exp(torch.where(low, gap, float('-inf')))            # [b, to, from, g, k]
    states = torch.einsum('bijgk,bjgkpn->bigkpn', pass_on, add)
    y = y + torch.einsum('bctgn,bcgkpn->bctgkp', C, states[:, :-1]) * torch.exp(at.float())[..., None]
    y = y.flatten(1, 2)[:, :length].flatten(2, 3) + skip
    if there is not None:
        y = torch.where(there[..., None, None], y, 0.0)
    return y, states[:, -1].flatten(1, 2)


def _plain_pack(x):
    """(the values that 8 bits hold, in 32 bits, the scales) of x [..., width]."""
    width = x.shape[-1]
    blocks = -(-width // BLOCK)
    v = torch.cat([x.float(), x.new_zeros(*x.shape[:-1], blocks * BLOCK - width, dtype=torch.float32)], -1).unflatten(-1, (blocks, BLOCK))
    scale = v.abs().amax(-1) / 127.0
    codes = torch.round(v / torch.where(scale == 0, 1.0, scale)[..., None]).clamp(-127, 127)
    return (codes * scale[..., None]).flatten(-2)[..., :width], scale


def _plain_token(s):
    case, x, dtype = s['case'], s['x'].float(), s['x'].dtype
    heads, groups, dim = case['heads'], case['groups'], case['dim']
    w, b = s['weight'].float(), s['bias'].float()
    whole = torch.cat([s['carried'].float(), x[:, None]], 1)
    z = (whole * w.T).sum(1) + b
    z = z * torch.sigmoid(z)
    s['carried'].copy_(whole[:, 1:])
    u, B, C = z.split([heads * dim, groups * N, groups * N], -1)
    u = u.unflatten(1, (heads, dim))
    B, C = (v.unflatten(1, (groups, N)).repeat_interleave(heads // groups, 1) for v in (B, C))
    dt = _softplus(s['dt'].float() + s['dt_bias'].float())
    state = s['state'] * torch.exp(dt * s['A'])[..., None, None] + (dt[..., None] * u)[..., None] * B[:, :, None]
    s['state'].copy_(state)
    y = (state * C[:, :, None]).sum(-1) + s['D'].float()[:, None] * u
    return y.to(dtype), s['carried'], s['state']


def _split(s, z):
    case = s['case']
    heads, groups, dim = case['heads'], case['groups'], case['dim']
    x, B, C = z.split([heads * dim, groups * N, groups * N], -1)
    return x.unflatten(2, (heads, dim)), B.unflatten(2, (groups, N)), C.unflatten(2, (groups, N))


def _plain(s):
    case, dtype = s['case'], s['x'].dtype
    op = case['op']
    if op == 'conv':
        y, last = _plain_conv(s, s['x'])
        return y.to(dtype), last.to(dtype)
    if op == 'conv_train':
        y, _ = _plain_conv(s, s['x'])
        out = y.detach().to(dtype)
        if case['keep']:
            held = _plain_pack(s['x'].detach())[0].requires_grad_()
            dx, *rest = torch.autograd.grad(_plain_conv(s, held)[0], [held, *s['leaves'][1:]], s['dy'].float())
            return [out, dx.to(dtype), *rest]
        return [out, *torch.autograd.grad(y, s['leaves'], s['dy'].float())]
    if op == 'pack':
        values, scales = _plain_pack(s['x'])
        return values.to(dtype), scales
    if op == 'token':
        return _plain_token(s)
    if op == 'scan':
        y, last = _plain_scan(s, s['x'], s['dt'], s['B'], s['C'])
        return y.to(dtype), last
    if op == 'train':
        y, _ = _plain_scan(s, s['x'], s['dt'], s['B'], s['C'])
        return [y.detach().to(dtype), *torch.autograd.grad(y, s['leaves'], s['dy'].float())]
    forward = lambda v: _plain_scan(s, *(lambda x, B, C: (x, s['dt'], B, C))(*_split(s, _plain_conv(s, v)[0])))[0]
    if not case['keep']:
        y = forward(s['x'])
        return [y.detach().to(dtype), *torch.autograd.grad(y, s['leaves'], s['dy'].float())]
    with torch.no_grad():
        out = forward(s['x']).to(dtype)
    held = _plain_pack(s['x'].detach())[0].requires_grad_()
    dx, *rest = torch.autograd.grad(forward(held), [held, *s['leaves'][1:]], s['dy'].float())
    return [out, dx.to(dtype), *rest]


# ---------------------------------------------------------------- the library's calls

def _own(s):
    sq325 = _package()
    case = s['case']
    op, keep = case['op'], 'int8' if case['keep'] else None
    if op == 'conv':
        return sq325.causal_conv(s['x'], s['weight'], s['bias'], initial_state=s['carried'], lengths=s['lengths'],
                                 return_final_state=True)
    if op == 'conv_train':
        y = sq325.causal_conv(s['x'], s['weight'], s['bias'], lengths=s['lengths'], keep=keep)
        return [y.detach(), *torch.autograd.grad(y, s['leaves'], s['dy'])]
    if op == 'pack':
        packed = sq325.pack_activations(s['x'])
        return sq325.unpack_activations(packed), packed.scales
    if op == 'token':
        y = sq325.conv_scan_step(s['x'], s['dt'], s['A'], s['weight'], s['bias'], s['D'], s['dt_bias'], heads=case['heads'],
                                 groups=case['groups'], conv_state=s['carried'], state=s['state'])
        return y, s['carried'], s['state']
    if op == 'scan':
        return sq325.selective_scan(s['x'], s['dt'], s['A'], s['B'], s['C'], s['D'], s['dt_bias'],
                                    initial_state=s.get('state'), lengths=s['lengths'], return_final_state=True)
    if op == 'train':
        y = sq325.selective_scan(s['x'], s['dt'], s['A'], s['B'], s['C'], s['D'], s['dt_bias'],
                                 initial_state=s.get('state'), lengths=s['lengths'])
    else:
        y = sq325.conv_scan(s['x'], s['dt'], s['A'], s['weight'], s['bias'], s['D'], s['dt_bias'], heads=case['heads'],
                            groups=case['groups'], keep=keep)
    return [y.detach(), *torch.autograd.grad(y, s['leaves'], s['dy'])]


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- 64 bits, from the definitions

def _double(s, names):
    return {k: s[k].detach().double().requires_grad_() for k in names}


def _exact_conv(s, x, w, b):
    """The convolution's definition: its output at t is a sum over the inputs at t - taps + 1 .. t."""
    taps, length = s['case']['taps'], x.shape[1]
    there = _present(s, x)
    if there is not None:
        x = x * there[..., None]
    z = b.expand(x.shape).clone()
    for k in range(taps):                                    # the tap that looks back taps - 1 - k tokens
        back = taps - 1 - k
        far = x[:, :max(0, length - back)] * w[:, k]
        z = z + torch.nn.functional.pad(far, (0, 0, length - far.shape[1], 0))
        if s['carried'] is not None and back:
            n = min(back, length)
            old = s['carried'].double()[:, taps - 1 - back:taps - 1 - back + n] * w[:, k]
            z = z + torch.nn.functional.pad(old, (0, 0, 0, length - n))
    y = z / (1 + torch.exp(-z))
    return y if there is None else y * there[..., None]


def _exact_scan(s, x, dt, A, B, C, D, dt_bias, state, dy=None):
    """y and the last state from the whole sequence's pairs of tokens, one head at a time; with dy their gradients."""
    b, length, h, p = x.shape
    per = h // B.shape[2]
    y, last = torch.empty_like(x), x.new_empty(b, h, p, N)
    low = torch.ones(length, length, device='cuda', dtype=torch.bool).tril()
    given = [v for v in (x, dt, A, B, C, D, dt_bias, state) if v is not None]
    grads = [torch.zeros_like(v) for v in given] if dy is not None else None
    for i in range(b):
        end = length if s['lengths'] is None else int(s['lengths'][i])
        for j in range(h):
            g = j // per
            at = [(i, slice(0, end), j), (i, slice(0, end), j), (j,), (i, slice(0, end), g), (i, slice(0, end), g), (j,), (j,), (i, j)]
            leaf = [None if v is None else v.detach()[k].clone().requires_grad_(dy is not None)
                    for v, k in zip((x, dt, A, B, C, D, dt_bias, state), at)]
            xi, ti, Ai, Bi, Ci, Di, bi, hi = leaf
            with torch.set_grad_enabled(dy is not None):
                step = torch.logaddexp(ti + bi, torch.zeros_like(ti))
                l = torch.cumsum(step * Ai, 0)
                weight = torch.exp(torch.where(low[:end, :end], l[:, None] - l, -torch.inf)) * (Ci @ Bi.T) * step
                yi = weight @ xi + Di * xi
                tail = torch.exp(l[-1] - l) if end else l
                hN = (xi * (tail * step)[:, None]).T @ Bi
                if hi is not None:
                    yi = yi + torch.exp(l)[:, None] * (Ci @ hi.T)
                    hN = hN + (torch.exp(l[-1]) if end else 1.0) * hi
            y[i, :end, j], y[i, end:, j], last[i, j] = yi.detach(), 0.0, hN.detach()
            if dy is not None and end:
                real, places = zip(*[(v, k) for v, k in zip(leaf, at) if v is not None])
                got = torch.autograd.grad(yi, real, dy[i, :end, j])
                for total, k, v in zip(grads, places, got):
                    total[k] += v
    return y, last, grads


def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    kept = (lambda x: _exact_pack(x)[0]) if case['keep'] else (lambda x: x)
    if op == 'conv':
        y = _exact_conv(s, s['x'].double(), s['weight'].double(), s['bias'].double())
        return y, None
    if op == 'conv_train':
        v = _double(s, ('x', 'weight', 'bias'))
        y = _exact_conv(s, v['x'], v['weight'], v['bias']).detach()
        held = kept(v['x'].detach()).requires_grad_()
        got = torch.autograd.grad(_exact_conv(s, held, v['weight'], v['bias']), [held, v['weight'], v['bias']], s['dy'].double())
        return [y, *got]
    if op == 'pack':
        return _exact_pack(s['x'].double())
    if op == 'token':
        heads, groups, dim = case['heads'], case['groups'], case['dim']
        w = s['weight'].double()
        z = s['bias'].double() + s['x'].double() * w[:, -1] + torch.einsum('bkc,ck->bc', s['carried'].double(), w[:, :-1])
        u, B, C = (z / (1 + torch.exp(-z))).split([heads * dim, groups * N, groups * N], -1)
        u, per = u.unflatten(1, (groups, heads // groups, dim)), heads // groups
        B, C = B.unflatten(1, (groups, N)), C.unflatten(1, (groups, N))
        dt = torch.logaddexp(s['dt'].double() + s['dt_bias'].double(), torch.zeros_like(s['dt'], dtype=torch.double)).unflatten(1, (groups, per))
        decay = torch.exp(dt * s['A'].double().unflatten(0, (groups, per)))
        state = s['state'].double().unflatten(1, (groups, per))
        state = torch.einsum('bgk,bgkpn->bgkpn', decay, state) + torch.einsum('bgk,bgkp,bgn->bgkpn', dt, u, B)
        y = torch.einsum('bgkpn,bgn->bgkp', state, C) + torch.einsum('gk,bgkp->bgkp', s['D'].double().unflatten(0, (groups, per)), u)
        return y.flatten(1, 2), None, state.flatten(1, 2)
    if case['batch'] * case['heads'] * max(1.0, (case['length'] / 2048) ** 2) > 4096:
        return None                                          # too long a wait
    if op in ('scan', 'train'):
        v = [None if s.get(k) is None else s[k].detach().double() for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias', 'state')]
        y, last, grads = _exact_scan(s, *v, dy=s['dy'].double() if op == 'train' else None)
        return [y, *grads] if op == 'train' else (y, last)
    v = _double(s, ('x', 'dt', 'weight', 'bias', 'D', 'dt_bias'))
    parts = lambda x: [t.contiguous() for t in _split(s, _exact_conv(s, x, v['weight'], v['bias']))]
    scan = lambda t, dy=None: _exact_scan(s, t[0], v['dt'].detach(), s['A'].double(), t[1], t[2], v['D'].detach(), v['dt_bias'].detach(), None, dy)
    y = scan([t.detach() for t in parts(v['x'])])[0]
    held = kept(v['x'].detach()).requires_grad_()
    t = parts(held)
    _, _, (dx, ddt, _, dB, dC, dD, dbias) = scan([u.detach() for u in t], s['dy'].double())
    dheld, dw, db = torch.autograd.grad(t, [held, v['weight'], v['bias']], [dx, dB, dC])
    return [y, dheld, ddt, dw, db, dD, dbias]


def _exact_pack(x):
    """The values and scales that 8 bits hold of x in 64 bits; blocks of whole columns, the last one cut."""
    values, scales = torch.empty_like(x), []
    for at in range(0, x.shape[-1], BLOCK):
        part = x[..., at:at + BLOCK]
        scale = part.abs().amax(-1, keepdim=True) / 127
        values[..., at:at + BLOCK] = torch.round(torch.nan_to_num(part / scale, 0.0)).clamp(-127, 127) * scale
        scales.append(scale)
    return values, torch.cat(scales, -1)


def work(case):
    """Bytes: each input read once, each output written once.  Operations: products and sums of the definition taken
    token by token (scan: the state's update and its readout, 4 a state element, and their three gradients)."""
    b, length, size = case['batch'], case['length'], torch.tensor([], dtype=getattr(torch, case['dtype'])).element_size()
    op, taps = case['op'], case['taps']
    if op in ('conv', 'conv_train', 'pack'):
        width, tokens = case['channels'], b * length
        if op == 'pack':     # the input, codes and scales, and the values made of them
            return dict(bytes=tokens * (width * (2 * size + 2) + 8 * -(-width // BLOCK)), flops=4 * tokens * width)
        if op == 'conv':
            last = b * (taps - 1) * width * size
            return dict(bytes=tokens * width * 2 * size + (1 + case['carried']) * last + (taps + 1) * width * size, flops=2 * taps * tokens * width)
        return dict(bytes=tokens * width * 4 * size + 2 * (taps + 1) * width * size, flops=3 * 2 * taps * tokens * width)
    h, g, p = case['heads'], case['groups'], case['dim']
    tokens, state = b * length, b * h * p * N
    inner = tokens * (h * p + h + 2 * g * N) * size          # x, dt, B, C
    params = h * (4 + 2 * size)
    out = tokens * h * p * size
    if op == 'token':
        width = h * p + 2 * g * N
        return dict(bytes=b * (width * (2 * (taps - 1) + 1) + h + h * p) * size + width * (taps + 1) * size + params + 8 * state,
                    flops=b * width * 2 * taps + 5 * state)
    if op == 'scan':
        return dict(bytes=inner + out + params + 4 * state * (1 + case['carried']), flops=5 * tokens * h * p * N)
    both = 2 * inner + 2 * out + 2 * params + (8 * state if case['carried'] else 0)
    if op == 'mix':
        both += 2 * (h * p + 2 * g * N) * (taps + 1) * size
    return dict(bytes=both, flops=15 * tokens * h * p * N)
