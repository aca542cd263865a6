"""GPU tests of the operators on rows of logits against the 64-bit oracle: sq325.sample,
top_logits, distillation_loss (with its backward) and distillation_loss_grad.

Tolerances.  A draw's weights carry a relative error of at most (|t| + 4) 2^-24 with t the
exponent (|t| <= 32 where the weight is not 0) plus half a step of 2^-31 each, so weight sums
are off by less than 3e-6 + vocab 2^-32 < 7e-5 of the largest sum in the worst case and by
about 1e-6 in practice: a draw whose margin is over 1e-4 must give the oracle's token, one with a
smaller margin is not compared.  The loss and gradient bounds are written at their use.
"""
import numpy as np
import pytest
import torch

from oracle import logits as ol

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]
MARGIN = 1e-4


def make(rows, vocab, dtype, seed, spread=3.0, pad=0, offset=0, banned=0.0):
    """Logits with a few that stand out; `offset` shifts the rows' start off 16-byte boundaries."""
    g = torch.Generator(device='cuda').manual_seed(seed)
    buf = torch.randn(rows * (vocab + pad) + offset, generator=g, device='cuda') * spread
    x = buf[offset:].view(rows, vocab + pad)
    few = max(1, min(20, vocab // 4))
    at = (torch.arange(few, device='cuda') * (vocab // few)).expand(rows, few)
    x.scatter_(1, at, 3.0 + 9.0 * torch.rand((rows, few), generator=g, device='cuda'))
    if banned:
        x[:, :vocab].masked_fill_(torch.rand(vocab, generator=g, device='cuda') < banned, float('-inf'))
    out = torch.empty(rows * (vocab + pad) + offset, device='cuda', dtype=dtype)
    out[offset:].copy_(x.reshape(-1).to(dtype))
    return out[offset:].view(rows, vocab + pad)[:, :vocab], g


def wide(x):
    return x.detach().cpu().double().numpy()


def check_draw(x, u, t=1.0, k=0, p=1.0, q=0.0, least=0.5):
    import sq325
    got = sq325.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=q).cpu().numpy()
    pick = lambda v, r: float(v[r]) if isinstance(v, torch.Tensor) else v
    xs, us = wide(x), u.cpu().numpy()
    compared = 0
    for r in range(len(xs)):
        want, margin = ol.draw(xs[r], us[r], pick(t, r), int(pick(k, r)), pick(p, r), pick(q, r))
        if margin > MARGIN:
            compared += 1
            assert got[r] == want, (r, got[r], want, margin)
        elif want >= 0:
            assert 0 <= got[r] < xs.shape[1] and xs[r, got[r]] > -np.inf
    assert compared >= least * len(xs)
    return got


SETTINGS = [dict(t=0.0), dict(t=0.7), dict(k=1), dict(k=7), dict(k=50, p=0.9, t=0.8), dict(p=0.8), dict(p=0.95, t=0.6),
            dict(q=0.1), dict(k=20, p=0.9, q=0.05, t=1.3), dict(p=1e-6)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [1, 2, 31, 257, 1000, 5003])
def test_draw_matches_oracle(vocab, dtype):
    x, g = make(16, vocab, dtype, seed=vocab, pad=3, offset=1)
    for s in SETTINGS:
        check_draw(x, torch.rand(16, generator=g, device='cuda'), **s)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [32003, 256000, 262144])
@pytest.mark.parametrize('spread', [1.0, 3.0])
def test_draw_large_vocab(vocab, dtype, spread):
    x, g = make(4, vocab, dtype, seed=vocab, spread=spread, pad=1, banned=0.05)
    for s in (dict(k=50, p=0.9, t=0.8), dict(k=2000, p=0.9), dict(p=0.7, t=0.8), dict(p=0.9), dict(q=0.02), dict(t=0.0)):
        check_draw(x, torch.rand(4, generator=g, device='cuda'), least=0.0, **s)


def test_draw_settings_per_row():
    x, g = make(64, 4099, torch.float16, seed=3)
    pick = lambda v, d: torch.tensor(v, device='cuda', dtype=d)[torch.randint(0, len(v), (64,), generator=g, device='cuda')]
    check_draw(x, torch.rand(64, generator=g, device='cuda'), t=pick([0.0, 0.5, 1.0], torch.float32),
               k=pick([0, 1, 40], torch.int32), p=pick([0.5, 0.9, 1.0], torch.float32), q=pick([0.0, 0.1], torch.float32))


@pytest.mark.parametrize('vocab,settings', [(37, dict()), (1500, dict(top_k=9)), (1500, dict(top_p=0.9)),
                                            (70001, dict(top_p=0.6)), (70001, dict(top_k=3000, top_p=0.5, temperature=1.5))])
def test_draw_follows_the_distribution(vocab, settings):
    """The same row drawn at an even grid of uniform numbers: every token as often as its share says."""
    import sq325
    x, _ = make(1, vocab, torch.float32, seed=5)
    n = 4096
    u = (torch.arange(n, device='cuda') + 0.5) / n
    got = sq325.sample(x.expand(n, vocab), u, **settings).cpu().numpy()
    xs = wide(x)[0]
    T = settings.get('temperature', 1.0)
    by = ol.order(xs)
    w = np.exp((xs[by] - xs.max()) / T)
    if settings.get('top_k'):
        w[settings['top_k']:] = 0
    if settings.get('top_p'):
        w[np.cumsum(w) - w >= settings['top_p'] * w.sum()] = 0
    share = np.zeros(vocab)
    share[by] = w / w.sum()
    assert (np.diff(got) >= 0).all()                     # the draw is monotone in the uniform number
    # a grid of n points puts n share +- 1 of them into an interval; sums are 1e-4 off at most, and
    # the cut of top-p may take one token more or less
    assert np.abs(np.bincount(got, minlength=vocab) - n * share).max() <= 2 + n * MARGIN


@pytest.mark.parametrize('dtype', TYPES)
def test_draw_ties_masks_and_nonfinite(dtype):
    import sq325
    inf = float('inf')
    u = lambda *v: torch.tensor(v, device='cuda')
    for vocab in (64, 5003, 70001):
        x = torch.zeros((4, vocab), device='cuda', dtype=dtype)
        # all equal: ties go by index
        got = sq325.sample(x, u(0.0, 0.25, 0.5, 0.999), top_k=4).tolist()
        assert got == [0, 1, 2, 3]
        got = sq325.sample(x, u(0.0, 0.25, 0.5, 0.999)).tolist()
        assert got == [0, vocab // 4, vocab // 2, int(np.floor(np.float32(0.999).astype(np.float64) * vocab))]
        p = 0.5
        last = int(np.ceil(p * vocab)) - 1
        assert sq325.sample(x, u(0.0, 0.0, 1.0 - 2 ** -24, 1.0 - 2 ** -24), top_p=p).tolist() == [0, 0, last, last]
        x[:, ::2] = -0.0                                 # -0 and +0 are equal
        assert sq325.sample(x, u(0.0, 0.25, 0.5, 0.999), top_k=4).tolist() == [0, 1, 2, 3]
        x = torch.full((6, vocab), -inf, device='cuda', dtype=dtype)
        x[1, vocab - 1] = -5.0                           # one token left
        x[2] = float('nan')
        x[2, 7] = 1.0
        x[3] = torch.finfo(dtype).min                    # masked by the lowest value: still tokens
        x[4, 3] = x[4, 9] = inf
        x[4, 5] = 2.0
        x[5] = float('nan')
        for s in (dict(), dict(top_k=3), dict(top_p=0.9), dict(min_p=0.2), dict(temperature=0.0),
                  dict(top_k=1100, top_p=0.99, min_p=0.1)):
            got = sq325.sample(x, u(0.6, 0.6, 0.6, 0.0, 0.6, 0.6), **s).tolist()
            assert got == [-1, vocab - 1, 7, 0, 3 if s.get('temperature') == 0.0 else 9, -1], s
    x, g = make(8, 3001, dtype, seed=9)
    r = torch.rand(8, generator=g, device='cuda')
    base = sq325.sample(x, r, top_k=100, top_p=0.9)
    holes = torch.cat([x, torch.full((8, 700), float('nan'), device='cuda', dtype=dtype),
                       torch.full((8, 5), torch.finfo(dtype).min, device='cuda', dtype=dtype)], 1)
    assert torch.equal(base, sq325.sample(holes, r, top_k=100, top_p=0.9))


def test_draw_extremes_of_temperature():
    import sq325
    x, g = make(8, 999, torch.float32, seed=1)
    u = torch.rand(8, generator=g, device='cuda')
    assert torch.equal(sq325.sample(x, u, temperature=1e-30), x.argmax(1))
    assert torch.equal(sq325.sample(x, u, temperature=1e-42), x.argmax(1))
    got = sq325.sample(x, u, temperature=1e30)           # even over the vocabulary
    assert (got.double() - torch.floor(u.double() * 999)).abs().max() <= 1
    t = torch.full((8,), float('nan'), device='cuda')    # a setting that is no temperature: greedy
    assert torch.equal(sq325.sample(x, u, temperature=t), x.argmax(1))


def test_draw_shapes_streams_and_repeats():
    import sq325
    x, g = make(12, 20011, torch.bfloat16, seed=2, pad=5)
    u = torch.rand(12, generator=g, device='cuda')
    want = sq325.sample(x, u, top_p=0.9)
    assert torch.equal(want.view(3, 4), sq325.sample(x.reshape(3, 4, -1), u.view(3, 4), top_p=0.9))
    assert torch.equal(want[5], sq325.sample(x[5], u[5], top_p=0.9))
    assert torch.equal(want, sq325.sample(x.t().contiguous().t(), u, top_p=0.9))      # not contiguous along the row
    assert sq325.sample(x[:0], u[:0]).shape == (0,)
    for _ in range(5):
        assert torch.equal(want, sq325.sample(x, u, top_p=0.9))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        y = x * 1.0
        got = sq325.sample(y, u, top_p=0.9)
    side.synchronize()
    assert torch.equal(want, got)


def test_draw_more_rows_than_fit_at_once():
    x, g = make(1500, 1013, torch.float16, seed=4)
    check_draw(x, torch.rand(1500, generator=g, device='cuda'), k=40, p=0.9, least=0.9)


# ------------------------------------------------------------------ the largest logits
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,vocab,k,pad,offset', [(1, 1, 1, 0, 0), (3, 2, 2, 1, 1), (5, 33, 33, 0, 3), (7, 1000, 1, 5, 0),
                                                     (7, 1000, 1000, 0, 0), (4, 5003, 64, 3, 1), (3, 70001, 1024, 1, 0),
                                                     (2, 256000, 20, 0, 0), (2, 262144, 333, 7, 1), (700, 1021, 17, 0, 0)])
def test_top_logits(rows, vocab, k, pad, offset, dtype):
    import sq325
    x, _ = make(rows, vocab, dtype, seed=vocab + k, pad=pad, offset=offset, banned=0.1 if vocab > 100 else 0.0)
    values, indices = sq325.top_logits(x, k)
    assert values.dtype == dtype and indices.dtype == torch.int32 and values.shape == indices.shape == (rows, k)
    xs = wide(x)
    for r in range(min(rows, 40)):
        v, i = ol.top(xs[r], k)
        assert np.array_equal(indices[r].cpu().numpy(), i)
        assert np.array_equal(wide(values[r]), v)


@pytest.mark.parametrize('dtype', TYPES)
def test_top_logits_ties_and_masks(dtype):
    import sq325
    inf = float('inf')
    for vocab in (50, 4097, 70001):
        x = torch.zeros((7, vocab), device='cuda', dtype=dtype)
        x[1] = -inf
        x[2] = -inf
        x[2, [3, 41]] = torch.tensor([1.0, 2.0], device='cuda', dtype=dtype)
        x[3] = float('nan')
        x[3, 40] = torch.finfo(dtype).min
        x[4, 10] = inf
        x[4, 49] = 3.0
        x[5, ::3] = -0.0
        x[6] = torch.finfo(dtype).min
        x[6, 5] = -inf
        values, indices = sq325.top_logits(x, 6)
        xs = wide(x)
        for r in range(7):
            v, i = ol.top(xs[r], 6)
            assert np.array_equal(indices[r].cpu().numpy(), i), (vocab, r)
            assert np.array_equal(wide(values[r]), v)


# ------------------------------------------------------------------ distillation
def record(g, rows, vocab, k, dtype, cut=0.3):
    at = torch.rand((rows, vocab), generator=g, device='cuda').argsort(1)[:, :k] if vocab <= 6000 else \
        (torch.randint(0, vocab, (rows, 1), generator=g, device='cuda') + torch.arange(k, device='cuda') * (vocab // k)) % vocab
    values = (torch.randn((rows, k), generator=g, device='cuda') * 3).to(dtype)
    gone = torch.rand((rows, k), generator=g, device='cuda') < cut
    return values, at.int().masked_fill(gone, -1)


UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}


def check_distill(x, values, indices, T, weight, loss, grad=None):
    """fp32 chains: the exponent t of a power carries |t| 2^-23 (a difference, a product), the
    hardware's power 2^-22, a sum of n terms added by 512 threads n / 512 + 20 roundings.  With
    e = (|t| + n / 512 + 40) 2^-23: p and q are off by e relative, the loss by T^2 e (1 + |log|) per
    unit of q, the gradient by T w e (p + q) and its own rounding."""
    vocab, k = x.shape[1], values.shape[1]
    xs, vs, js, ws = wide(x), wide(values), indices.cpu().numpy(), wide(weight)
    for r in range(len(xs)):
        want, g, p, q = ol.distill(xs[r], vs[r], js[r], T, ws[r])
        if not (js[r] >= 0).any():
            assert float(loss[r]) == 0.0
            assert grad is None or not grad[r].any()
            continue
        finite = xs[r][np.isfinite(xs[r])]
        far = (finite.max() - finite.min()) / T * 1.45
        e = (far + (vocab + k) / 512 + 40) * 2.0 ** -23
        assert abs(float(loss[r]) - want) <= T * T * e * (1 + 3 * far), r
        if grad is not None:
            got = wide(grad[r])
            bound = T * abs(ws[r]) * e * (p + q) + UNIT[x.dtype] * np.abs(g) * 1.01 + LEAST[x.dtype]
            assert (np.abs(got - g) <= bound).all(), (r, np.abs(got - g).max())


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,vocab,k,T,pad,offset', [(1, 1, 1, 1.0, 0, 0), (5, 2, 2, 2.0, 1, 1), (3, 33, 5, 0.7, 3, 0),
                                                       (9, 1000, 64, 1.0, 0, 0), (8, 5003, 17, 2.5, 1, 1),
                                                       (6, 5003, 1024, 1.0, 0, 3), (3, 70001, 100, 1.0, 2, 0),
                                                       (3, 256000, 64, 2.0, 0, 0), (2, 262143, 1, 1.0, 1, 0)])
def test_distillation(rows, vocab, k, T, pad, offset, dtype):
    import sq325
    x, g = make(rows, vocab, dtype, seed=vocab + k, pad=pad, offset=offset)
    values, indices = record(g, rows, vocab, k, dtype)
    weight = torch.rand(rows, generator=g, device='cuda') * 8 - 2
    loss, grad = sq325.distillation_loss_grad(x, values, indices, temperature=T, weight=weight)
    assert loss.dtype == torch.float32 and grad.dtype == dtype and grad.shape == x.shape
    check_distill(x, values, indices, T, weight, loss, grad)
    check_distill(x, values, indices, T, weight, sq325.distillation_loss(x, values, indices, temperature=T))
    y = x.detach().requires_grad_(True)
    loss = sq325.distillation_loss(y, values, indices, temperature=T)
    check_distill(x, values, indices, T, weight, loss.detach(), torch.autograd.grad(loss, y, weight)[0])


def test_distillation_many_rows():
    import sq325
    x, g = make(1300, 777, torch.float16, seed=1)
    values, indices = record(g, 1300, 777, 9, torch.float16)
    weight = torch.ones(1300, device='cuda')
    loss, grad = sq325.distillation_loss_grad(x, values, indices)
    check_distill(x, values, indices, 1.0, weight, loss, grad)
    y = x.detach().requires_grad_(True)
    loss = sq325.distillation_loss(y, values, indices)
    check_distill(x, values, indices, 1.0, weight, loss.detach(), torch.autograd.grad(loss.sum(), y)[0])


@pytest.mark.parametrize('dtype', TYPES)
def test_distillation_masks_and_repeats(dtype):
    import sq325
    vocab = 3001
    x, g = make(8, vocab, dtype, seed=11)
    values, indices = record(g, 8, vocab, 40, torch.float32, cut=0.0)
    indices[0] = -1                                      # no teacher
    indices[1, 5:] = -1
    indices[2, ::2] = indices[2, 0].clone()              # one token twenty times
    indices[3, 3] = vocab                                # outside the vocabulary
    values[4, 1] = float('-inf')
    values[4, 2] = float('nan')
    values[5] = float('-inf')                            # a record without values
    free = torch.ones(vocab, dtype=torch.bool, device='cuda')
    free[indices[6].long()] = False
    x[6].masked_fill_(free & (torch.arange(vocab, device='cuda') % 2 == 0), float('-inf'))
    x[7].masked_fill_(torch.arange(vocab, device='cuda') % 3 == 0, torch.finfo(dtype).min)
    x[7].scatter_(0, indices[7].long(), torch.ones(40, device='cuda', dtype=dtype))
    weight = torch.linspace(-1, 2, 8, device='cuda')
    seen = indices.clone()
    seen[5] = -1
    values_seen = torch.where(torch.isnan(values), float('-inf'), values)
    loss, grad = sq325.distillation_loss_grad(x, values, indices, weight=weight)
    check_distill(x, values_seen, seen, 1.0, weight, loss, grad)
    y = x.detach().requires_grad_(True)
    loss = sq325.distillation_loss(y, values, indices)
    check_distill(x, values_seen, seen, 1.0, weight, loss.detach(), torch.autograd.grad(loss, y, weight)[0])


@pytest.mark.parametrize('dtype', TYPES)
def test_distillation_rows_of_the_lowest_value(dtype):
    """A student row masked by the type's lowest value everywhere is even; one logit above takes it all."""
    import sq325
    vocab = 2003
    x = torch.full((3, vocab), torch.finfo(dtype).min, device='cuda', dtype=dtype)
    x[1, 7] = 0.0
    x[2, ::2] = float('-inf')
    values = torch.zeros((3, 2), device='cuda')
    indices = torch.tensor([[7, 9]] * 3, device='cuda', dtype=torch.int32)
    left = [vocab, 1, vocab // 2]
    want = torch.zeros((3, vocab), dtype=torch.float64)
    want[0] = 1 / left[0]
    want[1, 7] = 1.0
    want[2, 1::2] = 1 / left[2]
    want[:, [7, 9]] -= 0.5
    y = x.detach().requires_grad_(True)
    again = sq325.distillation_loss(y, values, indices)
    for loss, grad in (sq325.distillation_loss_grad(x, values, indices), (again.detach(), torch.autograd.grad(again.sum(), y)[0])):
        assert abs(float(loss[0]) - np.log(left[0] / 2)) < 1e-5 and abs(float(loss[2]) - np.log(left[2] / 2)) < 1e-5
        assert float(loss[1]) > 1e4                      # half of the teacher's weight lies where the student has none
        assert ((grad.double().cpu() - want).abs() <= 2 ** -8 * want.abs() + 1e-6).all()


def test_distillation_undefined_student():
    import sq325
    x = torch.zeros((5, 600), device='cuda')
    x[0, 3] = float('nan')
    x[1, 3] = float('inf')
    x[2] = float('-inf')
    x[3, 4] = float('-inf')                              # the teacher's token is masked: the loss is infinite
    values = torch.zeros((5, 2), device='cuda')
    indices = torch.tensor([[4, 5]], device='cuda', dtype=torch.int32).expand(5, 2).contiguous()
    indices[4] = -1
    x[4] = float('nan')                                  # no teacher: nothing is learnt
    loss, grad = sq325.distillation_loss_grad(x, values, indices)
    y = x.clone().requires_grad_(True)
    again = sq325.distillation_loss(y, values, indices)
    back = torch.autograd.grad(again.sum(), y)[0]
    for l, g in ((loss, grad), (again, back)):
        assert l[:3].isnan().all() and g[:3].isnan().all()
        assert l[3] == float('inf') and g[3].isfinite().all() and g[3, 4] == -0.5
        assert l[4] == 0 and not g[4].any()


def test_distillation_gradient_against_differences():
    """Central differences of the loss along random directions: with a step h = 2^-5 the fp32 loss
    (about 5, off by 1e-6) gives slopes good to 1e-6 / h, the third derivative adds h^2."""
    import sq325
    x, g = make(6, 403, torch.float32, seed=8, spread=1.0)
    values, indices = record(g, 6, 403, 30, torch.float32)
    _, grad = sq325.distillation_loss_grad(x, values, indices, temperature=1.5)
    h = 2.0 ** -5
    for _ in range(8):
        d = torch.randn(x.shape, generator=g, device='cuda')
        up, down = (sq325.distillation_loss(x + s * h * d, values, indices, temperature=1.5) for s in (1, -1))
        slope = (up.double() - down.double()) / (2 * h)
        assert (slope - (grad.double() * d.double()).sum(1)).abs().max() <= 1e-4 + 4 * h * h


def test_distillation_shapes_strides_and_reductions():
    import sq325
    x, g = make(12, 2003, torch.bfloat16, seed=6, pad=4)
    values, indices = record(g, 12, 2003, 10, torch.bfloat16)
    loss, grad = sq325.distillation_loss_grad(x, values, indices)
    l3, g3 = sq325.distillation_loss_grad(x.reshape(3, 4, -1), values.view(3, 4, 10), indices.view(3, 4, 10))
    assert torch.equal(l3.view(-1), loss) and torch.equal(g3.view(12, -1), grad)
    l0, g0 = sq325.distillation_loss_grad(x[2], values[2], indices[2])
    assert l0.shape == () and torch.equal(l0, loss[2]) and torch.equal(g0, grad[2])
    y = x.detach().clone().requires_grad_(True)          # a mean's upstream gradient is one broadcast number
    sq325.distillation_loss(y, values, indices).mean().backward()
    _, want = sq325.distillation_loss_grad(x, values, indices, weight=torch.full((12,), 1 / 12, device='cuda'))
    assert torch.allclose(y.grad.float(), want.float(), rtol=2 ** -7, atol=1e-7)
    _, same = sq325.distillation_loss_grad(x, values, indices, weight=torch.full((1,), 1 / 12, device='cuda').expand(12))
    assert torch.equal(same, want)
    z = x.t().contiguous().t().detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(sq325.distillation_loss(z, values, indices).sum(), z)[0], grad)
    e = sq325.distillation_loss_grad(x[:0], values[:0], indices[:0])
    assert e[0].shape == (0,) and e[1].shape == (0, 2003)
    shared, _ = sq325.distillation_loss_grad(x[:1].expand(12, 2003), values, indices)     # one row read by all
    assert shared.isfinite().all() and torch.equal(shared[0], loss[0])


# ------------------------------------------------------------------ refusals
def test_refusals():
    import sq325
    x = torch.zeros((2, 10), device='cuda')
    u = torch.zeros(2, device='cuda')
    v, i = torch.zeros((2, 3), device='cuda'), torch.zeros((2, 3), device='cuda', dtype=torch.int32)
    bad = [lambda: sq325.sample(x.cpu(), u), lambda: sq325.sample(x.double(), u), lambda: sq325.sample(x, u[:1]),
           lambda: sq325.sample(x, u.double()), lambda: sq325.sample(x, u.cpu()), lambda: sq325.sample(x[:, :0], u),
           lambda: sq325.sample(torch.zeros((1, (1 << 18) + 1), device='cuda'), u[:1]),
           lambda: sq325.sample(x, u, temperature=-1.0), lambda: sq325.sample(x, u, temperature=float('inf')),
           lambda: sq325.sample(x, u, temperature=float('nan')), lambda: sq325.sample(x, u, top_k=-1),
           lambda: sq325.sample(x, u, top_k=2.0), lambda: sq325.sample(x, u, top_p=0.0), lambda: sq325.sample(x, u, top_p=1.5),
           lambda: sq325.sample(x, u, min_p=-0.1), lambda: sq325.sample(x, u, min_p=1.1),
           lambda: sq325.sample(x, u, temperature=u[:1]), lambda: sq325.sample(x, u, top_k=u),
           lambda: sq325.sample(torch.zeros((), device='cuda'), u),
           lambda: sq325.top_logits(x, 0), lambda: sq325.top_logits(x, 11), lambda: sq325.top_logits(x, 2.0),
           lambda: sq325.top_logits(torch.zeros((1, 2000), device='cuda'), 1025), lambda: sq325.top_logits(x.int(), 1),
           lambda: sq325.distillation_loss(x, v, i.long()), lambda: sq325.distillation_loss(x, v[:1], i[:1]),
           lambda: sq325.distillation_loss(x, v, i[:, :2]), lambda: sq325.distillation_loss(x, v.double(), i),
           lambda: sq325.distillation_loss(x, v, i, temperature=0.0),
           lambda: sq325.distillation_loss(x, v, i, temperature=float('nan')),
           lambda: sq325.distillation_loss(x, v.clone().requires_grad_(True), i),
           lambda: sq325.distillation_loss(x, v[:, :0], i[:, :0]), lambda: sq325.distillation_loss(x, v.cpu(), i),
           lambda: sq325.distillation_loss_grad(x, v, i, weight=u[:1]),
           lambda: sq325.distillation_loss_grad(x, v, i, weight=u.double())]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    # the context works on
    assert sq325.sample(x, u).tolist() == [0, 0]


# ------------------------------------------------------------------ rows that are hard in other ways
def hard_rows(vocab, dtype):
    """Rows of few values, in order, almost flat, and with all that counts in one place."""
    g = torch.Generator(device='cuda').manual_seed(vocab)
    r = lambda: torch.rand(vocab, generator=g, device='cuda')
    line = torch.arange(vocab, device='cuda') / vocab
    rows = [torch.floor(r() * 3), torch.floor(r() * 40) / 4, line * 20, (1 - line) * 20, 1e-3 * r(), 1e-30 * r(),
            torch.where(line < 0.98, -30.0, 10 * r()), torch.where(r() < 0.999, 5.0, 6.0), -50 * r().square(),
            torch.where(line > 0.999, r(), -1e4), 300 * (r() - 0.5)]
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [1500, 20001, 256000])
def test_hard_rows_top_logits(vocab, dtype):
    import sq325
    x = hard_rows(vocab, dtype)
    xs = wide(x)
    for k in (1, 64, 1000):
        values, indices = sq325.top_logits(x, k)
        for r in range(len(xs)):
            v, i = ol.top(xs[r], k)
            assert np.array_equal(indices[r].cpu().numpy(), i), (k, r)
            assert np.array_equal(wide(values[r]), v), (k, r)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [1500, 20001, 256000])
def test_hard_rows_draws(vocab, dtype):
    x = hard_rows(vocab, dtype)
    g = torch.Generator(device='cuda').manual_seed(1)
    for s in (dict(), dict(k=200), dict(k=3000), dict(p=0.6), dict(p=0.99, t=0.5), dict(q=0.5), dict(k=1000, p=0.7, q=0.01, t=2.0),
              dict(t=50.0, p=0.5), dict(t=0.01, p=0.9)):
        check_draw(x, torch.rand(len(x), generator=g, device='cuda'), least=0.0, **s)


def test_hard_rows_draws_agree_with_whole_weights():
    """Ties decide most of these rows, so the cut's place among equal logits is exact: against the definition
    in whole weights, computed in torch."""
    import sq325
    x = hard_rows(20001, torch.float16)
    g = torch.Generator(device='cuda').manual_seed(2)
    for k, p, q in ((0, 0.3, 0.0), (0, 0.8, 0.0), (700, 1.0, 0.0), (700, 0.5, 0.0), (100, 0.9, 0.2), (0, 1.0, 0.0), (5000, 0.9, 0.0)):
        u = torch.rand(len(x), generator=g, device='cuda')
        f = x.float()
        m = f.amax(1, keepdim=True)
        c = torch.tensor(1.4426950408889634, device='cuda') / torch.tensor(1.0, device='cuda')
        y = torch.where(f == m, 1.0, torch.exp2((f - m) * c))
        w = torch.round(y * 2.0 ** 31).long()
        order = torch.sort(f, dim=1, descending=True, stable=True)[1]
        ws, ys = w.gather(1, order), y.gather(1, order)
        rank = torch.arange(x.shape[1], device='cuda')
        ws = torch.where((rank < k) | (k == 0), ws, 0)
        before = ws.cumsum(1) - ws
        keep = (before.double() < float(np.float32(p)) * ws.sum(1, keepdim=True).double()) & (ys >= np.float32(q)) | (rank == 0)
        run = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0)).cumsum(1)
        target = (u.double()[:, None] * run[:, -1:].double()).long()
        want = (run <= target).sum(1)
        assert torch.equal(sq325.sample(x, u, top_k=k, top_p=p, min_p=q), want), (k, p, q)


def test_rows_past_32_bit_offsets():
    """Rows that begin more than 2^32 bytes and 2^31 elements into their buffer."""
    import sq325
    rows, vocab = 9000, 262144
    x = torch.zeros((rows, vocab), device='cuda', dtype=torch.float16)
    last, g = make(3, vocab, torch.float16, seed=12)
    x[-3:] = last
    u = torch.rand(3, generator=g, device='cuda')
    wide_u = torch.cat([torch.zeros(rows - 3, device='cuda'), u])
    for s in (dict(top_p=0.9), dict(top_k=50)):
        assert torch.equal(sq325.sample(x, wide_u, **s)[-3:], sq325.sample(last, u, **s))
    values, indices = sq325.top_logits(x, 5)
    v, i = sq325.top_logits(last, 5)
    assert torch.equal(values[-3:], v) and torch.equal(indices[-3:], i) and indices[0].tolist() == [0, 1, 2, 3, 4]
    loss, grad = sq325.distillation_loss_grad(x, values, indices)
    l, d = sq325.distillation_loss_grad(last, v, i)
    assert torch.allclose(loss[-3:], l, rtol=1e-5) and torch.allclose(grad[-3:].float(), d.float(), atol=1e-5)
    del grad
    y = x.requires_grad_(True)
    again = sq325.distillation_loss(y, values, indices)
    back, = torch.autograd.grad(again.sum(), y)
    assert torch.allclose(again.detach()[-3:], l, rtol=1e-5) and torch.allclose(back[-3:].float(), d.float(), atol=1e-5)


@pytest.mark.parametrize('rows', [5, 700])
def test_operators_in_a_cuda_graph(rows):
    """Captured once, replayed on new contents."""
    import sq325
    x, g = make(rows, 20011, torch.bfloat16, seed=3)
    values, indices = record(g, rows, 20011, 12, torch.bfloat16)
    u = torch.rand(rows, generator=g, device='cuda')
    calls = (lambda: (sq325.sample(x, u, top_p=0.9),), lambda: (sq325.sample(x, u, top_k=40),), lambda: sq325.top_logits(x, 30),
             lambda: (sq325.distillation_loss(x, values, indices),), lambda: sq325.distillation_loss_grad(x, values, indices))
    for call in calls:
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        x.copy_(torch.randn(x.shape, generator=g, device='cuda') * 3)
        u.copy_(torch.rand(rows, generator=g, device='cuda'))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, call()):
            assert torch.equal(a, b)


def test_backward_again_and_after_a_change():
    """A retained graph gives the same gradient twice; logits changed in place are refused."""
    import sq325
    x, g = make(6, 1500, torch.float32, seed=2)
    values, indices = record(g, 6, 1500, 8, torch.float32)
    y = x.clone().requires_grad_(True)
    loss = sq325.distillation_loss(y, values, indices, temperature=1.5)
    first, = torch.autograd.grad(loss.sum(), y, retain_graph=True)
    second, = torch.autograd.grad(loss, y, torch.full((6,), 2.0, device='cuda'))
    assert torch.allclose(second, 2 * first, rtol=1e-6)
    z = x.clone().requires_grad_(True)
    w = z * 1.0
    loss = sq325.distillation_loss(w, values, indices)
    w.add_(1.0)
    with pytest.raises(RuntimeError, match='modified'):
        loss.sum().backward()
    with pytest.raises(RuntimeError):                    # the gradient itself is not differentiable
        loss = sq325.distillation_loss(y, values, indices)
        grad, = torch.autograd.grad(loss.sum(), y, create_graph=True)
        grad.sum().backward()


def test_backward_from_saved_tensors_elsewhere():
    """Hooks that offload what forward saved, or compute it again, give the same gradient: backward reads what the
    graph hands it, not forward's memory."""
    import sq325
    from torch.utils.checkpoint import checkpoint
    x, g = make(7, 1501, torch.float32, seed=3)
    values, indices = record(g, 7, 1501, 9, torch.float32)
    y = x.clone().requires_grad_(True)

    def head(t):
        return sq325.distillation_loss((t * 1.25)[:, 1:], values, indices, temperature=2.0).sum()

    indices.clamp_(max=1499)
    want, = torch.autograd.grad(head(y), y)
    with torch.autograd.graph.save_on_cpu():
        loss = head(y)
    full = torch.full((1 << 20,), 3.0, device='cuda')    # takes up what forward released
    offloaded, = torch.autograd.grad(loss, y)
    loss = checkpoint(head, y, use_reentrant=False)
    full = torch.full((1 << 20,), 3.0, device='cuda')
    again, = torch.autograd.grad(loss, y)
    assert torch.equal(offloaded, want) and torch.equal(again, want)


def whole_weight_draw(x, u, t, p):
    """The draw by top-p by the definition in whole weights (no rounding is left open: tokens are equal)."""
    f = x.float()
    m = f.amax(1, keepdim=True)
    c = torch.tensor(1.4426950408889634, device='cuda') / torch.tensor(t, device='cuda')
    w = torch.round(torch.exp2((f - m) * c) * 2.0 ** 31).long()
    order = torch.sort(f + 0.0, dim=1, descending=True, stable=True)[1]
    ws = w.gather(1, order)
    before = ws.cumsum(1) - ws
    keep = before.double() < float(np.float32(p)) * ws.sum(1, keepdim=True).double()
    run = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0)).cumsum(1)
    target = (u.double()[:, None] * run[:, -1:].double()).long()
    return (run <= target).sum(1)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [701, 60001])
def test_draw_cut_in_any_range(vocab, dtype):
    """Top-p whose cut falls on positive, negative and tiny logits, on both sides of 0 at once, among few values that
    many tokens share, on signed zeros, and among tokens that are all alike."""
    import sq325
    g = torch.Generator(device='cuda').manual_seed(vocab)
    flat = torch.randn((6, vocab), generator=g, device='cuda')
    u = torch.rand(6, generator=g, device='cuda')
    zeros = torch.where(flat > 0.4, 0.0, torch.where(flat > -0.4, -0.0, -0.5))
    rows = [(flat * 3 + 40, 1.0), (flat * 3 - 40, 1.0), (flat * 0.25 - 0.125, 0.05), (flat * 1e-6, 1e-6),
            (flat.abs() * -1e-6, 3e-7), (flat * 0.01, 0.002), (torch.round(flat * 2) - 1, 1.0), (torch.round(flat) * 2 + 9, 2.0),
            (zeros, 1.0), (flat.abs() * 100, 50.0)]
    rows += [(torch.full_like(flat, v), 1.0) for v in (3.0, -3.0, 0.0, -0.0)]
    for number, (x, t) in enumerate(rows):
        x = x.to(dtype)
        for p in (0.05, 0.25, 0.5, 0.9):
            assert torch.equal(sq325.sample(x, u, temperature=t, top_p=p), whole_weight_draw(x, u, t, p)), (number, p)
