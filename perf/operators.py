"""Cases of the operators on rows of logits: drawing a token (`sq325.sample`), the largest
logits of a row (`sq325.top_logits`), and the distillation loss from a teacher's largest
logits (`sq325.distillation_loss` with its backward, `sq325.distillation_loss_grad`).

`own = False` computes the plain form in elementary torch operations, `own = True` makes
the library's calls.  A case is a dict of plain values:

  op       'sample' | 'top' | 'loss' | 'train' | 'grad'
  rows, vocab, dtype ('float16' | 'bfloat16' | 'float32')
  pad      columns of the logits' buffer beyond `vocab` (a row stride that is not the width)
  banned   share of the vocabulary masked to -inf in every row
  temperature, top_k, top_p, min_p (sample; 'mixed': each row has settings of its own)
  k        entries kept of each row (top), entries of the teacher's record (loss, train, grad)
  unused   share of rows whose record is cut short, one in eight of them to nothing
"""
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parent.parent
LOG2E = 1.4426950408889634
GRID = float(2 ** 31)            # weights of a draw are whole multiples of 2^-31 of the largest


def _package():
    path = str(ROOT / 'mamb2_8b_fp4_recall_sq3.25_b200')
    if path not in sys.path:
        sys.path.insert(0, path)
    import sq325
    return sq325


def _sample(name, rows, vocab, dtype, temperature, top_k, top_p, min_p, pad=0, banned=0.0, mixed=False):
    return dict(name=name, op='sample', rows=rows, vocab=vocab, dtype=dtype, temperature=temperature, top_k=top_k,
                top_p=top_p, min_p=min_p, pad=pad, banned=banned, mixed=mixed)


def _record(name, op, rows, vocab, dtype, k, temperature=1.0, pad=0, banned=0.0, unused=0.0):
    return dict(name=name, op=op, rows=rows, vocab=vocab, dtype=dtype, k=k, temperature=temperature, pad=pad,
                banned=banned, unused=unused)


def listed():
    return [
        # one request answering with the usual settings, the model's vocabulary: latency
        _sample('sample_1', 1, 256000, 'float16', 0.8, 50, 0.9, 0.0),
        # a served batch of 32 requests, each with settings of its own
        _sample('sample_32_mixed', 32, 256000, 'float16', 1.0, 0, 1.0, 0.0, banned=0.01, mixed=True),
        # a smaller odd vocabulary in 32 bits, min-p alone
        _sample('sample_96_minp_odd', 96, 32003, 'float32', 1.2, 0, 1.0, 0.05, pad=5),
        # many continuations at once (data for a student), top-p alone
        _sample('sample_512_topp', 512, 256000, 'bfloat16', 1.0, 0, 0.95, 0.0),
        # alternatives beside each answered token of a batch of 32
        _record('top_32', 'top', 32, 256000, 'float16', 20),
        # 32-bit logits of an odd vocabulary, rows of a wider buffer
        _record('top_333_odd', 'top', 333, 50001, 'float32', 128, pad=3, banned=0.02),
        # the teacher's record of a window of 2,048 tokens
        _record('top_2048', 'top', 2048, 256000, 'float16', 64),
        # held-out loss, no gradient
        _record('loss_512', 'loss', 512, 256000, 'float16', 64, banned=0.01, unused=0.1),
        # a small step through autograd, odd sizes
        _record('train_33_odd', 'train', 33, 5003, 'float32', 17, temperature=2.0, pad=1, unused=0.25),
        # a step of 1,024 tokens through autograd
        _record('train_1024', 'train', 1024, 256000, 'bfloat16', 64, temperature=2.0),
        # loss and gradient in one call: an odd vocabulary, and a window of 2,048 tokens
        _record('grad_127_odd', 'grad', 127, 32003, 'float16', 33, pad=2, banned=0.05, unused=0.25),
        _record('grad_2048', 'grad', 2048, 256000, 'bfloat16', 64, unused=0.05),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(('sample', 'sample', 'top', 'loss', 'train', 'grad'))
    vocab = rng.choice((256000, _log_uniform(rng, 1000, 262144), _log_uniform(rng, 1000, 262144)))
    most = {'sample': 512, 'top': 2048, 'loss': 512, 'train': 1024, 'grad': 2048}[op]
    rows = _log_uniform(rng, 1, max(1, min(most, most * 128000 // vocab)))
    dtype = rng.choice(('float16', 'bfloat16', 'float32'))
    pad = rng.choice((0, 0, 1, 3, 8))
    banned = rng.choice((0.0, 0.01, 0.3))
    if op == 'sample':
        return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, pad=pad, banned=banned,
                    temperature=round(rng.uniform(0.5, 1.5), 2), top_k=rng.choice((0, 0, 1, _log_uniform(rng, 2, 2000))),
                    top_p=rng.choice((1.0, round(rng.uniform(0.3, 0.99), 3))),
                    min_p=rng.choice((0.0, 0.0, round(rng.uniform(0.001, 0.3), 3))), mixed=rng.random() < 0.3)
    return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, pad=pad, banned=banned, k=_log_uniform(rng, 1, 512),
                temperature=1.0 if op == 'top' else round(rng.uniform(0.7, 4.0), 2),
                unused=0.0 if op == 'top' else rng.choice((0.0, 0.25)))


def _spread(rows, few, vocab, gen):
    """`few` distinct tokens of each row, at even distances from a drawn one."""
    start = (torch.rand((rows, 1), generator=gen, device='cuda') * vocab).long()
    return (start + torch.arange(few, device='cuda') * (vocab // few)) % vocab


def _logits(case, gen, spread=2.0):
    """A bulk of about normal logits and some forty that stand out, as a language model's rows have."""
    rows, vocab = case['rows'], case['vocab']
    dtype = getattr(torch, case['dtype'])
    buf = torch.empty((rows, vocab + case['pad']), device='cuda', dtype=dtype)
    few = min(40, vocab)
    step = max(1, (1 << 27) // (vocab + case['pad']))
    for r in range(0, rows, step):                       # in blocks: the 32-bit draft stays small
        n = min(step, rows - r)
        x = torch.randn((n, vocab + case['pad']), generator=gen, device='cuda') * spread
        at = _spread(n, few, vocab, gen)
        x.scatter_(1, at, 4.0 + 10.0 * torch.rand((n, few), generator=gen, device='cuda'))
        if case['banned']:
            out = torch.rand(vocab, generator=gen, device='cuda') < case['banned']
            x[:, :vocab].masked_fill_(out, float('-inf'))
        buf[r:r + n] = x.to(dtype)
    return buf[:, :vocab]


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    rows, vocab = case['rows'], case['vocab']
    s = dict(case=case, logits=_logits(case, gen))
    if case['op'] == 'sample':
        s['uniform'] = torch.rand(rows, generator=gen, device='cuda')
        if case['mixed']:
            pick = lambda values, dtype: torch.tensor(values, device='cuda', dtype=dtype)[
                torch.randint(0, len(values), (rows,), generator=gen, device='cuda')]
            s['settings'] = dict(temperature=pick([0.0, 0.6, 1.0, 1.3], torch.float32),
                                 top_k=pick([0, 0, 20, 100], torch.int32),
                                 top_p=pick([0.5, 0.9, 0.95, 1.0], torch.float32),
                                 min_p=pick([0.0, 0.0, 0.02], torch.float32))
        else:
            s['settings'] = {k: case[k] for k in ('temperature', 'top_k', 'top_p', 'min_p')}
    elif case['op'] != 'top':
        k = min(case['k'], vocab)
        # the teacher's record: distinct tokens, logits falling along the row, near the student's where they meet
        at = _spread(rows, k, vocab, gen)
        values = 12.0 - 8.0 * torch.rand((rows, k), generator=gen, device='cuda')
        s['values'] = values.sort(1, descending=True)[0].to(getattr(torch, case['dtype']))
        s['indices'] = at.int()
        if case['unused']:
            cut = torch.rand(rows, generator=gen, device='cuda') < case['unused']
            left = (torch.rand(rows, generator=gen, device='cuda') * k).long()
            left = torch.where(torch.rand(rows, generator=gen, device='cuda') < 0.125, 0, left)
            left = torch.where(cut, left, k)
            gone = torch.arange(k, device='cuda') >= left[:, None]
            s['indices'].masked_fill_(gone, -1)
            s['values'].masked_fill_(gone, float('-inf'))
        # the student's own logits stand where the teacher's do, within a few nats, and none of them is masked
        near = values + 1.5 * torch.randn((rows, k), generator=gen, device='cuda')
        s['logits'].scatter_(1, at, near.to(s['logits'].dtype))
        if case['op'] == 'train':
            s['logits'].requires_grad_(True)
            s['upstream'] = torch.full((rows,), 64.0 / rows, device='cuda')
        if case['op'] == 'grad':
            s['weight'] = 0.5 + torch.rand(rows, generator=gen, device='cuda')
    return s


def _rows(value, like, dtype):
    """A setting as a column, one value a row."""
    return (value if isinstance(value, torch.Tensor) else torch.full((like.shape[0],), value, device=like.device)).to(dtype)[:, None]


def _plain_sample(logits, uniform, temperature, top_k, top_p, min_p):
    x = logits.float()
    x = torch.where(torch.isnan(x), float('-inf'), x)
    t, k = _rows(temperature, x, torch.float32), _rows(top_k, x, torch.int64)
    p, least = _rows(top_p, x, torch.float32).double(), _rows(min_p, x, torch.float32).clamp(max=1.0)
    m = x.amax(1, keepdim=True)
    y = torch.exp2((x - m) * (torch.full_like(t, LOG2E) / t))
    y = torch.where(x == m, 1.0, torch.where(t > 0, y, 0.0))
    order = torch.sort(x, dim=1, descending=True, stable=True)[1]
    ys = y.gather(1, order)
    w = torch.round(ys * GRID).long()
    rank = torch.arange(x.shape[1], device=x.device)
    w = torch.where((rank < k) | (k <= 0), w, 0)
    before = w.cumsum(1) - w
    keep = (before.double() < p * w.sum(1, keepdim=True).double()) & (ys >= least) & (t > 0) | (rank == 0)
    prefix = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0)).cumsum(1)
    total = prefix[:, -1:]
    target = torch.minimum((uniform.double()[:, None] * total.double()).long(), total - 1)
    token = (prefix <= target).sum(1)
    return torch.where(m[:, 0] == float('-inf'), -1, token)


def _plain_top(logits, k):
    x = logits.float()
    x = torch.where(torch.isnan(x), float('-inf'), x)
    values, at = torch.sort(x, dim=1, descending=True, stable=True)
    values, at = values[:, :k], at[:, :k].int()
    return values.to(logits.dtype), torch.where(values == float('-inf'), -1, at)


def _plain_teacher(values, indices, vocab, t):
    used = (indices >= 0) & (indices < vocab) & (values > float('-inf'))
    v = torch.where(used, values.float(), float('-inf')) / t
    m = v.amax(1, keepdim=True)
    e = torch.where(used, torch.exp(v - m), 0.0)
    total = e.sum(1, keepdim=True)
    q = torch.where(total > 0, e / total, 0.0)
    logq = v - m - torch.log(total)
    return used, q, logq


def _plain_loss(logits, values, indices, t):
    z = logits.float() / t
    at = indices.long().clamp(0, z.shape[1] - 1)
    used, q, logq = _plain_teacher(values, indices, z.shape[1], t)
    m = z.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(z - m).sum(1, keepdim=True))
    logp = z.gather(1, at) - lse
    loss = t * t * torch.where(used & (q > 0), q * (logq - logp), 0.0).sum(1)
    return loss, z, lse, used, q, at


def _plain_loss_grad(logits, values, indices, t, weight):
    loss, z, lse, used, q, at = _plain_loss(logits, values, indices, t)
    g = torch.exp(z - lse).scatter_add_(1, at, torch.where(used, -q, 0.0))
    g = torch.where(used.any(1, keepdim=True), g * (t * weight[:, None]), 0.0)
    return loss, g.to(logits.dtype)


def run(state):
    case, logits = state['case'], state['logits']
    op = case['op']
    if own:
        sq = _package()
        if op == 'sample':
            return sq.sample(logits, state['uniform'], **state['settings'])
        if op == 'top':
            return sq.top_logits(logits, min(case['k'], case['vocab']))
        record = (state['values'], state['indices'])
        if op == 'loss':
            return sq.distillation_loss(logits, *record, temperature=case['temperature'])
        if op == 'train':
            loss = sq.distillation_loss(logits, *record, temperature=case['temperature'])
            return loss.detach(), torch.autograd.grad(loss, logits, state['upstream'])[0]
        return sq.distillation_loss_grad(logits, *record, temperature=case['temperature'], weight=state['weight'])
    with torch.no_grad():
        if op == 'sample':
            return _plain_sample(logits, state['uniform'], **state['settings'])
        if op == 'top':
            return _plain_top(logits, min(case['k'], case['vocab']))
        record = (state['values'], state['indices'], case['temperature'])
        if op == 'loss':
            return _plain_loss(logits, *record)[0]
        return _plain_loss_grad(logits, *record, state['upstream' if op == 'train' else 'weight'])


def work(case):
    size = 4 if case['dtype'] == 'float32' else 2
    n, rows = case['rows'] * case['vocab'], case['rows']
    if case['op'] == 'sample':       # logits, the number drawn from and the token; subtract, scale, power, sum
        return dict(bytes=n * size + rows * 12, flops=4 * n)
    k = min(case['k'], case['vocab'])
    record = rows * k * (size + 4)
    if case['op'] == 'top':          # logits in, record out; one comparison a logit
        return dict(bytes=n * size + record, flops=n)
    if case['op'] == 'loss':         # logits and record in, loss out; scale, subtract, power, sum
        return dict(bytes=n * size + record + 4 * rows, flops=4 * n)
    # logits and record in, loss and gradient out; the power again, scaled
    return dict(bytes=2 * n * size + record + 8 * rows, flops=7 * n)


def exact(case, seed):
    """The floating outputs in 64 bits, row by row from the definitions; a draw has none."""
    if case['op'] == 'sample':
        return None
    s = prepare(case, seed)
    logits, vocab, rows = s['logits'].detach(), case['vocab'], case['rows']
    if case['op'] == 'top':
        k = min(case['k'], vocab)
        out = torch.empty((rows, k), dtype=torch.float64, device='cuda')
        for r in range(rows):
            out[r] = torch.topk(logits[r].double(), k)[0]
        return out, None
    t = float(case['temperature'])
    loss = torch.zeros(rows, dtype=torch.float64, device='cuda')
    wants = case['op'] != 'loss'
    grad = torch.zeros((rows, vocab), dtype=torch.float64, device='cuda') if wants else None
    record = [(v.double(), i) for v, i in zip(s['values'].cpu(), s['indices'].cpu().long())]
    scale = s['upstream' if case['op'] == 'train' else 'weight'].double().cpu() if wants else None
    for r, (values, at) in enumerate(record):
        values, at = values[at >= 0].cuda(), at[at >= 0].cuda()
        if not len(at):
            continue
        logp = torch.log_softmax(logits[r].double() / t, 0)
        logq = torch.log_softmax(values / t, 0)
        loss[r] = t * t * (logq.exp() * (logq - logp[at])).sum()
        if wants:
            g = logp.exp()
            g.index_add_(0, at, logq.exp(), alpha=-1.0)
            grad[r] = g * (t * float(scale[r]))
    return (loss, grad) if wants else loss
