"""The distillation loss and its gradient where a bound taken from the whole row says nothing (rows masked by
the type's lowest value), and on the stepping kernel's unaligned path, against 64 bits.

Bounds.  With t an exponent of 2 and e = (max |t| + (vocab + k) / 512 + 40) 2^-23 (a difference, a product, the
hardware's power, a sum), over the logits that carry weight (within 150 of the largest in units of T; the others'
powers are 0 in fp32): p and q are off by e relative, the loss by T^2 e (1 + 3 max |t|), the gradient by T w e (p + q) and its
own rounding."""
import pytest
import torch

from _logits64 import distill64
from test_gpu_logits import LEAST, TYPES, UNIT, make, record

pytestmark = pytest.mark.gpu


def check(x, values, indices, T, weight, loss, grad=None, block=100):
    for r in range(0, len(x), block):
        part = slice(r, r + block)
        want, p, q, rq, _ = distill64(x[part], values[part], indices[part], T)
        s = x[part].double()
        far = (s.amax(1, keepdim=True) - s) / T * 1.45
        at = indices[part].long().clamp(min=0)
        far = torch.maximum(torch.where(far <= 150, far, 0.0).amax(1), torch.where(rq > 0, far.gather(1, at), 0.0).amax(1))
        e = (far + (x.shape[1] + values.shape[1]) / 512 + 40) * 2.0 ** -23
        most = T * T * e * (1 + 3 * far)
        assert float(e.max()) < 1e-4 and float(most.max()) < 0.03 * T * T      # neither bound is empty
        assert ((loss[part].double() - want).abs() <= most).all()
        if grad is not None:
            w = weight[part].double()[:, None]
            g = w * T * (p - q)
            bound = T * w.abs() * e[:, None] * (p + q) + UNIT[x.dtype] * g.abs() * 1.01 + LEAST[x.dtype]
            assert ((grad[part].double() - g).abs() <= bound).all()


def both_ways(x, values, indices, T, weight):
    import sq325
    check(x, values, indices, T, weight, *sq325.distillation_loss_grad(x, values, indices, temperature=T, weight=weight))
    y = x.detach().requires_grad_(True)
    loss = sq325.distillation_loss(y, values, indices, temperature=T)
    check(x, values, indices, T, weight, loss.detach(), torch.autograd.grad(loss, y, weight)[0])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab,k', [(3001, 40), (70001, 64), (256000, 300)])
def test_rows_masked_by_the_lowest_value(vocab, k, dtype):
    """A third or all but the record's neighbourhood masked by the type's lowest value, -inf beside it."""
    x, g = make(6, vocab, dtype, seed=vocab, pad=3)
    values, indices = record(g, 6, vocab, k, dtype, cut=0.1)
    indices[:, 0] = indices[:, 0].clamp(min=0)                     # every row has a record
    low, taken = torch.finfo(dtype).min, torch.zeros((6, vocab), device='cuda', dtype=torch.bool)
    taken.scatter_(1, indices.long().clamp(min=0), True)
    column = torch.arange(vocab, device='cuda')
    masks = [column % 3 == 0, column % 64 != 1, column < vocab // 2, column % 2 == 1, column > 900, column == 5]
    for r, mask in enumerate(masks):
        x[r].masked_fill_(mask & ~taken[r], low)
    x[3].masked_fill_((column % 4 == 0) & ~taken[3], float('-inf'))
    for T in (0.7, 1.0, 3.0):
        both_ways(x, values, indices, T, torch.linspace(-1, 2, 6, device='cuda'))


@pytest.mark.parametrize('dtype,rows,vocab,pad,offset', [(torch.float16, 700, 70001, 3, 1), (torch.bfloat16, 700, 70001, 1, 5),
                                                         (torch.float32, 500, 70001, 2, 3), (torch.float32, 170, 262143, 2, 1),
                                                         (torch.float16, 170, 256000, 4, 0)])
def test_stepping_clusters_with_unaligned_gradients(dtype, rows, vocab, pad, offset):
    """More clusters of several CTAs than run at once, each refilling its part of the row while the gradient, whose
    rows lie otherwise in their 16 bytes than the logits' rows, leaves through shared memory."""
    x, g = make(rows, vocab, dtype, seed=rows, pad=pad, offset=offset, spread=2.0)
    values, indices = record(g, rows, vocab, 24, dtype)
    indices[:, 0] = indices[:, 0].clamp(min=0)
    both_ways(x, values, indices, 1.5, torch.rand(rows, generator=g, device='cuda') * 4 - 1)
