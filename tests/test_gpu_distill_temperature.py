"""The distillation loss over the whole range of temperatures that is accepted, against 64 bits.

Bounds.  The powers carry e = (150 + (vocab + k) / 512 + 40) 2^-23 relative (their exponents are at most 150 where they
are not 0 in fp32).  With D the largest |gap| (teacher's distance to its largest logit less the student's) of an entry that
has weight and B = |log S - log Q|, the loss T sum q (gap + T B) is off by T (2 e D + 2 T e (1 + B)) and, where it is
subnormal, by a few units of 2^-149; the gradient by T e (p + q) and T 2^-120 for powers that are 0."""
import numpy as np
import pytest
import torch

from _logits64 import distill64
from test_gpu_logits import make, record

pytestmark = pytest.mark.gpu

TEMPERATURES = [1e-42, 1e-38, 1e-30, 1e-21, 1e-12, 1e-3, 1e4, 1e12, 1e18, 1e20, 1e30, 3e38]
MOST = torch.finfo(torch.float32).max


@pytest.mark.parametrize('T', TEMPERATURES)
@pytest.mark.parametrize('vocab,k', [(403, 30), (70001, 64)])
def test_loss_and_gradient_at_any_temperature(vocab, k, T):
    import sq325
    x, g = make(5, vocab, torch.float32, seed=vocab)
    values, indices = record(g, 5, vocab, k, torch.float32)
    indices[:, 0] = indices[:, 0].clamp(min=0)
    T32 = float(np.float32(T))
    want, p, q, rq, gap = distill64(x, values, indices, T32)
    e = (150 + (vocab + k) / 512 + 40) * 2.0 ** -23
    D = torch.where(rq > 1e-30, gap.abs(), 0.0).amax(1)
    B = np.log(vocab) + 1
    most = T32 * (2 * e * D + 2 * T32 * e * (1 + B)) + 2.0 ** -146
    y = x.detach().requires_grad_(True)
    again = sq325.distillation_loss(y, values, indices, temperature=T)
    back = torch.autograd.grad(again.sum(), y)[0]
    for loss, grad in (sq325.distillation_loss_grad(x, values, indices, temperature=T), (again.detach(), back)):
        large = want > 2 * MOST
        assert (loss[large] == float('inf')).all()
        off = (loss.double() - want).abs()
        assert (off <= most)[~large].all(), (off, most)
        bound = T32 * (e * (p + q) + 2.0 ** -120) + 2.0 ** -140
        assert ((grad.double() - T32 * (p - q)).abs() <= bound).all()


@pytest.mark.parametrize('T', TEMPERATURES)
def test_one_token_has_nothing_to_learn(T):
    """A vocabulary of one token: loss and gradient are 0 at every temperature."""
    import sq325
    x, values = torch.full((3, 1), 2.5, device='cuda'), torch.full((3, 1), -7.0, device='cuda')
    loss, grad = sq325.distillation_loss_grad(x, values, torch.zeros((3, 1), dtype=torch.int32, device='cuda'), temperature=T)
    assert loss.tolist() == [0.0] * 3 and not grad.any()
