"""conv_scan: the gradient of the convolution's output, which no caller sees, has fp32's range and bits.

Tolerance of norms: test_gpu_mixer_fused derives 4 u for eight roundings.  Gradients of fp32 weights have no rounding of their own and none
of the gradient between the two; what is left are x, B and C in fp16, the pairs' weights in the type (bf16 beside x and dy are scaled
fp16, too) and the operands of dB and dC in fp16: at most seven of 2^-11, whatever the input's type."""
import pytest
import torch

from test_gpu_mixer import HALF, sq, u  # noqa: F401
from test_gpu_mixer_fused import check, close, definition, inputs

pytestmark = pytest.mark.gpu
HEADS, GROUPS, DIM = 32, 1, 64
INNER = HEADS * DIM


def run(sq, a, dy, keep=None):  # noqa: F811
    names = [k for k, v in a.items() if v is not None]
    leaves = {k: a[k].detach().requires_grad_() for k in names}
    y = sq.conv_scan(leaves['xbc'], leaves['dt'], leaves['A'], leaves['w'], leaves['b'], leaves['D'], leaves['bias'], heads=HEADS, groups=GROUPS, keep=keep)
    grads = dict(zip(names, torch.autograd.grad(y, list(leaves.values()), dy)))
    return names, grads


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('size', [2.0 ** -12, 1.0])
def test_gradients_of_32_bit_weights(sq, dtype, size):  # noqa: F811
    a, dy, _, _ = inputs(2, 300, HEADS, GROUPS, DIM, 4, dtype, param=torch.float32, seed=11)
    dy = (dy.float() * size).to(dtype)
    names, grads = run(sq, a, dy)
    _, _, want = definition(a, HEADS, GROUPS, DIM, None, dy, None, None, names)
    check({k: grads[k] for k in ('w', 'b')}, want, HEADS, GROUPS, DIM, 4 * 2 ** -11)
    check({k: grads[k] for k in ('A', 'D', 'bias')}, want, HEADS, GROUPS, DIM, 4 * 2 ** -11)
    check({k: grads[k] for k in ('xbc', 'dt')}, want, HEADS, GROUPS, DIM, 4 * u(dtype))


def test_fp16_gradients_that_overflow_between_the_two(sq):  # noqa: F811
    """B's and C's gradients of more than 65,504, sums over 32 heads, meet taps of 2^-10 on their way to dx: finite there, and in fp32 weights'."""
    a, dy, _, _ = inputs(1, 200, HEADS, GROUPS, DIM, 4, torch.float16, param=torch.float32, seed=12)
    a['w'][INNER:] *= 2.0 ** -8
    a['w'][:INNER] *= 8
    a['dt'] += 2
    dy = dy * 256
    names, grads = run(sq, a, dy)
    _, _, want = definition(a, HEADS, GROUPS, DIM, None, dy, None, None, names)
    part = slice(INNER, None)
    # ddt has a type of its own and its own range; the others are what the gradient between the two is made into
    assert want['xbc'][..., part].abs().max() < 6e4 and float(want['b'][part].abs().max()) > 65504
    close(grads['xbc'][..., part], want['xbc'][..., part], 4 * 2 ** -11, 'dxbc of B and C')
    close(grads['w'][part], want['w'][part], 4 * 2 ** -11, 'dw of B and C')
    close(grads['b'][part], want['b'][part], 4 * 2 ** -11, 'db of B and C')


def test_fp16_gradients_that_vanish_between_the_two(sq):  # noqa: F811
    """Gradients of 2^-22, a few of fp16's smallest steps: what comes in is exact, and taps of 2^7 bring dx back."""
    a, dy, _, _ = inputs(1, 200, HEADS, GROUPS, DIM, 4, torch.float16, param=torch.float32, seed=13)
    a['w'] *= 2.0 ** 7
    a['w'][INNER:] *= 2.0 ** -5
    a['xbc'] *= 2.0 ** -6
    dy = (dy.float() * 2.0 ** -14).half()
    names, grads = run(sq, a, dy)
    _, _, want = definition(a, HEADS, GROUPS, DIM, None, dy, None, None, names)
    for k in ('w', 'b'):
        for part in (slice(0, INNER), slice(INNER, None)):
            close(grads[k][part], want[k][part], 4 * 2 ** -11, k)
