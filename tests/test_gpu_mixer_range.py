"""The scan over the range of bf16.  Bounds are those of test_gpu_mixer."""
import pytest
import torch

import _mixer64 as ref
from test_gpu_mixer import check_scan, near, scan_inputs, sq, u  # noqa: F401

pytestmark = pytest.mark.gpu
NAMES = ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias')


def run(sq, a, dy, dlast=None):  # noqa: F811
    names = [k for k in (*NAMES, 'state') if a.get(k) is not None]
    leaves = {k: a[k].detach().requires_grad_() for k in names}
    y, last = sq.selective_scan(*(leaves.get(k) for k in NAMES), leaves.get('state'), None, True)
    up = [(y, dy)] + ([] if dlast is None else [(last, dlast)])
    grads = torch.autograd.grad([p for p, _ in up], list(leaves.values()), [q for _, q in up])
    values, sums = ref.scan_with_grads(*(a.get(k) for k in NAMES), a.get('state'), None, dy, dlast)
    return names, dict(y=y, last=last, **{'d' + k: g for k, g in zip(names, grads)}), values, sums


# of x, B, C, dy and the state; every product below stays within fp32 and bf16
WIDE = [dict(x=1e30, B=1e-3, dy=1e-10), dict(x=1e-6, dy=1e28), dict(B=1e35, C=1e-10, x=1e-8, dy=1e-8), dict(state=1e29, dy=1e-10), dict(C=2e37, B=1e-9, x=1e-3, dy=1e-15),
        dict(x=1e37, B=1e-6, C=1e-6, dy=1e-12),
        dict(x=1e-25), dict(dy=1e-28), dict(x=1e-20, state=1e-20, dy=1e-12), dict(B=1e-20, C=1e-10, x=1e15)]


@pytest.mark.parametrize('scales', WIDE, ids=str)
def test_large_and_small_bf16_values(sq, scales):  # noqa: F811
    a = scan_inputs(1, 300, 2, 1, 64, torch.float32, seed=31, carried=True)
    for k in ('x', 'B', 'C'):
        a[k] = (a[k].clamp(-3, 3) * scales.get(k, 1.0)).bfloat16()
    a['dt'] = a['dt'].bfloat16()
    a['state'] = a['state'] * scales.get('state', scales.get('x', 1.0) * scales.get('B', 1.0))
    dy = (torch.randn(1, 300, 2, 64, device='cuda') * scales.get('dy', 1.0)).bfloat16()
    names, got, values, sums = run(sq, a, dy)
    assert all(v.abs().max() < 3e38 for v in values.values())
    check_scan(a, got, names, values, sums, torch.bfloat16)


@pytest.mark.parametrize('scale', [1e-25, 1e25, 1e33])
def test_large_and_small_bf16_values_behind_a_convolution(sq, scale):  # noqa: F811
    """silu(z) z of large z is z or nothing: the scan of the convolution's fp32 output, x, B and C once each in 11 bits."""
    heads, groups, width = 2, 1, 128 + 256
    gen = torch.Generator(device='cuda').manual_seed(8)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    xbc = rnd(1, 200, width)
    xbc[..., :128] *= scale
    xbc, dt = xbc.bfloat16(), (0.5 * rnd(1, 200, heads) - 3).bfloat16()
    A, w, D = -(0.2 + 3 * rnd(heads).abs()), (0.5 * rnd(width, 4)).bfloat16(), rnd(heads).bfloat16()
    y, _, last = sq.conv_scan(xbc, dt, A, w, None, D, heads=heads, groups=groups, return_final_state=True)

    def definition(f):
        z, _ = ref.conv(f(xbc.double()), f(w.double()))
        x, B, C = z.split([128, 128, 128], -1)
        return ref.scan(x.unflatten(2, (heads, 64)), dt.double(), A.double(), B.unflatten(2, (1, 128)), C.unflatten(2, (1, 128)), f(D.double()))
    (vy, vl), (sy, sl) = definition(lambda t: t), definition(torch.abs)
    near(y, vy, u(torch.bfloat16) * vy.abs() + (3 * 2 ** -11 + 2 ** -10) * sy, 'y')
    near(last, vl, 3 * 2 ** -11 * sl, 'last')
