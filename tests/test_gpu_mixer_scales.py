"""The scan of heads that are zero beside heads with small gradients, and of steps among the smallest numbers.  Bounds are those of
test_gpu_mixer."""
import pytest
import torch

import _mixer64 as ref
from test_gpu_mixer import HALF, check_scan, near, scan_inputs, sq, u  # noqa: F401

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


@pytest.mark.parametrize('dtype', HALF)
@pytest.mark.parametrize('dim', [64, 72])
def test_steps_among_the_smallest_numbers(sq, dtype, dim):  # noqa: F811
    """softplus(-87) to softplus(-104) are fp32's subnormal numbers; from there on steps are zero."""
    a = scan_inputs(1, 260, 2, 1, dim, dtype, seed=5)
    a['dt_bias'] = None
    a['dt'][0, 40:75, 0] = -torch.arange(86.0, 121.0).to('cuda', dtype)
    a['dt'][0, 130:165, 1] = -torch.arange(86.0, 121.0).to('cuda', dtype)
    a['dt'][0, 200:220, 0] = torch.finfo(dtype).min
    dy = torch.randn(1, 260, 2, dim, device='cuda').to(dtype)
    names, got, values, sums = run(sq, a, dy)
    check_scan(a, got, names, values, sums, dtype)


@pytest.mark.parametrize('dtype,size', [(torch.float16, 1e-4), (torch.bfloat16, 1e-5), (torch.bfloat16, 1e-12)])
@pytest.mark.parametrize('dead', ['dy', 'x', 'both'])
def test_a_dead_head_takes_no_bits_from_its_group(sq, dtype, size, dead):  # noqa: F811
    """A head whose tokens or gradients are zero adds nothing to dB and dC, beside heads of the same CTA whose gradients are
    small."""
    batch, length, heads, groups = 25, 300, 40, 8
    a = scan_inputs(batch, length, heads, groups, 64, dtype, seed=14)
    dy = (torch.randn(batch, length, heads, 64, device='cuda') * size).to(dtype)
    a['x'] = a['x'].clone()
    if dead in ('dy', 'both'):
        dy[:, :, 1::5] = 0
    if dead in ('x', 'both'):
        a['x'][:, :, 2::5] = 0
    leaves = [a[k].detach().requires_grad_() for k in NAMES]
    dB, dC = torch.autograd.grad(sq.selective_scan(*leaves), leaves[3:5], dy)
    for g in (0, 7):
        h = slice(5 * g, 5 * g + 5)
        cut = lambda t: t[:2, :, g:g + 1]
        values, sums = ref.scan_with_grads(a['x'][:2, :, h], a['dt'][:2, :, h], a['A'][h], cut(a['B']), cut(a['C']), a['D'][h], a['dt_bias'][h], None, None, dy[:2, :, h])
        for k, got in (('dB', dB), ('dC', dC)):
            near(cut(got), values[k], u(dtype) * values[k].abs() + 2 ** -10 * sums[k], k)


@pytest.mark.parametrize('dtype', HALF)
def test_nothing_but_zeros(sq, dtype):  # noqa: F811
    a = scan_inputs(1, 260, 2, 1, 64, dtype, seed=2)
    dy = torch.zeros(1, 260, 2, 64, device='cuda', dtype=dtype)
    _, got, _, _ = run(sq, a, dy)
    assert not any(got['d' + k].any() for k in NAMES)
    a['x'] = torch.zeros_like(a['x'])
    dy = torch.randn(1, 260, 2, 64, device='cuda').to(dtype)
    names, got, values, sums = run(sq, a, dy)
    check_scan(a, got, names, values, sums, dtype)
