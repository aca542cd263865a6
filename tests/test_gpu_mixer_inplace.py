"""The one-token calls write states in place, and autograd is told."""
import pytest
import torch

from test_gpu_mixer import sq  # noqa: F401

pytestmark = pytest.mark.gpu
HEADS, GROUPS, DIM = 4, 2, 64
WIDTH = HEADS * DIM + 256 * GROUPS


@pytest.fixture
def a():
    gen = torch.Generator(device='cuda').manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=gen, device='cuda')
    return dict(xbc=rnd(2, 9, WIDTH).half(), dt=(rnd(2, 9, HEADS) - 3).half(), A=-rnd(HEADS).abs(), w=rnd(WIDTH, 4).half(), D=rnd(HEADS).half(),
                conv_state=rnd(2, 3, WIDTH).half(), state=rnd(2, HEADS, DIM, 128))


def parts(z):
    x, B, C = z.split([HEADS * DIM, GROUPS * 128, GROUPS * 128], -1)
    return x.unflatten(-1, (HEADS, DIM)), B.unflatten(-1, (GROUPS, 128)), C.unflatten(-1, (GROUPS, 128))


def step(sq, a, which):  # noqa: F811
    token, dt = a['xbc'][:, 0].detach(), a['dt'][:, 0]
    if which == 'conv':
        return sq.causal_conv_step(token, a['conv_state'], a['w'])
    if which == 'scan':
        x, B, C = parts(token)
        return sq.selective_step(x, dt, a['A'], B, C, a['state'], a['D'])
    return sq.conv_scan_step(token, dt, a['A'], a['w'], None, a['D'], heads=HEADS, groups=GROUPS, conv_state=a['conv_state'], state=a['state'])


@pytest.mark.parametrize('which,changed', [('conv', 'conv_state'), ('scan', 'state'), ('both', 'conv_state'), ('both', 'state')])
def test_a_gradient_through_a_state_that_has_moved_on_is_refused(sq, a, which, changed):  # noqa: F811
    leaf = a['xbc'].requires_grad_()
    x, B, C = parts(leaf)
    calls = {'conv_state': [lambda: sq.causal_conv(leaf, a['w'], initial_state=a['conv_state']),
                            lambda: sq.conv_scan(leaf, a['dt'], a['A'], a['w'], heads=HEADS, groups=GROUPS, conv_state=a['conv_state'])],
             'state': [lambda: sq.selective_scan(x, a['dt'], a['A'], B, C, initial_state=a['state']),
                       lambda: sq.conv_scan(leaf, a['dt'], a['A'], a['w'], heads=HEADS, groups=GROUPS, initial_state=a['state'])]}[changed]
    for call in calls:
        y = call()
        step(sq, a, which)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            y.sum().backward()
        call().sum().backward()                   # the state as it is now


@pytest.mark.parametrize('which,changed', [('conv', ['conv_state']), ('scan', ['state']), ('both', ['conv_state', 'state'])])
def test_versions_and_inference_tensors(sq, a, which, changed):  # noqa: F811
    before = {k: a[k]._version for k in ('conv_state', 'state', 'xbc', 'w')}
    step(sq, a, which)
    assert {k: a[k]._version - v for k, v in before.items()} == {k: int(k in changed) for k in before}
    with torch.inference_mode():                  # tensors without versions, in and out of the mode
        held = {k: a[k].clone() for k in ('conv_state', 'state')}
        want = step(sq, dict(a, **held), which)
    assert torch.equal(step(sq, dict(a, **held), which).isfinite(), want.isfinite())
