"""Forward-mode: the mixer's operators have no such derivative and say so."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_gpu_mixer import sq  # noqa: F401

pytestmark = pytest.mark.gpu


def test_a_tangent_is_not_dropped(sq):  # noqa: F811
    """There is no forward-mode derivative: a call with a tangent raises."""
    x = torch.randn(1, 5, 384, device='cuda').half()
    w, dt, A = torch.randn(384, 4, device='cuda').half(), torch.randn(1, 5, 2, device='cuda').half(), -torch.ones(2, device='cuda')
    parts = lambda t: [p.unflatten(-1, s) for p, s in zip(t.split([128, 128, 128], -1), ((2, 64), (1, 128), (1, 128)))]

    def scan(t):
        xx, B, C = parts(t)
        return sq.selective_scan(xx, dt, A, B, C)
    calls = [lambda t: sq.causal_conv(t, w), scan, lambda t: sq.conv_scan(t, dt, A, w, heads=2, groups=1),
             lambda t: sq.causal_conv_step(t[:, 0], torch.zeros(1, 3, 384, device='cuda').half(), w),
             lambda t: sq.conv_scan_step(t[:, 0], dt[:, 0], A, w, heads=2, groups=1, conv_state=torch.zeros(1, 3, 384, device='cuda').half(),
                                         state=torch.zeros(1, 2, 64, 128, device='cuda')),
             lambda t: sq.selective_step(*(lambda p: (p[0], dt[:, 0], A, p[1], p[2]))(parts(t[:, 0])), torch.zeros(1, 2, 64, 128, device='cuda'))]
    for call in calls:
        with fwd.dual_level():
            with pytest.raises(NotImplementedError, match='forward'):
                call(fwd.make_dual(x, torch.ones_like(x)))
            call(x)                                # without a tangent, also inside the level
            call(x.detach())
        call(x)
    y = torch.zeros(1, 2, 64, 128, device='cuda')
    with fwd.dual_level(), pytest.raises(NotImplementedError, match='forward'):
        sq.selective_scan(*(lambda p: (p[0], dt, A, p[1], p[2]))(parts(x)), initial_state=fwd.make_dual(y, y))
