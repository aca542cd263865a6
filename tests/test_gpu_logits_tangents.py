"""Forward-mode: the distillation loss has no such derivative and says so."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_gpu_mixer import sq  # noqa: F401

pytestmark = pytest.mark.gpu


def test_a_tangent_of_logits_is_not_dropped(sq):  # noqa: F811
    logits = torch.randn(3, 40, device='cuda')
    values, indices = sq.top_logits(logits, 8)
    for call in (sq.distillation_loss, sq.distillation_loss_grad):
        with fwd.dual_level():
            with pytest.raises(NotImplementedError, match='forward'):
                call(fwd.make_dual(logits, logits), values, indices)
            with pytest.raises(NotImplementedError, match='forward'):
                call(logits, fwd.make_dual(values, values), indices)
            call(logits, values, indices)
