"""What causal_conv(keep='int8') keeps of its input."""
import pytest
import torch

import _mixer64 as ref
from test_gpu_mixer import HALF, sq  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [*HALF, torch.float32])
@pytest.mark.parametrize('channels', [4, 100, 129, 260, 516, 1001, 1280])
def test_a_convolution_keeps_the_codes_of_its_input(sq, channels, dtype):  # noqa: F811
    """Also where a warp's last channels are not there."""
    x = torch.randn(2, 70, channels, device='cuda', generator=torch.Generator(device='cuda').manual_seed(channels)).to(dtype)
    n = torch.tensor([70, 33], dtype=torch.int32, device='cuda')
    held = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t) or t, lambda t: t):
        sq.causal_conv(x.requires_grad_(), torch.randn(channels, 4, device='cuda').to(dtype), lengths=n, keep='int8')
    codes, scales, _ = ref.pack(torch.where(ref.present(n, 2, 70, 'cuda')[..., None], x.detach(), torch.zeros_like(x)))
    assert torch.equal(next(t for t in held if t.dtype == torch.int8), codes)
    assert any(t.shape == scales.shape and torch.equal(t, scales) for t in held)
