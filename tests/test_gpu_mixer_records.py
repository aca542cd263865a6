"""Records of activations in 8 bits that are refused."""
import pytest
import torch

from test_gpu_mixer import sq  # noqa: F401

pytestmark = pytest.mark.gpu


def test_odd_records_are_refused(sq):  # noqa: F811
    codes, scales = torch.zeros(2, 0, dtype=torch.int8, device='cuda'), torch.zeros(2, 0, device='cuda')
    for bad in ((codes, scales, torch.float16), (codes[:, :0], None, torch.float16), ([1], [2], torch.float16), (codes, scales, torch.float64)):
        with pytest.raises(ValueError):
            sq.unpack_activations(bad)
