"""Host side of PredictorState.logits without a GPU: what the entry point and the method refuse."""
import pytest
import torch


def test_entry_point_refuses():
    from sq325 import _lib
    lib = _lib.load()
    assert lib.sq_model_logits(None, 4096, 1, 4096, None, 0, None) == _lib.SQ_EINVAL
    assert b'logits' in lib.sq_last_error()


def test_method_needs_an_installed_controller():
    from sq325 import PredictorState
    controller = PredictorState.__new__(PredictorState)
    controller._handle = None
    with pytest.raises(RuntimeError, match='not installed'):
        controller.logits(torch.zeros(1, 4096, dtype=torch.float16))
    controller._handle, controller.device = object(), torch.device('cpu')
    for bad in (torch.zeros(1, 4096), torch.zeros(1, 4095, dtype=torch.float16), torch.zeros(0, 4096, dtype=torch.float16), None):
        with pytest.raises(ValueError, match='hidden'):
            controller.logits(bad)
