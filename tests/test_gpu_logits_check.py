"""PredictorState.logits: failures inside it reach the controller's check()."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_expired_wait_in_logits_raises_device_timeout():
    """A bounded wait that runs out in the head's projection (one row: the skinny GEMM) leaves logits that are not
    whole; check() says so, and the next call is whole again."""
    from _models import build_pair
    from sq325 import PredictorState, _lib
    gm, _, statics = build_pair(n_layer=2, vocab=512, seed=6, adapter=True)
    ids = torch.from_numpy(np.random.default_rng(8).integers(0, 512, (1, 9))).cuda()
    with PredictorState(gm, *statics) as ex:
        hidden = ex.backbone(ids, reset=True)[:, -1]
        want = ex.logits(hidden)
        ex.check()
        try:
            _lib.call('sq_set_wait_limit_ns', 1)
            ex.logits(hidden)
            with pytest.raises(_lib.DeviceTimeout):
                ex.check()
        finally:
            _lib.call('sq_set_wait_limit_ns', 0)
        assert torch.equal(ex.logits(hidden), want)
        ex.check()


@pytest.mark.parametrize('rows', [1, 2, 64, 65, 256, 257, 700])
def test_logits_are_those_of_the_decoded_head(rows):
    """The bits of fp4.linear on the head, on both sides of the sizes where another kernel runs."""
    import sq325
    from sq325 import fp4
    from sq325.model import benchmark_layouts, synthetic_statics
    model = sq325.synthetic_model(seed=2, n_layer=1, vocab=40000)
    table, layouts, bases, scales, predictors = synthetic_statics(benchmark_layouts(1), seed=2)
    g = torch.Generator(device='cuda').manual_seed(rows)
    hidden = torch.randn((rows, 4096), generator=g, device='cuda').half()
    with sq325.PredictorState(model, table, layouts, bases, scales, predictors) as ex:
        got = ex.logits(hidden)
        assert got.shape == (rows, 40000) and torch.equal(got, fp4.linear(model.lm_head, hidden))
        strided = torch.cat([hidden, hidden], 1)[:, :4096].view(1, rows, 4096)
        assert torch.equal(ex.logits(strided)[0], got)
        ex.check()


def test_entry_point_refuses_bad_buffers():
    """Nothing is launched: a null or misaligned buffer, no rows, a workspace that is too small."""
    import sq325
    from sq325 import _lib
    from sq325.model import benchmark_layouts, synthetic_statics
    model = sq325.synthetic_model(seed=2, n_layer=1, vocab=512)
    with sq325.PredictorState(model, *synthetic_statics(benchmark_layouts(1), seed=2)) as ex:
        hidden = torch.zeros((300, 4096), device='cuda', dtype=torch.float16)
        out = torch.empty((300, 512), device='cuda', dtype=torch.float16)
        h, o, call = hidden.data_ptr(), out.data_ptr(), _lib.load().sq_model_logits
        for args in ((None, 1, o, None, 0), (h + 2, 1, o, None, 0), (h, 0, o, None, 0), (h, 1, None, None, 0), (h, 1, o + 1, None, 0),
                     (h, 300, o, None, 0), (h, 300, o, h, 300 * 4096)):
            assert call(ex._handle, *args, None) == _lib.SQ_EINVAL, args
        ex.check()
