"""Host side of the operators on rows of logits, without a GPU: refusals of the C entry points and of the
Python functions, and the oracle against plain torch in 64 bits."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import logits as ol


@pytest.fixture(scope='module')
def lib():
    from sq325 import _lib
    return _lib.load()


def _fields(**kw):
    from sq325 import _lib
    a = dict(data=4096, row_stride=10, rows=2, vocab=10, type=_lib.F32)
    a.update(kw)
    return [a[k] for k in ('data', 'row_stride', 'rows', 'vocab', 'type')]


def _logits(**kw):
    from sq325 import _lib
    return _lib.Logits(*_fields(**kw))


def test_bindings_lay_the_fields_out_as_the_header_does():
    """sq_logits is 32 bytes, and what follows it in the two argument blocks begins there."""
    from sq325 import _lib
    assert C.sizeof(_lib.Logits) == 32
    assert _lib.SampleArgs.uniform.offset == 32 and C.sizeof(_lib.SampleArgs) == 96
    assert _lib.DistillArgs.values.offset == 32 and _lib.DistillArgs.weight.offset == 64 and C.sizeof(_lib.DistillArgs) == 112


BAD_LOGITS = [dict(data=None), dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(vocab=0),
              dict(vocab=(1 << 18) + 1), dict(row_stride=-1), dict(data=4098)]


@pytest.mark.parametrize('bad', BAD_LOGITS)
def test_entry_points_refuse_logits(lib, bad):
    """Nothing is read or launched: the pointers are not valid ones."""
    from sq325 import _lib
    a = _lib.SampleArgs(*_fields(**bad), 4096, None, None, None, None, 1.0, 0, 1.0, 0.0, 4096)
    assert lib.sq_sample(C.byref(a), None) == _lib.SQ_EINVAL
    assert lib.sq_top_logits(C.byref(_logits(**bad)), 2, 4096, 4096, None) == _lib.SQ_EINVAL
    d = _lib.DistillArgs(*_fields(**bad), 4096, 4096, 2, _lib.F32, 1.0, None, 0, 4096, 4096, 4096, 10)
    for name in ('sq_distill_forward', 'sq_distill_backward', 'sq_distill_loss_grad'):
        assert getattr(lib, name)(C.byref(d), None) == _lib.SQ_EINVAL
        assert name[3:].encode() in lib.sq_last_error()


def test_entry_points_refuse_the_rest(lib):
    from sq325 import _lib
    for name in ('sq_sample', 'sq_distill_forward', 'sq_distill_backward', 'sq_distill_loss_grad'):
        assert getattr(lib, name)(None, None) == _lib.SQ_EINVAL
    assert lib.sq_top_logits(None, 1, 4096, 4096, None) == _lib.SQ_EINVAL
    for k in (0, 11, 1025):
        assert lib.sq_top_logits(C.byref(_logits()), k, 4096, 4096, None) == _lib.SQ_EINVAL
    assert lib.sq_top_logits(C.byref(_logits()), 2, None, 4096, None) == _lib.SQ_EINVAL
    assert lib.sq_top_logits(C.byref(_logits()), 2, 4096, None, None) == _lib.SQ_EINVAL
    for uniform, tokens in ((None, 4096), (4096, None)):
        a = _lib.SampleArgs(*_fields(), uniform, None, None, None, None, 1.0, 0, 1.0, 0.0, tokens)
        assert lib.sq_sample(C.byref(a), None) == _lib.SQ_EINVAL
    good = dict(values=4096, indices=4096, k=2, value_type=_lib.F32, temperature=1.0, weight=None, weight_stride=0,
                loss=4096, stats=4096, grad=4096, grad_stride=10)
    every = ('sq_distill_forward', 'sq_distill_backward', 'sq_distill_loss_grad')
    forward, backward, fused = every
    for bad, names in ((dict(values=None), every), (dict(indices=None), every), (dict(values=4098), every),
                       (dict(indices=4098), every), (dict(k=0), every), (dict(k=1025), every),
                       (dict(value_type=5), every), (dict(temperature=0.0), every),
                       (dict(temperature=float('nan')), every), (dict(temperature=float('inf')), every),
                       (dict(weight_stride=-1), every), (dict(loss=None), (forward, fused)),
                       (dict(stats=4104), (forward, backward)), (dict(stats=None), (backward,)),
                       (dict(grad=None), (backward, fused)), (dict(grad=4098), (backward, fused)),
                       (dict(grad_stride=9), (backward, fused))):
        a = dict(good, **bad)
        d = _lib.DistillArgs(*_fields(), *(a[k] for k in good))
        for name in names:
            assert getattr(lib, name)(C.byref(d), None) == _lib.SQ_EINVAL, (name, bad)


def test_entry_points_accept_no_rows(lib):
    from sq325 import _lib
    none = _logits(rows=0, data=None)
    fields = _fields(rows=0, data=None)
    a = _lib.SampleArgs(*fields, None, None, None, None, None, 1.0, 0, 1.0, 0.0, None)
    assert lib.sq_sample(C.byref(a), None) == _lib.SQ_OK
    assert lib.sq_top_logits(C.byref(none), 2, None, None, None) == _lib.SQ_OK
    d = _lib.DistillArgs(*fields, None, None, 2, _lib.F32, 1.0, None, 0, None, None, None, 0)
    for name in ('sq_distill_forward', 'sq_distill_backward', 'sq_distill_loss_grad'):
        assert getattr(lib, name)(C.byref(d), None) == _lib.SQ_OK


def test_functions_refuse_host_tensors():
    import sq325
    x, u = torch.zeros(2, 8), torch.zeros(2)
    v, i = torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32)
    for f in (lambda: sq325.sample(x, u), lambda: sq325.top_logits(x, 2), lambda: sq325.distillation_loss(x, v, i),
              lambda: sq325.distillation_loss_grad(x, v, i), lambda: sq325.sample(np.zeros((2, 8)), u)):
        with pytest.raises(ValueError, match='CUDA'):
            f()


def test_generate_checks_its_sampling_arguments():
    from sq325 import generate

    class Execution:
        device = torch.device('cpu')
    for kw in (dict(uniform=torch.zeros(2, 1)), dict(generator=torch.Generator()),
               dict(sampling=dict(top_k=2), graphs=True), dict(sampling=dict(top_k=2), uniform=torch.zeros(3, 1)),
               dict(sampling=dict(top_k=2), uniform=torch.zeros(2, 1), generator=torch.Generator())):
        with pytest.raises(ValueError):
            generate(Execution(), [1, 2], 2, **kw)


def test_generate_samples_through_the_execution():
    """The loop's order on a stand-in: prompt, one draw per step from that step's numbers, stop at EOS."""
    from sq325 import generate
    seen = []

    class Execution:
        device = torch.device('cpu')

        def backbone(self, ids, reset=False):
            return torch.zeros(ids.shape[0], ids.shape[1], 4)

        def sample(self, hidden, uniform, **settings):
            seen.append((uniform.clone(), settings))
            return torch.full((hidden.shape[0],), len(seen))
    uniform = torch.arange(8.0).view(4, 2) / 8
    out = generate(Execution(), [[1, 2], [3, 4]], 4, eos_token_id=3, sampling=dict(top_k=5), uniform=uniform)
    assert out.tolist() == [[1, 2, 3], [1, 2, 3]]
    assert [s for _, s in seen] == [dict(top_k=5)] * 3 and all(torch.equal(u, uniform[n]) for n, (u, _) in enumerate(seen))


# ------------------------------------------------------------------ the oracle
def test_oracle_distillation_against_torch():
    rng = np.random.default_rng(0)
    for T in (0.7, 1.0, 3.0):
        s = torch.tensor(rng.standard_normal(50) * 3, requires_grad=True)
        values, indices = rng.standard_normal(6), rng.permutation(50)[:6]
        logq = torch.log_softmax(torch.tensor(values) / T, 0)
        logp = torch.log_softmax(s / T, 0)[torch.tensor(indices)]
        loss = T * T * (logq.exp() * (logq - logp)).sum()
        grad, = torch.autograd.grad(loss, s)
        got = ol.distill(s.detach().numpy(), np.append(values, [9.0, -np.inf]), np.append(indices, [-1, 3]), T)
        assert np.isclose(got[0], float(loss.detach()), rtol=1e-12) and np.allclose(got[1], grad.numpy(), atol=1e-14)
    assert ol.distill(rng.standard_normal(5), [1.0], [-1])[0] == 0.0


def test_oracle_draw_follows_its_definition():
    x = np.array([0.0, 3.0, -np.inf, 3.0, np.nan, 1.0])
    assert ol.order(ol.plain(x)).tolist()[:4] == [1, 3, 5, 0]
    assert ol.draw(x, 0.99, temperature=0.0)[0] == 1
    assert ol.draw(x, 0.99, top_k=1)[0] == 1 and ol.draw(x, 0.99, top_k=2)[0] == 3
    w = np.exp(ol.plain(x))
    share = w / w.sum()
    grid = (np.arange(4000) + 0.5) / 4000
    count = np.bincount([ol.draw(x, u)[0] for u in grid], minlength=6)
    assert np.abs(count - 4000 * share).max() <= 1
    assert {ol.draw(x, u, top_p=0.5)[0] for u in grid} == {1, 3}        # the first alone holds less than half
    assert {ol.draw(x, u, min_p=0.2)[0] for u in grid} == {1, 3} and {ol.draw(x, u, min_p=0.1)[0] for u in grid} == {1, 3, 5}
    assert ol.draw(np.full(4, -np.inf), 0.5)[0] == -1
    assert ol.top(x, 5)[1].tolist() == [1, 3, 5, 0, -1]
