"""The operators on rows of logits as the model's loops and the example use them."""
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from _models import build_pair
from oracle import logits as ol

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def pair():
    return build_pair(n_layer=2, vocab=512, seed=1, adapter=True)


def _prompt(vocab, batch=3, length=9):
    return torch.from_numpy(np.random.default_rng(4).integers(0, vocab, (batch, length)).astype(np.int64))


def test_generate_without_sampling_or_with_one_choice_is_greedy(pair):
    from sq325 import PredictorState, generate
    gm, _, statics = pair
    with PredictorState(gm, *statics) as ex:
        want = generate(ex, _prompt(gm.vocab), 6)
        assert torch.equal(want, generate(ex, _prompt(gm.vocab), 6, sampling=dict(temperature=0.0)))
        assert torch.equal(want, generate(ex, _prompt(gm.vocab), 6, sampling=dict(top_k=1)))
        per_row = dict(temperature=torch.zeros(3, device='cuda'))
        assert torch.equal(want, generate(ex, _prompt(gm.vocab), 6, sampling=per_row))
        ex.check()


def test_generate_draws_from_the_given_numbers(pair):
    """Step by step: the drawn token is the oracle's draw from the step's own logits."""
    from sq325 import PredictorState, generate
    gm, _, statics = pair
    settings = dict(temperature=1.2, top_k=40, top_p=0.9)
    gen = torch.Generator(device='cuda').manual_seed(3)
    uniform = torch.rand((5, 3), generator=gen, device='cuda')
    with PredictorState(gm, *statics) as ex:
        got = generate(ex, _prompt(gm.vocab), 5, sampling=settings, uniform=uniform)
        again = generate(ex, _prompt(gm.vocab), 5, sampling=settings, generator=torch.Generator(device='cuda').manual_seed(3))
        assert got.shape == (3, 5) and torch.equal(got, again)
        hidden = ex.backbone(_prompt(gm.vocab).cuda(), reset=True)[:, -1]
        for step in range(5):
            logits = torch.empty((3, gm.vocab), device='cuda', dtype=torch.float16)
            ex.greedy(hidden, logits=logits)
            rows = logits.double().cpu().numpy()
            for b in range(3):
                token, margin = ol.draw(rows[b], float(uniform[step, b]), settings['temperature'], 40, 0.9)
                assert margin < 1e-4 or token == int(got[b, step])
            hidden = ex.backbone(got[:, step:step + 1].contiguous())[:, 0]
        ex.check()


def test_generate_refuses_mixed_arguments(pair):
    from sq325 import PredictorState, generate
    gm, _, statics = pair
    with PredictorState(gm, *statics) as ex:
        with pytest.raises(ValueError):
            generate(ex, _prompt(gm.vocab), 4, uniform=torch.rand(4, 3, device='cuda'))
        with pytest.raises(ValueError):
            generate(ex, _prompt(gm.vocab), 4, graphs=True, sampling=dict(top_k=5))
        with pytest.raises(ValueError):
            generate(ex, _prompt(gm.vocab), 4, sampling=dict(top_k=5), uniform=torch.rand(3, 3, device='cuda'))


def test_model_logits_and_many_rows(pair):
    """logits() is the exactly decoded lm_head; sample() takes it for more than 64 rows."""
    from sq325 import PredictorState, fp4, top_logits
    gm, _, statics = pair
    with PredictorState(gm, *statics) as ex:
        hidden = ex.backbone(_prompt(gm.vocab, batch=5, length=16).cuda(), reset=True)
        logits = ex.logits(hidden)
        assert logits.shape == (5, 16, gm.vocab) and logits.dtype == torch.float16
        want = hidden.float() @ fp4.decode_packet(gm.lm_head).float().T
        assert (logits.float() - want).abs().max() <= 2e-3 * want.abs().max()
        values, indices = top_logits(logits, 8)
        assert torch.equal(values[..., 0], logits.amax(-1)) and indices.shape == (5, 16, 8)
        tokens = ex.sample(hidden, torch.full((80,), 0.5, device='cuda'), temperature=0.0)
        assert torch.equal(tokens.view(5, 16), indices[..., 0].long())
        few = ex.sample(hidden[:, -1], torch.full((5,), 0.5, device='cuda'), top_k=1)
        assert torch.equal(few, ex.greedy(hidden[:, -1]))
        ex.check()


def test_example_learns_from_the_teacher():
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / 'examples'))
    import distill_head
    text, losses = distill_head.run(steps=12, vocab=2048, batch=3, prompt=8, answer=10)
    again, _ = distill_head.run(steps=1, vocab=2048, batch=3, prompt=8, answer=10)
    assert text.shape == (3, 10) and torch.equal(text, again)
    assert all(np.isfinite(losses)) and losses[-1] < 0.9 * losses[0]
