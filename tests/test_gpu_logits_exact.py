"""Draws from long rows against the definition in whole weights: tokens are equal, none is left out of the
comparison.  Few rows run on CTAs of 512 threads, some hundred on 256 (fp32 rows over 768 KB: 512 again)."""
import pytest
import torch

from _logits64 import whole_draw
from test_gpu_logits import TYPES, make

pytestmark = pytest.mark.gpu

SETTINGS = [dict(), dict(p=0.9), dict(p=0.5, q=0.01), dict(q=0.02, t=0.8), dict(k=300), dict(k=2000, p=0.9),
            dict(k=100000, p=0.7, t=1.5), dict(k=5000, p=0.95, q=1e-4), dict(k=40, p=0.9, t=0.7)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,vocab,spread', [(3, 256000, 1.0), (3, 262144, 3.0), (300, 256000, 3.0), (300, 131001, 1.0)])
def test_long_rows_draw_the_defined_token(rows, vocab, spread, dtype):
    import sq325
    x, g = make(rows, vocab, dtype, seed=rows + vocab, spread=spread, pad=1, banned=0.02)
    for s in SETTINGS:
        u = torch.rand(rows, generator=g, device='cuda')
        got = sq325.sample(x, u, temperature=s.get('t', 1.0), top_k=s.get('k', 0), top_p=s.get('p', 1.0), min_p=s.get('q', 0.0))
        assert torch.equal(got, whole_draw(x, u, **s)), s


@pytest.mark.parametrize('dtype', TYPES)
def test_rows_of_few_values_draw_the_defined_token(dtype):
    """Ties at the cut spread over eight CTAs: rows of two to some hundred values, signed zeros among them."""
    import sq325
    g = torch.Generator(device='cuda').manual_seed(7)
    r = torch.rand((6, 256000), generator=g, device='cuda')
    x = torch.stack([torch.floor(r[0] * 2), torch.floor(r[1] * 40) / 4, torch.where(r[2] < 0.999, 5.0, 6.0), torch.zeros_like(r[3]),
                     torch.where(r[4] < 0.5, 0.0, -0.0), torch.floor(-200 * r[5]) / 16]).to(dtype)
    for s in (dict(p=0.3), dict(p=0.85), dict(k=70001), dict(k=70001, p=0.5), dict(k=3000, p=0.9, q=0.3), dict(k=255, p=0.5)):
        u = torch.rand(len(x), generator=g, device='cuda')
        got = sq325.sample(x, u, top_k=s.get('k', 0), top_p=s.get('p', 1.0), min_p=s.get('q', 0.0))
        assert torch.equal(got, whole_draw(x, u, **s)), s
