"""Distillation of a head from a teacher's own text, with the operators on rows of logits.

A synthetic FP4 teacher answers random prompts by sampling (generate with sampling=...), its
largest logits over the text are recorded (PredictorState.logits, top_logits), and a student's
head, the teacher's decoded weights plus noise, learns from the record (distillation_loss and its
backward, Adam).  The distillation loss falls.

    python examples/distill_head.py [--steps 30] [--vocab 4096] [--layers 2]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / 'mamb2_8b_fp4_recall_sq3.25_b200'))

import sq325  # noqa: E402
from sq325.model import benchmark_layouts, synthetic_statics  # noqa: E402


def run(steps=30, vocab=4096, layers=2, batch=4, prompt=16, answer=24, record=32, temperature=2.0, rate=0.01, seed=0):
    """Returns (text, losses): the teacher's text int64 [batch, answer] and the mean loss before each step."""
    gen = torch.Generator(device='cuda').manual_seed(seed)
    teacher = sq325.synthetic_model(seed=seed, n_layer=layers, vocab=vocab)
    layouts = benchmark_layouts(layers)
    table, layouts, bases, scales, predictors = synthetic_statics(layouts, seed=seed)
    with sq325.PredictorState(teacher, table, layouts, bases, scales, predictors) as execution:
        ids = torch.randint(0, vocab, (batch, prompt), generator=gen, device='cuda')
        text = sq325.generate(execution, ids, answer, sampling=dict(temperature=0.8, top_k=50, top_p=0.95), generator=gen)
        hidden = execution.backbone(torch.cat([ids, text], 1), reset=True)
        values, indices = sq325.top_logits(execution.logits(hidden), record)
        execution.check()
    head = sq325.fp4.decode_packet(teacher.lm_head).float()
    head += head.std() * torch.randn(head.shape, generator=gen, device='cuda')
    head.requires_grad_(True)
    hidden = hidden.float()
    adam = torch.optim.Adam([head], lr=rate * float(head.detach().std()))
    losses = []
    for _ in range(steps):
        loss = sq325.distillation_loss(hidden @ head.T, values, indices, temperature=temperature).mean()
        adam.zero_grad()
        loss.backward()
        adam.step()
        losses.append(float(loss.detach()))
    return text, losses


if __name__ == '__main__':
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, default in (('steps', 30), ('vocab', 4096), ('layers', 2), ('batch', 4), ('seed', 0)):
        ap.add_argument('--' + name, type=int, default=default)
    text, losses = run(**vars(ap.parse_args()))
    print('teacher text', tuple(text.shape), text[0, :8].tolist())
    print('loss', ' '.join(f'{x:.4f}' for x in losses[::max(1, len(losses) // 10)]), '->', f'{losses[-1]:.4f}')
