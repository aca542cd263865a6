"""Definitions of the operators on rows of logits in torch on the device, for tests at sizes where the numpy
oracle is slow: whole weights for a draw (its token is exact), 64 bits for the distillation loss."""
import numpy as np
import torch

LOG2E = 1.4426950408889634


def whole_draw(x, u, t=1.0, k=0, p=1.0, q=0.0, block=50):
    """The tokens of sample(x, u, t, k, p, q) by its definition in whole weights: nothing is left to rounding."""
    out = []
    for r in range(0, len(x), block):
        f, v = x[r:r + block].float(), u[r:r + block]
        m = f.amax(1, keepdim=True)
        c = torch.tensor(LOG2E, device='cuda') / torch.tensor(t, device='cuda')
        y = torch.where(f == m, 1.0, torch.exp2((f - m) * c))
        w = torch.round(y * 2.0 ** 31).long()
        order = torch.sort(f + 0.0, dim=1, descending=True, stable=True)[1]
        ws, ys = w.gather(1, order), y.gather(1, order)
        rank = torch.arange(x.shape[1], device='cuda')
        if k:
            ws = torch.where(rank < k, ws, 0)
        keep = ys >= np.float32(q)
        if p < 1.0:
            keep &= (ws.cumsum(1) - ws).double() < float(np.float32(p)) * ws.sum(1, keepdim=True).double()
        run = torch.zeros_like(w).scatter_(1, order, torch.where(keep | (rank == 0), ws, 0)).cumsum(1)
        target = (v.double()[:, None] * run[:, -1:].double()).long()
        out.append((run <= target).sum(1))
    return torch.cat(out)


def distill64(x, values, indices, T):
    """(loss, p, q over the vocabulary, record's q, gap) in 64 bits of rows that have a record; gap [rows, k] is
    the difference of the teacher's and the student's distance to their largest logits."""
    s, v = x.double(), values.double()
    at = indices.long().clamp(0, x.shape[1] - 1)
    used = (indices >= 0) & (indices < x.shape[1]) & (values > float('-inf'))
    v = torch.where(used, v, float('-inf'))
    dv, ds = v - v.amax(1, keepdim=True), s - s.amax(1, keepdim=True)
    logq, logp = torch.log_softmax(dv / T, 1), torch.log_softmax(ds / T, 1)
    rq = torch.where(used, logq.exp(), 0.0)
    here = rq > 0
    loss = T * T * torch.where(here, rq * (logq - logp.gather(1, at)), 0.0).sum(1)
    gap = torch.where(here, dv - ds.gather(1, at), 0.0)
    p = logp.exp()
    q = torch.zeros_like(p).scatter_add_(1, at, rq)
    return loss, p, q, rq, gap
