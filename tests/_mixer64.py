"""The mixer's operators from their definitions in 64 bits, token by token, with the magnitudes that bound rounding.

`scan` returns values and, from the same recurrence over absolute values, the sum of the magnitudes of the terms that each
value is made of: a relative error e of every term changes the value by at most e times that."""
import torch


def present(lengths, batch, length, device):
    t = torch.arange(length, device=device)
    return (t < lengths[:, None]) if lengths is not None else torch.ones(batch, length, dtype=torch.bool, device=device)


def conv(x, weight, bias=None, state=None, lengths=None, silu=True):
    """(y, last inputs); differentiable in double tensors."""
    batch, length, channels = x.shape
    taps = weight.shape[1]
    there = present(lengths, batch, length, x.device)[..., None]
    first = x.new_zeros(batch, taps - 1, channels) if state is None else state
    whole = torch.cat([first, torch.where(there, x, torch.zeros_like(x))], 1)
    z = sum(whole[:, k:k + length] * weight[:, k] for k in range(taps))
    if bias is not None:
        z = z + bias
    y = z * torch.sigmoid(z) if silu else z
    ends = torch.full((batch,), length, device=x.device) if lengths is None else lengths.long()
    last = torch.stack([whole[b, int(e):int(e) + taps - 1] for b, e in enumerate(ends)])
    return torch.where(there, y, torch.zeros_like(y)), last


def scan(x, dt, A, B, C, D=None, dt_bias=None, state=None, lengths=None, step=None):
    """(y, last state).  step: softplus(dt + dt_bias) as it weighs the tokens, where it is a leaf of its own."""
    batch, length, heads, dim = x.shape
    per = heads // B.shape[2]
    there = present(lengths, batch, length, x.device)
    v = dt if dt_bias is None else dt + dt_bias
    s = torch.logaddexp(v, torch.zeros_like(v))
    weigh = s if step is None else step
    H = x.new_zeros(batch, heads, dim, 128) if state is None else state
    ys = []
    for t in range(length):
        Bt, Ct = B[:, t].repeat_interleave(per, 1), C[:, t].repeat_interleave(per, 1)
        new = torch.exp(A * s[:, t])[..., None, None] * H + (weigh[:, t, :, None] * x[:, t])[..., None] * Bt[:, :, None]
        on = there[:, t, None, None, None]
        H = torch.where(on, new, H)
        y = (new * Ct[:, :, None]).sum(-1)
        if D is not None:
            y = y + D[:, None] * x[:, t]
        ys.append(torch.where(on[..., 0], y, torch.zeros_like(y)))
    return torch.stack(ys, 1), H


def scan_with_grads(x, dt, A, B, C, D, dt_bias, state, lengths, dy, dlast=None):
    """({name: value}, {name: sum of magnitudes}) of y, last and the gradients of every given tensor."""
    given = dict(x=x, dt=dt, A=A, B=B, C=C, D=D, dt_bias=dt_bias, state=state)

    def clean(t):
        """What is not there is zero, whatever was written in its place."""
        if lengths is None:
            return t
        there = present(lengths, t.shape[0], t.shape[1], t.device)
        return torch.where(there.reshape(*there.shape, *[1] * (t.ndim - 2)), t, torch.zeros_like(t))

    def run(f):
        leaves = {}
        for k, v in given.items():
            if v is not None:
                v = clean(v.detach().double()) if k in ('x', 'dt', 'B', 'C') else v.detach().double()
                leaves[k] = (v if k in ('dt', 'A', 'dt_bias') else f(v)).requires_grad_()
        full = {k: leaves.get(k) for k in given}
        y, last = scan(*(full[k] for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias', 'state')), lengths)
        up = f(clean(dy.double()))
        loss = (y * up).sum()
        if dlast is not None:
            loss = loss + (last * f(dlast.double())).sum()
        names = list(leaves)
        grads = dict(zip(names, torch.autograd.grad(loss, [leaves[k] for k in names], allow_unused=True)))
        return dict(y=y.detach(), last=last.detach(), **{'d' + k: torch.zeros_like(leaves[k]) if g is None else g for k, g in grads.items()}), full, up
    values, _, _ = run(lambda t: t)
    sums, full, up = run(torch.abs)
    # the two ways a step acts, decay and weight, have gradients of opposite signs: their magnitudes add
    v = full['dt'].detach() if dt_bias is None else full['dt'].detach() + full['dt_bias'].detach()
    leaf = torch.logaddexp(v, torch.zeros_like(v)).requires_grad_()
    fixed = {k: None if t is None else t.detach() for k, t in full.items()}
    y, last = scan(*(fixed[k] for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias', 'state')), lengths, step=leaf)
    loss = (y * up).sum() if dlast is None else (y * up).sum() + (last * dlast.double().abs()).sum()
    weigh = torch.autograd.grad(loss, leaf)[0] * torch.sigmoid(v)
    decay = weigh - sums['ddt']                      # minus the decays' part, which A < 0 makes negative
    sums['ddt'] = weigh + decay.abs()
    if dt_bias is not None:
        sums['ddt_bias'] = sums['ddt'].sum((0, 1))
    sums['dA'] = sums['dA'].abs()
    return values, sums


def pack(x):
    """(codes, scales, values) of x [..., width], the scales' and quotients' fp32 arithmetic written out."""
    width = x.shape[-1]
    blocks = -(-width // 128)
    v = torch.zeros(*x.shape[:-1], blocks * 128, dtype=torch.float32, device=x.device)
    v[..., :width] = x.float()
    v = v.unflatten(-1, (blocks, 128))
    scale = v.abs().amax(-1) * torch.tensor(1.0 / 127.0, dtype=torch.float32, device=x.device)
    codes = torch.round(v / torch.where(scale == 0, torch.ones_like(scale), scale)[..., None]).clamp(-127, 127)
    values = codes * scale[..., None]
    return codes.flatten(-2)[..., :width].to(torch.int8), scale, values.flatten(-2)[..., :width]
