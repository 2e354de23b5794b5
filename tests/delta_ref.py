"""The gated delta rule token by token in 64 bits, the tests' oracle: written from its definition alone."""
import math

import torch


def delta64(q, k, v, log_decay, beta, state=None, scale=1.0):
    """q, k: (b, l, hk, dk); v: (b, l, h, dv); log_decay, beta: (b, l, h); state: (b, h, dv, dk).
    Everything in float64, differentiable.  Returns (out, final state)."""
    b, l, h, dv = v.shape
    group = h // q.shape[2]
    q, k, v, log_decay, beta = (t.double() for t in (q, k, v, log_decay, beta))
    s = torch.zeros(b, h, dv, k.shape[3], dtype=torch.float64, device=v.device) if state is None else state.double()
    outs = []
    for t in range(l):
        kt = k[:, t].repeat_interleave(group, 1)
        qt = q[:, t].repeat_interleave(group, 1)
        a = torch.exp(log_decay[:, t])[..., None, None]
        s = torch.where(a > 0, a * s, 0.0)  # exp(-inf) = 0: a reset, with no slope in log_decay
        e = v[:, t] - (s * kt[:, :, None, :]).sum(-1)
        s = s + (beta[:, t, :, None] * e)[..., None] * kt[:, :, None, :]
        outs.append(scale * (s * qt[:, :, None, :]).sum(-1))
    return torch.stack(outs, 1), s


def make(b, l, hk, group, dk, dv, dtype, seed=0, device="cuda", decay=1.0, resets=0.0, zero_beta=0.0,
         state=False):
    """Inputs of a call, as a layer makes them: unit keys and queries, write strengths in (0, 1)."""
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    h = hk * group
    q, k = r(b, l, hk, dk), r(b, l, hk, dk)
    q, k = q / q.norm(dim=-1, keepdim=True), k / k.norm(dim=-1, keepdim=True)
    g = -decay * torch.nn.functional.softplus(r(b, l, h) - 1)
    beta = torch.sigmoid(r(b, l, h))
    if resets:
        g = torch.where(torch.rand(b, l, h, generator=gen) < resets, -math.inf, g)
    if zero_beta:
        beta = torch.where(torch.rand(b, l, h, generator=gen) < zero_beta, 0.0, beta)
    x = [t.to(dtype).to(device) for t in (q, k, r(b, l, h, dv), g, beta)]
    s = (0.3 * r(b, h, dv, dk)).float().to(device) if state else None
    return x, s


def off(x, want):
    """Norm of the difference over the norm of what is wanted."""
    x, want = x.detach().double(), want.detach().double()
    d, n = (x - want).norm(), want.norm()
    return float(d / n) if n > 0 else float(d)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tolerance(dtype, wide, products):
    """Rounding of the result, and of `products` products one after another.  A product of operands in bf16
    parts leaves out terms of 3 x 2^-17 at most (two parts; 3 x 2^-25 with three), and sums of up to 16
    steps, truncated to 24 bits, are off by 16 x 2^-23 at most (wide: rounded and stepwise, 8 x 2^-24)."""
    unit = 3 * 2 ** -25 + 8 * 2 ** -24 if wide or dtype == torch.float32 else 3 * 2 ** -17 + 16 * 2 ** -23
    return half_step(dtype) + products * unit


def decay_gradient_sizes(x, state, go, gs, scale):
    """How large the terms of dlog_decay are that cross each token t: the sum over i >= t > j of the norms that
    meet in them, a token's own error and gradient counted with all that they are differences of.  go, gs:
    gradients of the output and of the last state (or None).  In 64 bits, the whole sequence at once."""
    q, k, v, g, beta = (t.detach().double() for t in x)
    b, l, h, dv = v.shape
    group = h // q.shape[2]
    norm = lambda t: t.norm(dim=-1).transpose(1, 2)  # noqa: E731  (b, h, l)
    q, k = norm(q).repeat_interleave(group, 1), norm(k).repeat_interleave(group, 1)
    v, go, beta = norm(v), norm(go.double()), beta.transpose(1, 2)
    cum = g.clamp(min=-10000.0).transpose(1, 2).cumsum(-1)
    lower = torch.ones(l, l, dtype=torch.bool, device=v.device).tril()
    d = torch.where(lower, torch.exp(torch.where(lower, cum[..., :, None] - cum[..., None, :], 0.0)), 0.0)
    strict = d.tril(-1)
    first = 0.0 if state is None else state.double().flatten(2).norm(dim=-1)[..., None]
    last = 0.0 if gs is None else gs.double().flatten(2).norm(dim=-1)[..., None]
    enter, leave = cum.exp(), (cum[..., -1:] - cum).exp()
    # e_j = v_j - what the state says; dv_i = what e_i's write is read for
    kk = strict * k[..., :, None] * (beta * k)[..., None, :]
    e = v + enter * k * first
    for _ in range(3):  # each write is read by the next ones' errors, and so on: three rounds are enough for a size
        e = v + enter * k * first + (kk @ e[..., None])[..., 0]
    reads = (d * (scale * q * go)[..., :, None]).sum(-2) * beta * k + leave * beta * k * last
    dv = reads
    for _ in range(3):
        dv = reads + (kk.mT @ dv[..., None])[..., 0]
    a = strict * (scale * q * go + k * dv)[..., :, None] * (beta * k * e)[..., None, :]
    left = a.cumsum(-1) - a  # of the columns before t (sums of positive numbers)
    t = torch.where(lower, left, 0.0).sum(-2)
    t = t + (enter * (scale * q * go + k * dv) * first).flip(-1).cumsum(-1).flip(-1)
    w = leave * beta * k * e * last
    t = t + (w.cumsum(-1) - w) + enter[..., -1:] * first * last
    return t.transpose(1, 2)
