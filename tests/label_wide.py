"""The label-vocabulary operators' distillation in 64 bits for many rows at once: its loss from the definition, its gradient
from that by autograd (apart from the formulas of oracle/label_ref.py), and the bounds of label_cases.check_distill by row."""
import math

import torch

import label_cases as C


def rows64(x, ids, top, lse, T):
    """The row losses of weight 1, differentiable in x [n, v] (float64)."""
    v = x.shape[1]
    there = (ids >= 0) & (ids < v)
    at = ids.long().masked_fill(~there, 0)
    t = top.double().masked_fill(~there, -math.inf) / T
    dead = (x == -math.inf).all(1) | ~there.any(1)
    if lse is None:
        dead = dead | (t == -math.inf).all(1)
        logp = torch.log_softmax(t.masked_fill(dead[:, None], 0.0), 1)
    else:
        logp = t - lse.double().masked_fill(dead, 0.0)[:, None]
    p = logp.exp()
    logq = torch.log_softmax(x.masked_fill(dead[:, None], 0.0) / T, 1)
    kl = torch.where(p > 0, p * (logp - logq.gather(1, at)), 0.0).sum(1)
    if lse is not None:
        listed = torch.zeros_like(logq).scatter_add_(1, at, there.double()) > 0
        full = listed.all(1)
        rest = (1.0 - p.sum(1)).clamp(min=0.0).masked_fill(full, 0.0)
        logo = torch.logsumexp(logq.masked_fill(listed & ~full[:, None], -math.inf), 1)
        kl = kl + torch.where(rest > 0, rest * (torch.log(rest.clamp(min=1e-300)) - logo), 0.0)
    return torch.where(dead, 0.0, kl * (T * T))


def distill64(x, ids, top, lse, w, T, reduction, up):
    """(loss, gradient, row losses of weight 1, their gradients)."""
    x = x.detach().double().requires_grad_(True)
    weight = torch.ones(x.shape[0], dtype=torch.float64, device=x.device) if w is None else w.double()
    live = weight != 0
    rows = rows64(x.masked_fill(~live[:, None], 0.0), ids, top, None if lse is None else lse, T)
    g1, = torch.autograd.grad(rows.sum(), x)
    rows = rows.detach().masked_fill(~live, 0.0)
    norm = 1.0 if reduction != 'mean' else 0.0 if weight.sum() == 0 else 1.0 / float(weight.sum())
    loss = weight * rows * norm
    return loss if reduction == 'none' else loss.sum(), g1 * (weight * norm * up)[:, None], rows, g1.masked_fill(~live[:, None], 0.0)


def check(loss, grad, x, ids, top, lse, w, T, reduction, up=1.0):
    """As label_cases.check_distill derives it; a factor of the kept mass, where that is above 1, on what it multiplies."""
    dt, (n, v) = x.dtype, x.shape
    if w is not None:   # (a row of weight 0 is not read)
        x = x.detach().masked_fill((w == 0)[:, None], 0.0)
    up = up.double() if torch.is_tensor(up) else torch.tensor(float(up), dtype=torch.float64, device=x.device)
    up = up.expand(n)
    want, gwant, rows, g1 = distill64(x, ids, top, lse, w, T, reduction, up)
    weight = torch.ones_like(rows) if w is None else w.double()
    norm = 1.0 if reduction != 'mean' else 0.0 if weight.sum() == 0 else 1.0 / float(weight.sum())

    def fin(a):
        return torch.where(a.isfinite() & (a.abs() < 1e30), a, torch.zeros_like(a))

    xf, tf = fin(x.detach().double()), fin(top.double())
    A = (xf.amax(1).clamp(min=0) - xf.amin(1).clamp(max=0)) / T
    B = tf.abs().amax(1) / T + (0 if lse is None else fin(lse.double()).abs())
    rel = C.STEP * (105 + 4 * A + 4 * B + ids.shape[1] + 4 * math.log(v + 1.0))
    there = (ids >= 0) & (ids < v)
    mass = torch.ones_like(rows)
    if lse is not None:
        mass = torch.where(there, torch.exp(top.double() / T - fin(lse.double())[:, None]), 0.0).sum(1).clamp(min=1.0)
    row_tol = T * T * rel * (2 + A + B) * weight.abs() * mass
    loss = loss.detach().double()
    if reduction == 'none':
        assert torch.all((loss - want).abs() <= row_tol + 4 * C.STEP * want.abs())
    else:
        assert (loss - want).abs() <= (row_tol.sum() + 4 * C.STEP * (weight * rows).abs().sum()) * norm + 1e-37, (loss, want)
    q = torch.softmax((x.detach().double() / T).masked_fill((x == -math.inf).all(1, keepdim=True), 0.0), 1) * mass[:, None]
    scale = weight.abs() * norm * up.abs() * T
    slack = g1.abs() / T + q
    if lse is not None:
        slack = slack + g1.abs() / T + 2 * q
        other = q.scatter(1, ids.long().masked_fill(~there, 0), 0.0) if bool(there.all()) else torch.where(
            torch.zeros_like(q).scatter_add_(1, ids.long().masked_fill(~there, 0), there.double()) > 0, 0.0, q)
        slack = slack + other / other.sum(1, keepdim=True).clamp(min=1e-300)
    tol = C.half_step(dt) * 1.001 * gwant.abs() + C.smallest(dt) + (scale * rel * 2)[:, None] * slack
    off = (grad.double() - gwant).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (bad.nonzero()[:5], grad[bad][:5], gwant[bad][:5], tol[bad][:5])


def over_full(n, v, k, dt, top_dt, T, seed):
    """Rows whose kept mass is not the whole of what 1 - mass gives a bucket: teacher logits kept in 16 bits beside the lse of
    a float32 row (mass 0.96 to 1.05), an entry listed twice, one absent, and plain rows."""
    g = torch.Generator().manual_seed(seed)
    x, ids, _, _ = C.distill_inputs(n, v, k, dt, seed)
    top = (4.0 * torch.rand(n, k, generator=g) + 14.0).to(top_dt)
    lse = torch.logsumexp(top.double() / T, 1)
    lse = lse + torch.tensor([-0.05, 0.04, -0.02, 1.0])[torch.arange(n) % 4]
    if k > 2 and n > 5:
        ids[4, 1] = ids[4, 0]
        ids[5, 2] = -1
    return x, ids, top, lse.float()
