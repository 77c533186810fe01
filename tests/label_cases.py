"""Shared by test_label_ops.py (CPU) and test_gpu_label_ops.py: inputs, and the bounds the results are held to."""
import numpy as np
import torch

from oracle import label_ref as R

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
STEP = 2.0 ** -24   # half a step of float32, relative


def half_step(t):
    return torch.finfo(t).eps / 2


def smallest(t):
    """What a value may lose by underflow: half a subnormal step, and 2^-126 below which 2^x is 0."""
    return {torch.float32: 2.0 ** -125, torch.bfloat16: 2.0 ** -125, torch.float16: 2.0 ** -25}[t]


def distill_inputs(n, v, k, dt, seed, tail=False, spread=3.0, wide=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, v, generator=g) * spread).to(dt)
    ids = torch.stack([torch.randperm(v, generator=g)[:k] if v >= k else torch.randint(0, v, (k,), generator=g)
                       for _ in range(max(n, 1))])[:n]
    top = (2.0 + 2.0 * torch.rand(n, k, generator=g)).to(dt)
    lse = None
    if tail:
        lse = torch.logaddexp(torch.logsumexp(top.float(), 1), torch.randn(n, generator=g) + 1.0)
    return x, ids if wide else ids.int(), top, lse


def check_distill(loss, grad, x, ids, top, lse, weights, T, reduction, upstream=1.0):
    """loss, grad against 64 bits.  With A, B the largest |x - max| / T and |t / T| (+ |lse|) of finite entries:
    an exponent's argument is off by 3 roundings of itself and the exponential by 2 steps, a sum of V of them by
    the adds of its longest chain (32 in a thread, 9 to join a block, 64 over chunks), the log of it by as much,
    so each log q, log p is off by STEP (105 + 4 A + 4 B) and each q, p by that relatively; K terms add K roundings."""
    dt = x.dtype
    xn, tn = x.detach().double().cpu().numpy(), top.detach().double().cpu().numpy()
    ids = ids.cpu().numpy()
    ln = None if lse is None else lse.double().cpu().numpy()
    wn = None if weights is None else weights.double().cpu().numpy()
    up = upstream.double().cpu().numpy() if torch.is_tensor(upstream) else upstream
    want, gwant, rows = R.distill(xn, ids, tn, ln, wn, T, reduction, up)
    n, v = xn.shape
    w = np.ones(n) if wn is None else wn
    fin = lambda a: np.where(np.isfinite(a) & (np.abs(a) < 1e30), a, 0.0)  # noqa: E731
    A = (fin(xn).max(1, initial=0) - fin(xn).min(1, initial=0)) / T
    B = np.abs(fin(tn)).max(1, initial=0) / T + (0 if ln is None else np.abs(ln))
    rel = STEP * (105 + 4 * A + 4 * B + ids.shape[1] + 4 * np.log(v + 1.0))
    row_tol = T * T * rel * (2 + A + B) * np.abs(w)
    norm = 1.0 if reduction != 'mean' else (0.0 if w.sum() == 0 else 1.0 / w.sum())
    loss = loss.detach().double().cpu().numpy()
    # the loss is a float32: beyond 3.4028e38 the nearest one is infinity
    want = np.where(np.abs(want) > np.finfo(np.float32).max, np.copysign(np.inf, want), want)
    if reduction == 'none':
        ok = np.isfinite(want)
        assert np.array_equal(ok, np.isfinite(loss)) and np.array_equal(np.isnan(want), np.isnan(loss))
        assert np.all(np.abs(loss[ok] - want[ok]) <= row_tol[ok] + STEP * np.abs(want[ok]) * 4)
    elif np.isfinite(want):
        with np.errstate(invalid='ignore'):
            mags = np.abs(np.where(w == 0, 0, w * rows)).sum()
        assert abs(loss - want) <= (row_tol.sum() + 4 * STEP * mags) * norm + 1e-37, (loss, want)
    else:
        assert np.array_equal(loss, want, equal_nan=True), (loss, want)
    if grad is None:
        return
    grad = grad.double().cpu().numpy()
    # kept labels: q and p each off by rel; others by rel of q_o and of rest, which K roundings of 1 - sum p move too
    scale = np.abs(w) * norm * np.abs(np.broadcast_to(up, (n,))) * T
    tol = half_step(dt) * (1 + 1e-3) * np.abs(gwant) + smallest(dt)
    slack = np.zeros_like(gwant)
    for r in range(n):
        if w[r] == 0:
            continue
        _, g1 = R.distill_row(xn[r], ids[r], tn[r], None if ln is None else ln[r], T)
        z = fin(xn[r]) / T
        q = np.exp(z - z.max())
        q = np.where(np.isfinite(xn[r]), q / q.sum(), 0)
        slack[r] = scale[r] * rel[r] * 2 * (np.abs(g1) / T + q + (1.0 if ln is not None else 0.0) *
                                           (np.abs(g1) / T + 2 * q))
        if ln is not None:   # rest = 1 - sum p loses rel of the sum, shared out over the others by their q / q_o
            other = np.ones(v, bool)
            other[[i for i in ids[r] if 0 <= i < v]] = False
            if other.any() and q[other].sum() > 0:
                slack[r][other] += scale[r] * rel[r] * 2 * q[other] / q[other].sum()
    assert np.array_equal(np.isnan(gwant), np.isnan(grad))
    bad = np.abs(grad - gwant) > tol + slack
    assert not bad.any(), (np.argwhere(bad)[:5], grad[bad][:5], gwant[bad][:5], (tol + slack)[bad][:5])


def check_logits(got, want, mag, dt, adds):
    """Every step of a value rounds to float32 once (adds steps and the product's own), then to dt once."""
    got = got.double().cpu().numpy().reshape(want.shape)
    inf = ~np.isfinite(want)
    assert np.array_equal(got[inf], want[inf], equal_nan=True)
    tol = half_step(dt) * (1 + 1e-3) * np.abs(want) + STEP * (adds + 4) * mag + smallest(dt)
    top = torch.finfo(dt).max
    with np.errstate(invalid='ignore'):
        bad = ~inf & ~(np.abs(got - want) <= tol) & ~((np.abs(want) + tol > top) & np.isinf(got))
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])


def check_embedding_grad(got, ids, g, v, scale, pad):
    """Adding c rows in 32 bits rounds c times, each by STEP of what has been added so far."""
    want, mag, cnt = R.embedding_grad(ids.cpu().numpy(), g.double().cpu().numpy(), v, scale, pad)
    got_n = got.double().cpu().numpy()
    tol = half_step(got.dtype) * (1 + 1e-3) * np.abs(want) + STEP * (cnt[:, None] + 2) * mag + smallest(got.dtype)
    assert np.all(np.abs(got_n - want) <= tol)
    assert np.all(got_n[cnt == 0] == 0)
