"""Plain 64-bit forms of the label-vocabulary operators, row by row from their definitions (numpy)."""
import numpy as np


def distill_row(x, ids, top, lse, T):
    """(loss, gradient [V]) of one row of weight 1; lse None: the kept entries renormalised."""
    x, top = np.asarray(x, np.float64), np.asarray(top, np.float64)
    V = x.shape[0]
    keep = [(int(i), float(t)) for i, t in zip(ids, top) if 0 <= i < V]
    zero = np.zeros(V)
    if np.all(x == -np.inf):
        return 0.0, zero
    if not any(lse is not None or t > -np.inf or np.isnan(t) for _, t in keep):
        return 0.0, zero
    with np.errstate(all='ignore'):
        z = x / T
        m = z.max()
        logq = (z - m) - np.log(np.exp(z - m).sum())   # (m + log would round a large m)
        ts = np.array([t for _, t in keep]) / T
        if lse is None:
            tm = ts.max()
            logp = (ts - tm) - np.log(np.exp(ts - tm).sum())
        else:
            logp = ts - float(lse)
        p = np.exp(logp)
        kl, g = 0.0, np.exp(logq)
        for (i, _), lp, pk in zip(keep, logp, p):
            if pk != 0:
                kl += pk * (lp - logq[i])
            g[i] -= pk
        if lse is not None:   # (the masses sum to 1 with the bucket, unless it is cut off at 0 or has no label)
            other = np.ones(V, bool)
            other[[i for i, _ in keep]] = False
            rest = max(0.0, 1.0 - p.sum()) if other.any() else 0.0
            total = p.sum() + rest
            g += (total - 1.0) * np.exp(logq)
            if other.any():
                zo = logq[other]
                mo = zo.max()
                logo = -np.inf if mo == -np.inf else mo + np.log(np.exp(zo - mo).sum())
                if rest > 0:
                    kl += rest * (np.log(rest) - logo)
                share = np.zeros(zo.shape) if mo == -np.inf else np.exp(zo - mo) / np.exp(zo - mo).sum()
                g[other] = share * (total * np.exp(logo) - rest)
        return T * T * kl, T * g


def distill(x, ids, top, lse=None, weights=None, T=1.0, reduction='mean', upstream=1.0):
    """(loss or row losses, gradient [N, V], row losses of weight 1)."""
    N = len(x)
    w = np.ones(N) if weights is None else np.asarray(weights, np.float64)
    rows, grads = np.zeros(N), np.zeros(np.shape(x))
    for r in range(N):
        if w[r] != 0:
            rows[r], grads[r] = distill_row(x[r], ids[r], top[r], None if lse is None else lse[r], T)
    norm = 1.0
    if reduction == 'mean':
        norm = 0.0 if w.sum() == 0 else 1.0 / w.sum()
    with np.errstate(invalid='ignore'):
        loss = w * rows if reduction == 'none' else (0.0 if norm == 0 else (w * rows).sum() * norm)
    f = w * norm * np.broadcast_to(np.asarray(upstream, np.float64), (N,))
    return loss, np.where((w == 0)[:, None], 0.0, grads) * f[:, None], rows


def process_logits(x, history=None, history_len=None, prompt_len=None, repetition=1.0, presence=0.0, frequency=0.0,
                   bias=None, bias_ids=None, bias_values=None, allowed=None):
    """(logits, the sum of the magnitudes that went into each), allowed: truth values [N, V]."""
    x = np.array(x, np.float64)
    N, V = x.shape
    mag = np.abs(x)

    def row(a, r):
        a = np.asarray(a, np.float64)
        return a if a.ndim == 0 else a[r]

    for r in range(N):
        if history is not None:
            h = np.asarray(history if np.ndim(history) == 1 else history[r])
            n = len(h) if history_len is None else min(max(int(history_len[r]), 0), len(h))
            given = 0 if prompt_len is None else int(prompt_len[r])
            for v in set(int(i) for i in h[:n]):
                if not 0 <= v < V:
                    continue
                c = int((h[max(given, 0):n] == v).sum()) if given < n else 0
                rep = float(row(repetition, r))
                x[r, v] = x[r, v] / rep if x[r, v] > 0 else x[r, v] * rep
                mag[r, v] = np.abs(x[r, v])
                if c:   # (what was not answered keeps its value under an infinite penalty)
                    mag[r, v] += abs(row(frequency, r)) * c + abs(row(presence, r))
                    x[r, v] -= row(frequency, r) * c + row(presence, r)
        if bias is not None:
            b = np.asarray(bias, np.float64)
            x[r] += b if b.ndim == 1 else b[r]
            mag[r] += np.abs(b if b.ndim == 1 else b[r])
        if bias_ids is not None:
            ids = np.asarray(bias_ids if np.ndim(bias_ids) == 1 else bias_ids[r])
            val = np.asarray(bias_values if np.ndim(bias_values) == 1 else bias_values[r], np.float64)
            for i, b in zip(ids, val):
                if 0 <= i < V:
                    x[r, i] += b
                    mag[r, i] += abs(b)
        if allowed is not None:
            a = np.asarray(allowed)
            x[r][~(a if a.ndim == 1 else a[r])] = -np.inf
    return x, mag


def embedding_grad(ids, grad, V, scale, padding=-1):
    """(d table [V, D], the sum of magnitudes per entry, how many rows went into each)."""
    ids, grad = np.asarray(ids).reshape(-1), np.asarray(grad, np.float64)
    grad = grad.reshape(len(ids), grad.shape[-1])
    out, mag, cnt = np.zeros((V, grad.shape[1])), np.zeros((V, grad.shape[1])), np.zeros(V)
    ok = (ids >= 0) & (ids < V) & (ids != padding)
    np.add.at(out, ids[ok], grad[ok])
    np.add.at(mag, ids[ok], np.abs(grad[ok]))
    np.add.at(cnt, ids[ok], 1)
    return out * scale, mag * abs(scale), cnt
