"""Categorical actions and gradient clipping, restated from their definitions in float64 numpy, one row at a time."""
import numpy as np


def allowed_entries(x, mask):
    ok = x > -np.inf
    ok |= np.isnan(x)
    return ok if mask is None else ok & mask


def kept_entries(x, mask=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Indices (rising) that a draw chooses from, and their weights; x float64 (V,)."""
    idx = np.flatnonzero(allowed_entries(x, mask))
    if idx.size == 0:
        return idx, np.zeros(0)
    order = idx[np.lexsort((idx, -x[idx]))]
    if temperature == 0:
        return order[:1], np.ones(1)
    w = np.exp((x[order] - x[order[0]]) / temperature)
    n = len(order) if top_k <= 0 else min(int(top_k), len(order))
    if top_p < 1:
        total = w[:n].sum()
        before = np.concatenate([[0.0], np.cumsum(w[:n])[:-1]])
        n = max(1, int((before < max(top_p, 0.0) * total).sum()))
    n = max(1, min(n, int((w >= min(max(min_p, 0.0), 1.0)).sum())))
    back = np.argsort(order[:n])
    return order[:n][back], w[:n][back]


def sample_row(x, u, mask=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(action, log_prob) of one row; the settings are the values that 32 bits hold."""
    x = np.asarray(x, np.float64)
    ok = allowed_entries(x, mask)
    if np.isnan(x[ok]).any() or (x[ok] == np.inf).any() or not temperature >= 0:
        return -1, np.nan
    idx, w = kept_entries(x, mask, temperature, top_k, top_p, min_p)
    if idx.size == 0:
        return -1, 0.0
    u = 0.0 if not u > 0 else min(float(u), 1.0 - 2.0 ** -24)
    c = np.cumsum(w)
    i = min(int((c <= u * c[-1]).sum()), len(idx) - 1)
    return int(idx[i]), float(np.log(w[i] / c[-1]))


def evaluate_row(x, action, mask=None, temperature=1.0, gl=0.0, ge=0.0):
    """(log_prob, entropy, gradient (V,)) of one row."""
    x = np.asarray(x, np.float64)
    ok = allowed_entries(x, mask)
    V = len(x)
    if not ok.any():
        lp = 0.0 if action == -1 else np.nan if not 0 <= action < V else -np.inf
        return lp, 0.0, np.zeros(V)
    z = np.where(ok, x / temperature, -np.inf)
    with np.errstate(invalid="ignore"):
        d = z - z.max()
        e = np.where(ok, np.exp(d), 0.0)
        log_p = d - np.log(e.sum())
        p = np.where(ok, np.exp(log_p), 0.0)
        h = -np.where(ok, p * np.where(ok, log_p, 0.0), 0.0).sum()
        lp = 0.0 if action == -1 else np.nan if not 0 <= action < V else log_p[action] if ok[action] or np.isnan(h) else -np.inf
        if action == -1:
            gl = 0.0
        elif not 0 <= action < V:
            gl = np.nan
        grad = np.where(ok, -p * (gl + ge * (np.where(ok, log_p, 0.0) + h)), 0.0)
    if 0 <= action < V and ok[action]:
        grad[action] += gl
    return lp, h, grad / temperature


def grad_norm(grads, norm_type=2.0):
    if norm_type == np.inf:
        parts = [np.abs(g).max() for g in grads if g.size]
        return float(np.max(parts)) if parts else 0.0
    if norm_type == 1:
        return float(sum(np.abs(g).sum() for g in grads))
    return float(np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in grads)))


def clip_factor(norm, max_norm):
    f = max_norm / (norm + 1e-6)
    return f if f != f or f < 1.0 else 1.0
