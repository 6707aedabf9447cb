"""Distillation from a teacher's top logits in 64 bits: loss, log-sum-exp and gradient of each row."""
import numpy as np


def distill(logits, ids, teacher, temperature=1.0, weights=None, upstream=None, grad_scale=1.0):
    """logits: (rows, vocab); ids, teacher: (rows, k).  Returns (loss, lse, grad) as float64 arrays."""
    s = np.asarray(logits, np.float64)
    rows, vocab = s.shape
    t = float(temperature)
    w = np.ones(rows) if weights is None else np.asarray(weights, np.float64)
    up = np.ones(rows) if upstream is None else np.asarray(upstream, np.float64)
    loss, lse, grad = np.zeros(rows), np.zeros(rows), np.zeros((rows, vocab))
    for r in range(rows):
        entries = [(int(i), float(v)) for i, v in zip(ids[r], teacher[r]) if i >= 0 and not v == -np.inf]
        if w[r] == 0 or not entries:
            continue
        y = np.array([v for _, v in entries]) / t
        if any(i >= vocab for i, _ in entries) or not np.isfinite(y.max()) or not np.isfinite(s[r].max()):
            loss[r] = lse[r] = np.nan
            grad[r] = np.nan
            continue
        at = np.array([i for i, _ in entries])
        logp = y - y.max() - np.log(np.exp(y - y.max()).sum())
        p = np.exp(logp)
        x = s[r] / t
        lse[r] = x.max() + np.log(np.exp(x - x.max()).sum())
        some = p > 0
        loss[r] = w[r] * t * t * (p[some] * (logp[some] - x[at[some]] + lse[r])).sum()
        q = np.exp(x - lse[r])
        np.subtract.at(q, at, p)
        grad[r] = grad_scale * up[r] * w[r] * t * q
    return loss, lse, grad
