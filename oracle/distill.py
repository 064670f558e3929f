"""The distillation loss towards a record of top entries, row by row in numpy float64 from the definition."""

from __future__ import annotations

import numpy as np

from .choose import log_sum_exp


def distill(logits, indices, log_probs, log_rest=None, mask=None, weights=None, normalizer=None, temperature=1.0) -> dict:
    """loss, kl [rows], grad [rows, width]; and for bars: x = (m - z) / T and p [rows, width]."""

    rows, width = logits.shape
    weights = np.ones(rows) if weights is None else weights.astype(np.float64)
    n = rows if normalizer is None else normalizer
    out = {"kl": np.zeros(rows), "grad": np.zeros((rows, width)), "x": np.zeros((rows, width)), "p": np.zeros((rows, width)),
           "q": np.zeros((rows, width)), "size": np.zeros(rows)}
    for r in range(rows):
        z = logits[r].astype(np.float64) / temperature
        legal = (np.ones(width, dtype=bool) if mask is None else mask[r]) & ~(z == -np.inf)
        there = indices[r] != -1
        at, logq = indices[r][there], log_probs[r][there].astype(np.float64)
        if weights[r] == 0 or not legal.any():
            continue
        astray = ((at < 0) | (at >= width)).any() or len(set(at)) < len(at)
        if log_rest is None and not astray and (logq == -np.inf).all():
            continue
        if astray or np.isnan(z[legal]).any() or (z[legal] == np.inf).any():
            out["kl"][r], out["grad"][r] = np.nan, np.nan
            continue
        logp = np.where(legal, z - log_sum_exp(z[legal]), -np.inf)
        if log_rest is None:
            logq = logq - log_sum_exp(logq)
        q, p = np.exp(logq), np.exp(logp)
        some = q > 0
        terms = q[some] * (logq[some] - logp[at[some]])
        kl, mass = terms.sum(), q.sum()
        size = np.abs(q[some] * logq[some]).sum() + np.abs(terms).sum()
        grad = np.zeros(width)
        if log_rest is not None:
            q_rest = np.exp(np.float64(log_rest[r]))
            outside = legal.copy()
            outside[at] = False
            log_p_rest = log_sum_exp(logp[outside])
            mass += q_rest
            if q_rest > 0:
                kl += q_rest * (log_rest[r] - log_p_rest)
                size += np.abs(q_rest * log_rest[r]) + np.abs(q_rest * log_p_rest)
                grad[outside] -= q_rest * np.exp(logp[outside] - log_p_rest)
        grad += mass * p
        grad[at] -= np.where(legal[at], q, 0.0)
        out["kl"][r], out["grad"][r], out["size"][r] = kl, grad * weights[r] / (n * temperature), size
        out["p"][r], out["q"][r][at] = p, q
        out["x"][r] = np.where(legal, np.where(legal, z, -np.inf).max() - z, 0.0)
    live = weights != 0
    out["loss"] = float((weights[live] * out["kl"][live]).sum() / n)
    return out
