"""Sampling under controls and the record of a row's top entries, row by row in numpy float64 from the definitions."""

from __future__ import annotations

import numpy as np


def ordered(z: np.ndarray, legal: np.ndarray) -> np.ndarray:
    """A row's legal entries: larger logits first, of equal ones the lower index."""

    at = np.flatnonzero(legal & ~(z == -np.inf))
    return at[np.lexsort((at, -z[at]))]


def distances(z: np.ndarray, order: np.ndarray, temperature: float) -> np.ndarray:
    """(z - m) / T along the order; entries at +inf have 0, and others beside them -inf."""

    x = z[order]
    if len(x) and x[0] == np.inf:
        return np.where(x == np.inf, 0.0, -np.inf)
    return (x - x[:1]) / temperature


def kept_weights(z, legal, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The order and the weights that are kept along it (a beginning)."""

    order = ordered(z, legal)
    w = np.exp(distances(z, order, temperature))
    n = len(w)
    if 0 < top_k < n:
        n = top_k
    w = w[:n]
    if top_p < 1:
        ahead = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int((ahead < top_p * w.sum()).sum()))
    if min_p > 0:
        n = max(1, min(n, int((w >= min_p).sum())))
    return order, w[:n]


def sample(logits, uniforms, mask=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(actions, log_probs, margin): margin is how far u is, as a share, from another action."""

    rows, width = logits.shape
    each = lambda x: np.broadcast_to(np.asarray(x, dtype=np.float64), (rows,))  # noqa: E731
    t, k, p, m = each(temperature), each(top_k), each(top_p), each(min_p)
    actions, log_probs, margin = np.full(rows, -1), np.zeros(rows), np.ones(rows)
    for r in range(rows):
        z = logits[r].astype(np.float64)
        legal = np.ones(width, dtype=bool) if mask is None else mask[r]
        if np.isnan(z[legal]).any() or not t[r] >= 0:
            log_probs[r] = np.nan
            continue
        order = ordered(z, legal)
        if not len(order):
            continue
        if t[r] == 0:
            actions[r] = order[0]
            continue
        order, w = kept_weights(z, legal, t[r], int(k[r]), p[r], m[r])
        running = np.cumsum(w) / w.sum()
        beyond = np.flatnonzero(running > uniforms[r])
        at = beyond[0] if len(beyond) else np.flatnonzero(w > 0)[-1]
        actions[r] = order[at]
        log_probs[r] = distances(z, order, t[r])[at] - np.log(w.sum())
        margin[r] = np.abs(running[:-1] - uniforms[r]).min() if len(running) > 1 else 1.0
    return actions, log_probs, margin


def log_sum_exp(x: np.ndarray) -> float:
    return -np.inf if not len(x) or x.max() == -np.inf else float(x.max() + np.log(np.exp(x - x.max()).sum()))


def top(logits, k, mask=None, temperature=1.0):
    """(log_probs [rows, k], indices [rows, k], log_rest [rows])."""

    rows, width = logits.shape
    log_probs, indices, log_rest = np.full((rows, k), -np.inf), np.full((rows, k), -1), np.full(rows, -np.inf)
    for r in range(rows):
        z = logits[r].astype(np.float64)
        legal = np.ones(width, dtype=bool) if mask is None else mask[r]
        if np.isnan(z[legal]).any():
            log_probs[r], log_rest[r] = np.nan, np.nan
            continue
        order = ordered(z, legal)
        d = distances(z, order, temperature)
        n = min(k, len(order))
        whole = log_sum_exp(d)
        log_probs[r, :n], indices[r, :n] = d[:n] - whole, order[:n]
        log_rest[r] = log_sum_exp(d[n:]) - whole if len(d) > n else -np.inf
    return log_probs, indices, log_rest
