"""The clipped policy loss in numpy float64: value, per-row numbers and gradient from the formulas."""

from __future__ import annotations

import numpy as np


def log_softmax(z: np.ndarray, legal: np.ndarray) -> np.ndarray:
    """Over the legal entries; -inf elsewhere."""

    z = np.where(legal, z, -np.inf)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        x = z - z.max(1, keepdims=True)
        return np.where(legal, x - np.log(np.exp(x).sum(1, keepdims=True)), -np.inf)


def policy_loss(logits, actions, old, advantages, mask=None, weights=None, normalizer=None, clip=0.2, clip_high=None,
                entropy_coef=0.0, kl_coef=0.0, reference_logits=None, reference_log_probs=None) -> dict:
    rows = len(logits)
    legal = np.isfinite(logits) if mask is None else mask & (logits > -np.inf)
    weights = np.ones(rows) if weights is None else weights.astype(np.float64)
    live = (weights != 0) & legal.any(1)
    out = {"loss": 0.0, "log_probs": np.zeros(rows), "entropy": np.zeros(rows), "kl": np.zeros(rows),
           "ratio": np.zeros(rows), "grad": np.zeros(logits.shape), "x": np.zeros(logits.shape),
           "p": np.zeros(logits.shape), "own": np.zeros(rows), "gap": np.zeros(logits.shape)}
    if not live.any():
        return out
    i = np.flatnonzero(live)
    z, legal, action = logits[i].astype(np.float64), legal[i], actions[i]
    adv = advantages[i].astype(np.float64)
    scale = weights[i] / (rows if normalizer is None else normalizer)
    at = (np.arange(len(i)), action)
    logp = log_softmax(z, legal)
    p = np.exp(logp)
    finite = np.where(p > 0, logp, 0.0)
    entropy = -(p * finite).sum(1)
    log_prob = logp[at]
    ratio = np.exp(log_prob - old[i].astype(np.float64))
    lo, hi = 1 - clip, 1 + (clip if clip_high is None else clip_high)
    clipped = np.clip(ratio, lo, hi)
    value = -np.minimum(ratio * adv, clipped * adv) - entropy_coef * entropy
    own = np.where((ratio >= lo) & (ratio <= hi) | (ratio * adv < clipped * adv), -adv * ratio, 0.0)
    bracket = entropy_coef * (finite + entropy[:, None])
    if reference_logits is not None:
        mine = legal if mask is None else mask[i]
        with np.errstate(invalid="ignore"):
            gap = np.where(p > 0, logp - log_softmax(reference_logits[i].astype(np.float64), mine), 0.0)
        kl = (p * gap).sum(1)
        value = value + kl_coef * kl
        bracket = bracket + kl_coef * (gap - kl[:, None])
        out["kl"][i], out["gap"][i] = kl, gap
    elif reference_log_probs is not None:
        d = reference_log_probs[i].astype(np.float64) - log_prob
        kl = np.expm1(d) - d
        value = value + kl_coef * kl
        own = own - kl_coef * np.expm1(d)
        out["kl"][i] = kl
    grad = p * (bracket - own[:, None])
    grad[at] += own
    out["grad"][i] = grad * scale[:, None]
    out["loss"] = float((scale * value).sum())
    out["size"] = float((scale * (np.abs(value) + entropy_coef * entropy)).sum())
    out["log_probs"][i], out["entropy"][i], out["ratio"][i], out["own"][i] = log_prob, entropy, ratio, own
    out["p"][i] = p
    out["x"][i] = np.where(p > 0, z - np.where(legal, z, -np.inf).max(1, keepdims=True), 0.0)
    return out
