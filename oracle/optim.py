"""The optimiser step in numpy float64: AdamW with decoupled weight decay, moments in 32 bits or
in 8-bit blocks, and the clipping factor of a global norm.

``torch.optim.AdamW`` and ``clip_grad_norm_`` are the definition for 32 bits; the 8-bit blocks are
this project's own format, restated here from its definition with a table of the codes' values
and ``numpy.frexp`` (the kernel cuts the codes from a double's bits)."""

from __future__ import annotations

import numpy as np

BLOCK = 256
M32 = np.uint64(0xFFFFFFFF)


def clip_factor(norm: float, max_norm: float) -> float:
    return min(1.0, max_norm / (norm + 1e-6))


def adamw(p, g, m, v, t, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
    """New (p, m, v), float64; t counts from 1."""

    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * (g * g)
    update = lr / (1 - betas[0] ** t) * m / (np.sqrt(v / (1 - betas[1] ** t)) + eps)
    return p - lr * weight_decay * p - update, m, v


def mix(x: np.ndarray) -> np.ndarray:
    x = np.asarray(x, dtype=np.uint64) & M32
    x = x ^ x >> np.uint64(16)
    x = x * np.uint64(0xD2511F53) & M32
    x = x ^ x >> np.uint64(15)
    x = x * np.uint64(0xCD9E8D57) & M32
    return x ^ x >> np.uint64(16)


def words(seed: int, t: int, tensor: int, elements: np.ndarray) -> np.ndarray:
    """The 32 random bits of each element of a tensor at step t."""

    key = mix(mix(mix(np.uint64(seed & 0xFFFFFFFF)) + np.uint64(t)) + np.uint64(tensor))
    elements = elements.astype(np.uint64)
    high = (elements >> np.uint64(32)) * np.uint64(0x9E3779B9)
    return mix(((elements & M32) ^ key) + high)


def code_values(signed: bool) -> np.ndarray:
    """What each of the 256 codes stands for, in units of its block's scale."""

    q = np.arange(128 if signed else 256)
    u = q + (889 if signed else 761)
    f = np.where(q > 0, (1 + u % 8 / 8) * 2.0 ** (u // 8 - 127), 0.0)
    return np.concatenate([f, -f]) if signed else f


def decode(codes: np.ndarray, scales: np.ndarray, signed: bool) -> np.ndarray:
    return code_values(signed)[codes] * np.repeat(scales.astype(np.float64), BLOCK)[: codes.size]


def encode(x: np.ndarray, noise: np.ndarray, signed: bool) -> tuple[np.ndarray, np.ndarray]:
    """(codes, scales) of float64 x [n] from 16-bit random numbers [n]."""

    n, blocks = x.size, -(-x.size // BLOCK)
    size = np.zeros(blocks * BLOCK)
    size[:n] = np.abs(x)
    scales = size.reshape(blocks, BLOCK).max(1).astype(np.float32)
    inverse = np.zeros_like(scales)
    np.divide(np.float32(1), scales, out=inverse, where=scales >= np.finfo(np.float32).tiny)
    y = np.abs(x) * np.repeat(inverse.astype(np.float64), BLOCK)[:n]
    most, least = (127, 889) if signed else (255, 761)
    fraction, power = np.frexp(y)
    eighths = np.floor(fraction * 16 + (2 * noise.astype(np.int64) + 1) / 2.0**17).astype(np.int64)
    q = np.clip(8 * (power.astype(np.int64) + 126) + eighths - 8 - least, 0, most)
    q = np.where(y > 0, q if signed else np.maximum(q, 1), 0)
    return np.where((x < 0) & (q > 0), q + 128, q).astype(np.uint8) if signed else q.astype(np.uint8), scales


def adamw8(p, g, m, v, t, seed, tensor, *args, elements=None, **kwargs):
    """As ``adamw`` with m and v each a (codes, scales) pair; flat arrays."""

    elements = np.arange(p.size) if elements is None else elements
    p, m, v = adamw(p, g, decode(*m, True), decode(*v, False), t, *args, **kwargs)
    random = words(seed, t, tensor, elements)
    return p, encode(m, random & np.uint64(0xFFFF), True), encode(v, random >> np.uint64(16), False)
