"""A policy's answers straight from its logits (csrc/choose.hip): sampling under a temperature, top-k,
top-p and min-p, and the record of a row's top entries that ``distill_loss`` learns from.

Beside :func:`~card_playing_gym_amd.rl.masked_probabilities` and ``sample_rows``
(cardgym/rl/ppo.py:75-94), which restate the reference's sampling bit for bit: ``sample_logits`` is one
launch from logits of any type and up to 2^18 entries a row to the actions and their log-probabilities, as
``policy_loss`` takes them.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from .. import _native as nat
from ..nn.kv_cache import dtype_code, require_device, stream_handle
from ..nn.optim import _on
from .policy import _no_tangents

MAX_WIDTH = 2**18
MAX_TOP = 256


class Sample(NamedTuple):
    """``actions`` (int64 [rows]) and the log of each one's share of what was kept (float32 [rows])."""

    actions: torch.Tensor
    log_probs: torch.Tensor


class TopLogits(NamedTuple):
    """``log_probs`` (float32) and ``indices`` (int64), both [rows, k], and ``log_rest`` (float32 [rows])."""

    log_probs: torch.Tensor
    indices: torch.Tensor
    log_rest: torch.Tensor


def _entries(t: torch.Tensor) -> torch.Tensor:
    """Entries of a row side by side; rows at any stride."""

    return t if t.stride(1) == 1 else t.detach().contiguous()


def _policy_rows(logits: torch.Tensor, mask: torch.Tensor | None) -> tuple[nat.PolicyRows, tuple]:
    """The native descriptor, and the tensors that it points at."""

    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError("logits must be [rows, width] with at least one entry a row")
    require_device(logits)
    dtype = dtype_code(logits.dtype)
    rows, width = shape = logits.shape
    if rows >= 2**31 or width > MAX_WIDTH:
        raise ValueError(f"logits may have up to 2^31 - 1 rows of up to {MAX_WIDTH} entries")
    logits = _entries(logits)
    if mask is None:
        return nat.PolicyRows(logits.data_ptr(), None, logits.stride(0), 0, rows, width, dtype), (logits, None)
    if mask.shape != shape or mask.dtype != torch.bool or mask.device != logits.device:
        raise ValueError("mask must be bool [rows, width] on the logits' device")
    mask = _entries(mask)
    return (nat.PolicyRows(logits.data_ptr(), mask.data_ptr(), logits.stride(0), mask.stride(0), rows, width, dtype),
            (logits, mask))


def _control(x, name: str, none, dtype: torch.dtype, rows: int, device) -> tuple:
    """A control's value and its tensor; ``none``: what stands for no filter."""

    if not isinstance(x, torch.Tensor):
        return (none if x is None else x), None
    if x.shape != (rows,) or x.dtype != dtype or x.device != device:
        raise ValueError(f"{name} must be a number or {dtype} [rows] on the logits' device")
    return none, x.contiguous()


@torch.compiler.disable
def sample_logits(
    logits: torch.Tensor,
    uniforms: torch.Tensor,
    *,
    mask: torch.Tensor | None = None,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor | None = None,
    top_p: float | torch.Tensor | None = None,
    min_p: float | torch.Tensor | None = None,
) -> Sample:
    """One action a row of ``logits`` [rows, width] (float32, bfloat16 or float16; up to 2^18 entries), from
    the random numbers ``uniforms`` (float64 [rows] in [0, 1)).

    A row's legal entries are those that ``mask`` (bool [rows, width]) keeps and whose logit is above -inf.
    With m the largest, an entry weighs w = exp((z - m) / temperature).  In the order of their logits, larger
    ones first and of equal ones the lower index, the filters keep a beginning:

    * ``top_k``: the first k (None, 0 or less: all);
    * ``top_p``: of these, those before which less than ``top_p`` of their weights is summed up (None, 1 or more: all);
    * ``min_p``: of these, those of at least ``min_p`` of the largest weight (None, 0 or less: all);

    the first entry always.  The action is the first entry of the order at which the running sum over what is
    kept exceeds uniform times all of it; ``log_probs`` is the log of its share.  A temperature of 0 takes the first entry.

    Each control is a number, or a tensor [rows] (float32; ``top_k`` int64) with every row's own.  A number is looked at: a
    temperature that is negative, infinite or NaN, a ``top_p`` below 0 or NaN, a ``min_p`` above 1 or NaN is refused.
    A row's own, which is on the device, is taken as it stands: an infinite temperature weighs all legal entries alike, a
    ``top_p`` below 0 and a ``min_p`` above 1 leave the first entry, and a NaN in either is no filter.

    A row without a legal entry has action -1 and log-probability 0.  One with a NaN among its legal entries
    (or a negative or NaN temperature of its own) has action -1 and NaN.  Entries at +inf share everything.
    Weights are whole multiples of a unit, 2^-50 of the largest in rows of up to 4096 entries and up to 2^-44 in wider
    ones: an entry of less than half a unit is never drawn.
    The actions are the same whatever the launch: a row's sums are exact.  Nothing here is differentiable: ``log_probs``
    carry no gradient (``policy_loss`` forms its own from the logits), and forward-mode tangents are refused."""

    descriptor, held = _policy_rows(logits, mask)
    _no_tangents(logits, uniforms, temperature, top_p, min_p, name="sample_logits")
    rows, device = descriptor.rows, logits.device
    if uniforms.shape != (rows,) or uniforms.dtype != torch.float64 or uniforms.device != device:
        raise ValueError("uniforms must be float64 [rows] on the logits' device")
    uniforms = uniforms.contiguous()
    t, ts = _control(temperature, "temperature", 1.0, torch.float32, rows, device)
    p, ps = _control(top_p, "top_p", 1.0, torch.float32, rows, device)
    m, ms = _control(min_p, "min_p", 0.0, torch.float32, rows, device)
    k, ks = _control(top_k, "top_k", 0, torch.int64, rows, device)
    if not 0 <= t < math.inf:
        raise ValueError("temperature must be finite and not negative")
    if not p >= 0:
        raise ValueError("top_p must not be negative")
    if not m <= 1:
        raise ValueError("min_p may be 1 at most")
    if k % 1 != 0:  # (a share of the entries, say, would be cut to 0: all of them)
        raise ValueError("top_k must be a whole number")
    controls = nat.SampleControls(t, p, m, min(max(int(k), 0), MAX_WIDTH), *(None if x is None else x.data_ptr()
                                                                             for x in (ts, ps, ms, ks)))
    actions = torch.empty(rows, device=device, dtype=torch.int64)
    log_probs = torch.empty(rows, device=device)
    with _on(device):
        nat.call("cg_sample_logits", descriptor, uniforms.data_ptr(), controls, actions.data_ptr(), log_probs.data_ptr(),
                 stream_handle(device))
    return Sample(actions, log_probs)


@torch.compiler.disable
def top_logits(
    logits: torch.Tensor, k: int, *, mask: torch.Tensor | None = None, temperature: float = 1.0
) -> TopLogits:
    """The record of a policy's answers: of each row of ``logits`` [rows, width] (float32, bfloat16 or float16;
    up to 2^18 entries) the ``k`` largest legal entries (up to 256), larger first and of equal ones the lower
    index first.

    ``log_probs``: their logs under the softmax of logits / ``temperature`` over all legal entries (those that
    ``mask``, bool [rows, width], keeps and whose logit is above -inf); ``log_rest``: the log of what all
    others have together, summed by itself, so that a rest far below 1 keeps its digits.

    Where a row has fewer than k legal entries the places behind them hold -inf and index -1, and ``log_rest``
    is -inf, as ``distill_loss`` takes them.  A row with a NaN among its legal entries reports NaN and
    indices -1.  Entries at +inf share everything.  The record is a constant: it carries no gradient of the logits, and
    forward-mode tangents are refused."""

    descriptor, held = _policy_rows(logits, mask)
    _no_tangents(logits, name="top_logits")
    rows, device = descriptor.rows, logits.device
    if not 1 <= k <= MAX_TOP:
        raise ValueError(f"k must be from 1 to {MAX_TOP}")
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError("temperature must be from 1e-30 to 1e30")
    log_probs = torch.empty((rows, k), device=device)
    indices = torch.empty((rows, k), device=device, dtype=torch.int64)
    log_rest = torch.empty(rows, device=device)
    with _on(device):
        nat.call("cg_top_logits", descriptor, k, temperature, log_probs.data_ptr(), indices.data_ptr(),
                 log_rest.data_ptr(), stream_handle(device))
    return TopLogits(log_probs, indices, log_rest)
