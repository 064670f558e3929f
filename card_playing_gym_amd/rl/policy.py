"""The policy loss of an update on the device: the clipped objective with an entropy bonus and a
KL term over rows of policy logits, forward and gradient in one pass (csrc/loss.hip).

It scores what :func:`~card_playing_gym_amd.rl.masked_probabilities` and ``sample_rows`` chose in the
rollout (cardgym/rl/ppo.py:75-94): the same softmax over a row's legal entries, differentiable.

    out = policy_loss(logits, actions, old_log_probs, advantages, mask=legal, entropy_coef=0.01)
    (out.loss + value_loss).backward()
"""

from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

import torch

from .. import _native as nat
from ..nn.kv_cache import dtype_code, require_device, stream_handle
from ..nn.optim import _on


class PolicyLoss(NamedTuple):
    """``loss``: the scalar to differentiate.  ``log_probs``, ``entropy`` and ``kl`` (None without a
    reference): each row's, for logging, float32 and without a gradient."""

    loss: torch.Tensor
    log_probs: torch.Tensor
    entropy: torch.Tensor
    kl: torch.Tensor | None


def _constant(t: torch.Tensor, name: str, shape: tuple[int, ...], dtype: torch.dtype, device) -> torch.Tensor:
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {dtype} {list(shape)} on the logits' device")
    if t.requires_grad:
        raise ValueError(f"{name} is a constant of the loss: detach it")
    return t


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Entries of a row side by side; rows at any stride."""

    return t if t.stride(-1) == 1 else t.contiguous()


class _Call:
    """One loss: its inputs, their native descriptor and what the forward writes."""

    __slots__ = ("descriptor", "tensors", "kl", "log_probs", "entropy", "logits")

    def __init__(self, logits, tensors, options) -> None:
        self.logits = logits
        self.tensors = tensors  # alive as long as the descriptor's addresses
        address = [None if t is None else t.data_ptr() for t in tensors]
        actions, old, advantages, weights, mask, reference_logits, reference_log_probs = address[:7]
        rows, width = logits.shape
        self.descriptor = nat.PolicyLoss(
            logits.data_ptr(), mask, actions, old, advantages, weights, reference_logits, reference_log_probs,
            logits.stride(0), 0 if mask is None else tensors[4].stride(0),
            0 if reference_logits is None else tensors[5].stride(0), rows, width, dtype_code(logits.dtype), *options,
        )

    def forward(self, grad: torch.Tensor | None) -> torch.Tensor:
        device, rows = self.logits.device, self.logits.shape[0]
        loss = torch.empty((), device=device)
        self.log_probs = torch.empty(rows, device=device)
        self.entropy = torch.empty(rows, device=device)
        self.kl = None if self.tensors[5] is None and self.tensors[6] is None else torch.empty(rows, device=device)
        size = _workspace_size()
        workspace = torch.empty(size, device=device, dtype=torch.uint8)
        with _on(device):
            nat.call(
                "cg_policy_loss_forward", self.descriptor, loss.data_ptr(), self.log_probs.data_ptr(),
                self.entropy.data_ptr(), None if self.kl is None else self.kl.data_ptr(),
                None if grad is None else grad.data_ptr(), workspace.data_ptr(), size, stream_handle(device),
            )
        return loss


@lru_cache(maxsize=1)
def _workspace_size() -> int:
    return nat.lib().cg_policy_loss_workspace_size()


class PolicyLossFunction(torch.autograd.Function):
    """The forward writes the gradient of the loss itself; the backward keeps it where the gradient
    arriving is 1 and forms it again, from the inputs, where it is another."""

    @staticmethod
    def forward(ctx, logits, call):
        # (call.logits is what the kernel reads: logits, or its copy with the entries side by side)
        ctx.written = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
        ctx.save_for_backward(call.logits, *call.tensors)
        ctx.call = call
        return call.forward(ctx.written)

    @staticmethod
    def backward(ctx, upstream):
        if torch.is_grad_enabled():  # (create_graph; once_differentiable costs 13 us of a small loss's 96)
            raise RuntimeError("policy_loss is differentiable once: its gradient has no graph")
        call = ctx.call
        logits = ctx.saved_tensors[0]  # (an input changed since the forward raises here)
        grad, ctx.written = ctx.written, None  # handed over once: a second backward forms its own
        written = grad is not None
        if grad is None:
            grad = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
        upstream = upstream.contiguous()
        with _on(logits.device):
            nat.call("cg_policy_loss_backward", call.descriptor, upstream.data_ptr(), int(written),
                     grad.data_ptr(), stream_handle(logits.device))
        return grad, None


@torch.compiler.disable
def policy_loss(
    logits: torch.Tensor,
    actions: torch.Tensor,
    old_log_probs: torch.Tensor,
    advantages: torch.Tensor,
    *,
    mask: torch.Tensor | None = None,
    weights: torch.Tensor | None = None,
    normalizer: float | torch.Tensor | None = None,
    clip: float = 0.2,
    clip_high: float | None = None,
    entropy_coef: float | torch.Tensor = 0.0,
    kl_coef: float | torch.Tensor = 0.0,
    reference_logits: torch.Tensor | None = None,
    reference_log_probs: torch.Tensor | None = None,
) -> PolicyLoss:
    """sum_i weights_i l_i / normalizer over the rows of ``logits`` [rows, width] (float32, bfloat16
    or float16), differentiable in the logits, with

        r = exp(log p[action] - old_log_prob)
        l = -min(r A, clamp(r, 1 - clip, 1 + clip_high) A) + kl_coef KL - entropy_coef H

    p is the softmax over the row's legal entries: those that ``mask`` (bool [rows, width]) keeps
    and whose logit is above -inf.  KL is sum p (log p - log q) with ``reference_logits`` (q over the same
    mask), or exp(d) - d - 1 with d = ``reference_log_probs`` - log p[action].

    ``actions``: int64 [rows].  ``old_log_probs``, ``advantages``, ``weights`` (ones) and
    ``reference_log_probs``: float32 [rows].  ``normalizer``: the number of rows; pass the whole
    minibatch's count where a microbatch's gradients are accumulated.  ``clip_high``: ``clip``.
    ``normalizer`` and the coefficients may be float32 device scalars, which a captured loss reads at
    every replay.

    A row of weight 0 (padding) is not read: like a row without a legal entry it adds nothing, has a
    zero gradient and reports zeros.  An action outside the row makes its row, and the loss, NaN; one that
    is not legal has log p = -inf."""

    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError("logits must be [rows, width] with at least one entry a row")
    require_device(logits)
    dtype_code(logits.dtype)
    rows, width = logits.shape
    device = logits.device
    vector = (rows,)
    _constant(actions, "actions", vector, torch.int64, device)
    _constant(old_log_probs, "old_log_probs", vector, torch.float32, device)
    _constant(advantages, "advantages", vector, torch.float32, device)
    if weights is not None:
        _constant(weights, "weights", vector, torch.float32, device)
    if mask is not None:
        mask = _rows(_constant(mask, "mask", (rows, width), torch.bool, device))
    if reference_logits is not None and reference_log_probs is not None:
        raise ValueError("give reference_logits or reference_log_probs, not both")
    if reference_logits is not None:
        reference_logits = _rows(_constant(reference_logits, "reference_logits", (rows, width), logits.dtype, device))
    if reference_log_probs is not None:
        reference_log_probs = _constant(reference_log_probs, "reference_log_probs", vector, torch.float32, device)
        reference_log_probs = reference_log_probs.contiguous()
    elif reference_logits is None and (isinstance(kl_coef, torch.Tensor) or kl_coef != 0):
        raise ValueError("kl_coef needs a reference")
    clip_high = clip if clip_high is None else clip_high
    if not clip >= 0 or not clip_high >= 0:
        raise ValueError("clip and clip_high must be non-negative")
    if normalizer is None:
        normalizer = float(max(rows, 1))
    elif not isinstance(normalizer, torch.Tensor) and not normalizer > 0:
        raise ValueError("normalizer must be positive")
    scalars, kept = [], []
    for name, x in (("normalizer", normalizer), ("entropy_coef", entropy_coef), ("kl_coef", kl_coef)):
        if isinstance(x, torch.Tensor):
            kept.append(_constant(x, name, (), torch.float32, device))
            scalars.append(nat.Scalar(0.0, x.data_ptr()))
        else:
            scalars.append(nat.Scalar(x, None))
    tensors = (actions.contiguous(), old_log_probs.contiguous(), advantages.contiguous(),
               None if weights is None else weights.contiguous(), mask, reference_logits, reference_log_probs, *kept)
    entries = logits if logits.stride(1) == 1 else logits.detach().contiguous()
    call = _Call(entries, tensors, (1.0 - clip, 1.0 + clip_high, *scalars))
    if torch.is_grad_enabled() and logits.requires_grad:
        loss = PolicyLossFunction.apply(logits, call)
    else:
        loss = call.forward(None)
    return PolicyLoss(loss, call.log_probs, call.entropy, call.kl)
