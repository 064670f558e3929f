"""The policy loss of an update on the device: the clipped objective with an entropy bonus and a
KL term over rows of policy logits, forward and gradient in one pass (csrc/loss.hip).

It scores what :func:`~card_playing_gym_amd.rl.masked_probabilities` and ``sample_rows`` chose in the
rollout (cardgym/rl/ppo.py:75-94): the same softmax over a row's legal entries, differentiable.

    out = policy_loss(logits, actions, old_log_probs, advantages, mask=legal, entropy_coef=0.01)
    (out.loss + value_loss).backward()
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad

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


def _no_tangents(*tensors, name: str = "policy_loss") -> None:
    """Refuses forward-mode derivatives, which nothing behind this would carry on.  (Outside a level no tensor has
    one: asking each would be 6 us of a small loss's 96.)"""

    if getattr(forward_ad, "_current_level", 0) >= 0:
        if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
            raise RuntimeError(f"{name} has no forward-mode derivative: pass the inputs without tangents")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Entries of a row side by side; rows at any stride."""

    return t if t.stride(-1) == 1 else t.contiguous()


class _Call:
    """One loss: its native descriptor, and what the forward writes beside the loss."""

    __slots__ = ("descriptor", "kl", "log_probs", "entropy")

    def __init__(self, tensors, options) -> None:
        rows, width = tensors[0].shape
        self.descriptor = nat.PolicyLoss(*(8 * (None,)), 0, 0, 0, rows, width, dtype_code(tensors[0].dtype), *options)
        self.bind(tensors)

    def bind(self, tensors) -> None:
        """Points the descriptor at the inputs: logits, mask, reference logits, then the rows' and scalars."""

        logits, mask, reference_logits, actions, old, advantages, weights, reference_log_probs, *scalars = tensors
        d = self.descriptor
        d.logits, d.ld_logits = logits.data_ptr(), logits.stride(0)
        d.actions, d.old_log_probs, d.advantages = actions.data_ptr(), old.data_ptr(), advantages.data_ptr()
        if mask is not None:
            d.mask, d.ld_mask = mask.data_ptr(), mask.stride(0)
        if reference_logits is not None:
            d.reference_logits, d.ld_reference = reference_logits.data_ptr(), reference_logits.stride(0)
        if weights is not None:
            d.weights = weights.data_ptr()
        if reference_log_probs is not None:
            d.reference_log_probs = reference_log_probs.data_ptr()
        for name, x in zip(("normalizer", "entropy_coef", "kl_coef"), scalars):
            if x is not None:
                getattr(d, name).device = x.data_ptr()

    def forward(self, device: torch.device, grad: torch.Tensor | None) -> torch.Tensor:
        d = self.descriptor
        loss = torch.empty((), device=device)
        self.log_probs = torch.empty(d.rows, device=device)
        self.entropy = torch.empty(d.rows, device=device)
        self.kl = torch.empty(d.rows, device=device) if d.reference_logits or d.reference_log_probs else None
        size = nat.lib().cg_policy_loss_workspace_size(d)
        workspace = torch.empty(size, device=device, dtype=torch.uint8)
        with _on(device):
            nat.call(
                "cg_policy_loss_forward", d, loss.data_ptr(), self.log_probs.data_ptr(), self.entropy.data_ptr(),
                None if self.kl is None else self.kl.data_ptr(), None if grad is None else grad.data_ptr(),
                workspace.data_ptr(), size, stream_handle(device),
            )
        return loss


class PolicyLossFunction(torch.autograd.Function):
    """The forward writes the gradient of the loss itself; the backward keeps it where the gradient
    arriving is 1 and forms it again, from the inputs, where it is another."""

    @staticmethod
    def forward(ctx, logits, call, tensors):
        # (tensors[0] is what the kernel reads: logits, or its copy with the entries side by side)
        ctx.written = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
        ctx.save_for_backward(*tensors)
        ctx.call = call
        ctx.capturing = torch.cuda.is_current_stream_capturing()
        return call.forward(logits.device, ctx.written)

    @staticmethod
    def backward(ctx, upstream):
        if torch.is_grad_enabled():  # (create_graph; once_differentiable costs 13 us of a small loss's 96)
            raise RuntimeError("policy_loss is differentiable once: its gradient has no graph")
        tensors = ctx.saved_tensors  # (an input changed since the forward raises here)
        call, logits, device = ctx.call, tensors[0], upstream.device
        call.bind(tensors)  # (a saved-tensor hook may have brought them back elsewhere)
        grad, ctx.written = ctx.written, None  # handed over once: a second backward forms its own
        if torch.cuda.is_current_stream_capturing() != ctx.capturing:
            grad = None  # a replay of one alone would find, or leave, what the other's buffer holds by then
        written = grad is not None
        if grad is None:
            grad = torch.empty(logits.shape, device=device, dtype=logits.dtype)
        upstream = upstream.contiguous()
        size = nat.lib().cg_policy_loss_backward_workspace_size(call.descriptor)
        workspace = torch.empty(size, device=device, dtype=torch.uint8) if size else None
        with _on(device):
            nat.call("cg_policy_loss_backward", call.descriptor, upstream.data_ptr(), int(written), grad.data_ptr(),
                     workspace.data_ptr() if size else None, size, stream_handle(device))
        return grad, None, None


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
    or float16), differentiable in the logits (once, backwards; forward-mode tangents are refused), with

        r = exp(log p[action] - old_log_prob)
        l = -min(r A, clamp(r, 1 - clip, 1 + clip_high) A) + kl_coef KL - entropy_coef H

    p is the softmax over the row's legal entries: those that ``mask`` (bool [rows, width]) keeps
    and whose logit is above -inf.  KL is sum p (log p - log q) with ``reference_logits`` (of the logits'
    type; q over the same mask), or exp(d) - d - 1 with d = ``reference_log_probs`` - log p[action].

    ``actions``: int64 [rows].  ``old_log_probs``, ``advantages``, ``weights`` (ones) and
    ``reference_log_probs``: float32 [rows].  ``normalizer``: the number of rows, padding among them; pass the
    count of those with weight for their mean, the whole minibatch's where a microbatch's gradients are accumulated.  ``clip_high``: ``clip``.
    ``normalizer`` and the coefficients may be float32 device scalars, which a captured loss reads at
    every replay.  A backward captured in a graph of its own follows one replay of its forward's each time.

    A row of weight 0 (padding) is not read: like a row without a legal entry it adds nothing, has a
    zero gradient and reports zeros.  An action outside the row makes its row, and the loss, NaN; one that
    is not legal has log p = -inf.  With a ``kl_coef`` of 0 a reference is reported only, whatever it holds."""

    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError("logits must be [rows, width] with at least one entry a row")
    require_device(logits)
    dtype_code(logits.dtype)
    _no_tangents(logits, old_log_probs, advantages, weights, normalizer, entropy_coef, kl_coef, reference_logits,
                 reference_log_probs)
    rows, width = logits.shape
    if rows >= 2**31 or width > 2**30:  # (the descriptor's 32 bits would keep their lower ones)
        raise ValueError("logits may have up to 2^31 - 1 rows of up to 2^30 entries")
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
    values, scalars = [], []
    for name, x in (("normalizer", normalizer), ("entropy_coef", entropy_coef), ("kl_coef", kl_coef)):
        on_device = isinstance(x, torch.Tensor)
        scalars.append(_constant(x, name, (), torch.float32, device) if on_device else None)
        values.append(nat.Scalar(0.0 if on_device else x, None))
    entries = logits if logits.stride(1) == 1 else logits.detach().contiguous()
    tensors = (entries, mask, reference_logits, actions.contiguous(), old_log_probs.contiguous(), advantages.contiguous(),
               None if weights is None else weights.contiguous(), reference_log_probs, *scalars)
    call = _Call(tensors, (1.0 - clip, 1.0 + clip_high, *values))
    if torch.is_grad_enabled() and logits.requires_grad:
        loss = PolicyLossFunction.apply(logits, call, tensors)
    else:
        loss = call.forward(device, None)
    return PolicyLoss(loss, call.log_probs, call.entropy, call.kl)
