"""The distillation loss of an update on the device: a policy is trained towards another's top entries, as
``top_logits`` recorded them, forward and gradient in one pass (csrc/distill.hip).

    record = top_logits(teacher_logits, 64, mask=legal, temperature=2.0)
    out = distill_loss(logits, record.indices, record.log_probs, log_rest=record.log_rest, mask=legal, temperature=2.0)
    (policy.loss + out.loss).backward()

A record of k entries takes 12 k + 4 bytes a row where the logits would take 2 or 4 bytes for every entry.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _native as nat
from ..nn.kv_cache import stream_handle
from ..nn.optim import _on
from .choose import MAX_TOP, _policy_rows
from .policy import _constant, _no_tangents


class DistillLoss(NamedTuple):
    """``loss``: the scalar to differentiate.  ``kl``: each row's, for logging, float32 and without a gradient."""

    loss: torch.Tensor
    kl: torch.Tensor


class _Call:
    """One loss: its native descriptor, and what the forward writes beside the loss."""

    __slots__ = ("descriptor", "kl")

    def __init__(self, tensors, rows: nat.PolicyRows, temperature: float, normalizer: float) -> None:
        self.descriptor = nat.DistillLoss(rows, None, None, None, None, tensors[2].shape[1], temperature,
                                          nat.Scalar(normalizer, None))
        self.bind(tensors)

    def bind(self, tensors) -> None:
        """Points the descriptor at the inputs."""

        logits, mask, indices, log_probs, log_rest, weights, normalizer = tensors
        d = self.descriptor
        d.rows.logits, d.rows.ld_logits = logits.data_ptr(), logits.stride(0)
        if mask is not None:
            d.rows.mask, d.rows.ld_mask = mask.data_ptr(), mask.stride(0)
        d.indices, d.log_probs = indices.data_ptr(), log_probs.data_ptr()
        if log_rest is not None:
            d.log_rest = log_rest.data_ptr()
        if weights is not None:
            d.weights = weights.data_ptr()
        if normalizer is not None:
            d.normalizer.device = normalizer.data_ptr()

    def forward(self, device: torch.device, grad: torch.Tensor | None) -> torch.Tensor:
        loss = torch.empty((), device=device)
        self.kl = torch.empty(self.descriptor.rows.rows, device=device)
        size = nat.lib().cg_distill_loss_workspace_size(self.descriptor)
        workspace = torch.empty(size, device=device, dtype=torch.uint8)
        with _on(device):
            nat.call("cg_distill_loss_forward", self.descriptor, loss.data_ptr(), self.kl.data_ptr(),
                     None if grad is None else grad.data_ptr(), workspace.data_ptr(), size, stream_handle(device))
        return loss


class DistillLossFunction(torch.autograd.Function):
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
        if torch.is_grad_enabled():
            raise RuntimeError("distill_loss is differentiable once: its gradient has no graph")
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
        with _on(device):
            nat.call("cg_distill_loss_backward", call.descriptor, upstream.data_ptr(), int(written), grad.data_ptr(),
                     stream_handle(device))
        return grad, None, None


@torch.compiler.disable
def distill_loss(
    logits: torch.Tensor,
    indices: torch.Tensor,
    log_probs: torch.Tensor,
    *,
    log_rest: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    weights: torch.Tensor | None = None,
    normalizer: float | torch.Tensor | None = None,
    temperature: float = 1.0,
) -> DistillLoss:
    """sum_i weights_i KL_i / normalizer over the rows of ``logits`` [rows, width] (float32, bfloat16 or
    float16; up to 2^18 entries), differentiable in the logits (once, backwards; forward-mode tangents are refused).

    p is the softmax of logits / ``temperature`` over a row's legal entries: those that ``mask`` (bool [rows,
    width]) keeps and whose logit is above -inf.  The record R of a row is ``indices`` (int64 [rows, k], k up
    to 256) and the logs of the teacher's probabilities ``log_probs`` (float32 [rows, k]).

    With ``log_rest`` (float32 [rows], the log of what the teacher has outside R), as ``top_logits`` returns it:

        KL = sum_R q (log q - log p) + q_rest (log q_rest - log p_rest),  p_rest: p's mass outside R

    Without, q is made to sum to 1 over R and KL = sum_R q (log q - log p); the teacher's logits / temperature
    will then do for ``log_probs``.

    ``weights``: float32 [rows] (ones).  ``normalizer``: the number of rows, padding among them; pass the count of
    those with weight (1 at least: nothing over 0 is NaN) for their mean.  It may be a float32 device scalar, which a
    captured loss reads at every replay.  A factor of the loss belongs in it too (n / 0.1 for a tenth): the forward
    writes the gradient for an arriving 1, and for another one, as ``0.1 * out.loss`` sends, the backward forms it again.
    A backward captured in a graph of its own follows one replay of its forward's each time.

    Index -1 stands for no entry.  An index outside the row, or twice in it, makes its row, and the loss, NaN, as does
    a legal entry that is NaN or +inf.  An entry with a q above 0 that is not legal here makes its row's KL infinite, as
    does a ``log_rest`` above -inf where nothing outside the record is legal; the gradient stays finite.

    A row of weight 0 (padding) is not read: like a row without a legal entry, whatever its record, it adds nothing, has a
    zero gradient and reports 0.  So does, without ``log_rest``, a row whose record is empty or has no q above 0, whatever
    its logits are; an index outside the row, or twice in it, still makes it NaN."""

    descriptor, (entries, mask) = _policy_rows(logits, mask)
    _no_tangents(logits, log_probs, log_rest, weights, normalizer, name="distill_loss")
    rows, device = descriptor.rows, logits.device
    if indices.dim() != 2 or not 1 <= indices.shape[1] <= MAX_TOP:
        raise ValueError(f"indices must be [rows, k] with k from 1 to {MAX_TOP}")
    record = (rows, indices.shape[1])
    _constant(indices, "indices", record, torch.int64, device)
    _constant(log_probs, "log_probs", record, torch.float32, device)
    if log_rest is not None:
        log_rest = _constant(log_rest, "log_rest", (rows,), torch.float32, device).contiguous()
    if weights is not None:
        weights = _constant(weights, "weights", (rows,), torch.float32, device).contiguous()
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError("temperature must be from 1e-30 to 1e30")
    value = float(max(rows, 1)) if normalizer is None else 1.0
    if isinstance(normalizer, torch.Tensor):
        _constant(normalizer, "normalizer", (), torch.float32, device)
    elif normalizer is not None:
        if not normalizer > 0:
            raise ValueError("normalizer must be positive")
        value, normalizer = normalizer, None
    tensors = (entries, mask, indices.contiguous(), log_probs.contiguous(), log_rest, weights, normalizer)
    call = _Call(tensors, descriptor, temperature, value)
    if torch.is_grad_enabled() and logits.requires_grad:
        loss = DistillLossFunction.apply(logits, call, tensors)
    else:
        loss = call.forward(device, None)
    return DistillLoss(loss, call.kl)
