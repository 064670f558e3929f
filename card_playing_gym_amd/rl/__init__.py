"""Device ops around the trunk: sampling a wave's actions (the reference's cardgym.rl helpers that run
per wave, and sampling under controls), the record of a policy's top entries, and the losses of an update."""

from .choose import Sample, TopLogits, sample_logits, top_logits
from .distill import DistillLoss, distill_loss
from .policy import PolicyLoss, policy_loss
from .sampling import masked_probabilities, sample_rows

__all__ = ["DistillLoss", "PolicyLoss", "Sample", "TopLogits", "distill_loss", "masked_probabilities", "policy_loss",
           "sample_logits", "sample_rows", "top_logits"]
