"""Device ops around the trunk: sampling a wave's actions (the reference's cardgym.rl helpers that run
per wave) and the policy loss of an update."""

from .policy import PolicyLoss, policy_loss
from .sampling import masked_probabilities, sample_rows

__all__ = ["PolicyLoss", "masked_probabilities", "policy_loss", "sample_rows"]
