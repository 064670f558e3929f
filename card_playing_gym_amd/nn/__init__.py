"""The cardgym.nn API of the KV-cached self-play trunk step, on MI355X kernels."""

from .kv_cache import KVCache
from .model import SequenceModel, value_mlp
from .optim import AdamW, AdamWPlan, grad_norm, moment_values
from .trunk import DecoderBlock, RMSNorm, Trunk, TrunkConfig, init_weights

__all__ = [
    "AdamW",
    "AdamWPlan",
    "DecoderBlock",
    "KVCache",
    "RMSNorm",
    "SequenceModel",
    "Trunk",
    "TrunkConfig",
    "grad_norm",
    "init_weights",
    "moment_values",
    "value_mlp",
]
