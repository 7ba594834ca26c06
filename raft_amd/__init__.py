"""raft_amd -- MI355X-native correlation hot path of RAFT (drop-in for core/corr.py), and the encoders' norm and the optimizer
step that run around it in training."""
from .corr import CorrBlock, AlternateCorrBlock   # noqa: F401
from . import alt_cuda_corr                                          # noqa: F401
from .norm import GroupNorm, group_norm                              # noqa: F401
from .adamw import AdamW                                             # noqa: F401

__all__ = ["CorrBlock", "AlternateCorrBlock", "alt_cuda_corr", "GroupNorm", "group_norm", "AdamW"]
