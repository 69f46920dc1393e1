from .fused import LARS, FusedAdam, FusedSGD, default_no_decay
from .lr_scheduler import StepLR, WarmupCosineLR, WarmupPolyLR
from .muon import Muon

__all__ = ["FusedSGD", "LARS", "FusedAdam", "Muon", "default_no_decay", "StepLR", "WarmupPolyLR", "WarmupCosineLR"]
