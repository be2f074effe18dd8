"""Utility modules (GroupSum, GroupNorm, Dropout), sampling from logits, and warning helpers."""

from .dropout import Dropout, dropout
from .modules import GroupSum
from .normalization import GroupNorm, group_norm
from .sampling import sample_logits
from .warnings import (
    ConfigurationWarning,
    CUDAWarning,
    DefaultValueWarning,
    DiffLUTWarning,
    PerformanceWarning,
    configure_warnings,
    disable_all_warnings,
    disable_cuda_warnings,
    enable_all_warnings,
    enable_strict_mode,
    suppress_warnings,
    warn_default_value,
)
