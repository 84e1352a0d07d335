"""tda_b200: B200-native (sm_100a) Threshold (Differential) Attention (forward and backward).

Drop-in for the public API of snap-research/TDA's ``triton_threshold_attention``
module; see ``tda_b200.triton_threshold_attention`` for the same module name.
"""
from . import torch_ops  # noqa: F401  (registers the tda:: torch operators)
from .ops import (  # noqa: F401
    DifferentialThresholdRelaFunction,
    ThresholdRelaFunction,
    check_status,
    diff_forward,
    differential_threshold_rela_triton,
    rect_backward,
    rect_forward,
    threshold_rela_triton,
)
from .cache4 import (  # noqa: F401
    Cache4,
    PagePlan,
    cache4_append,
    cache4_read,
    cache4_softmax_attention,
    cache4_threshold_attention,
    plan_pages,
)
from .sdiff import (  # noqa: F401
    DifferentialSoftmaxFunction,
    differential_softmax_attention,
    sdiff_backward,
    sdiff_forward,
)

__all__ = [
    "threshold_rela_triton",
    "differential_threshold_rela_triton",
    "ThresholdRelaFunction",
    "DifferentialThresholdRelaFunction",
    "rect_forward",
    "rect_backward",
    "diff_forward",
    "check_status",
    "differential_softmax_attention",
    "DifferentialSoftmaxFunction",
    "sdiff_forward",
    "sdiff_backward",
    "Cache4",
    "PagePlan",
    "plan_pages",
    "cache4_append",
    "cache4_read",
    "cache4_softmax_attention",
    "cache4_threshold_attention",
]
