"""spanqr_amd: spanqr's orth(X) -- a robust shifted Cholesky-QR for tall fp32 matrices -- on AMD MI355X (gfx950).

    from orth import orth          # drop-in, as in the reference (orth.py)
    Q = orth(X)                    # X: fp32 GPU [K, r] -> Q: fp32 [K, r], Q^T Q = I, span(Q) = span(X)

The hot path is hand-written HIP in csrc/spanqr.hip behind the C ABI of include/spanqr.h, loaded with ctypes. Beside it
stand the operators of the training step that calls orth: the loss over the vocabulary (csrc/loss.hip), the
root-mean-square norm (csrc/norm.hip) and clipping by the global norm (csrc/clip.hip).
"""
from .clip import clip_grad_norm, grad_norm  # noqa: F401
from .kcholqr import borth, kcholqr_f, kcholqr_f_many, orth, orth_many, set_checked, status  # noqa: F401
from .loss import linear_cross_entropy, linear_cross_entropy_grad  # noqa: F401
from .norm import rms_norm, rms_norm_backward  # noqa: F401
from .plan import clear_plans, get_plan  # noqa: F401

__all__ = ["orth", "orth_many", "kcholqr_f", "kcholqr_f_many", "borth", "get_plan", "clear_plans", "set_checked",
           "status", "linear_cross_entropy", "linear_cross_entropy_grad", "rms_norm", "rms_norm_backward", "grad_norm",
           "clip_grad_norm"]
