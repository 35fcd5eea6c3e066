"""atomic_gdn2 (B200) -- Gated DeltaNet-2 operator on hand-written sm_100a kernels.

Drop-in for the reference package's public API (atomic_gdn2/__init__.py:1-10):
    BLRConfig, make_cfg, PROD, make_blr_trainable
and the serving operators: make_blr_recurrent (single tokens, any length), pack_w4 / quantize_w4 /
w4_linear (products with 4-bit weights), beam_select (one step of beam search); gated_scan, the diagonal
gated linear recurrence, and linear, the differentiable product with bias, GELU and residual in its epilogue.
"""
from .config import BLRConfig, make_cfg, PROD
from .pipeline import make_blr_trainable, set_checks, last_status
from .recurrent import make_blr_recurrent
from .w4 import W4Weight, pack_w4, quantize_w4, w4_linear
from .beam import beam_select
from .gated import gated_scan
from .linear import linear

__version__ = "0.1.0"
__all__ = ["BLRConfig", "make_cfg", "PROD", "make_blr_trainable", "set_checks", "last_status",
           "make_blr_recurrent", "W4Weight", "pack_w4", "quantize_w4", "w4_linear", "beam_select",
           "gated_scan", "linear"]
