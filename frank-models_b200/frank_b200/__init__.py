"""frank_b200: B200-native (sm_100a) MoE FFN hot path of frank-models.

Public surface
  B200Module            reference-shaped module: mul_mat_id / moe_ffn_block / swiglu
  MoEFFNBlock           weights packed once, reusable workspace (serving/bench path)
  Fp8MoEFFNBlock        the block with 8-bit weights (Fp8Experts), its sub-layer with norms on both sides
  fp8_matmul, quantize_fp8, rms_norm_fp8, post_norm_residual
                        the 8-bit path's operators (include/frank_fp8.h)
  ops.*                 typed torch wrappers over the C ABI (include/frank_moe.h)
"""

from . import _lib, fp8, ops  # noqa: F401
from .fp8 import (Fp8Experts, Fp8MoEFFNBlock, fp8_matmul, post_norm_residual, quantize_fp8,  # noqa: F401
                  rms_norm_fp8)
from .module import B200Module  # noqa: F401
from .ops import MoEFFNBlock, PackedExperts  # noqa: F401

__all__ = ["B200Module", "Fp8Experts", "Fp8MoEFFNBlock", "MoEFFNBlock", "PackedExperts", "fp8", "fp8_matmul", "ops",
           "post_norm_residual", "quantize_fp8", "rms_norm_fp8"]
