"""MXFP4 (microscaled 4-bit floating point) on gfx950: quantization, the linear
layer and the fused MoE.  No counterpart in the reference."""

from .ops import (fused_mxfp4_moe, mxfp4_dequantize, mxfp4_linear, mxfp4_matmul, mxfp4_quantize)

__all__ = ["fused_mxfp4_moe", "mxfp4_dequantize", "mxfp4_linear", "mxfp4_matmul", "mxfp4_quantize"]
