"""Quantized linear layer on the packed MTC GEMM (drop-in for mtc.nn), the
full-precision layer that callers compare it with, and the layers on 8-bit
weights (linear, mixture of experts)."""
from .layers import ExpertsFP8, LinearFP8, LinearFP32, LinearMTCAdaptive

__all__ = ["LinearMTCAdaptive", "LinearFP32", "LinearFP8", "ExpertsFP8"]
