"""MI355X-native fp8_flow_moe operator path (hand-written HIP for gfx950).

Exports the names nanopsyche imports from ``fp8_flow_moe`` (reference
``fp8/__init__.py:8-24``) plus the routing kernels.  All compute runs in
libfm_hip.so; see ``nanopysche_amd.build`` to compile it.
"""

from .recipes import BlockScalingGranularity, FP8RecipeConfig, FP8RecipeType
from .flow_moe import (
    FP8_BLOCK_SIZE,
    ExpertWeights,
    FP8FlowMoECompute,
    FP8FlowMoEConfig,
    FP8SharedExpertCompute,
    FP8Tensor,
    PermutedTokens,
    dequantize_from_fp8,
    fp8_grouped_gemm,
    fused_permute_pad,
    fused_silu_multiply_quantize,
    fused_swiglu_quantize,
    fused_unpermute_unpad,
    quantize_to_fp8,
    scaling_aware_transpose,
)
from .act8 import (Activation8, RMSNormKept, SwigluKept, compress_activation, rmsnorm_8bit, rmsnorm_backward_8bit,
                   rmsnorm_compress, swiglu_8bit, swiglu_backward_8bit, swiglu_compress)
from .balance import BalanceOutput, BalanceState, balance_backward, balance_forward, balance_loss
from .decode import DecodeOutput, expert_decode, moe_decode
from .graph import GraphedStep
from .int8 import (Int8Experts, Int8MoECompute, Int8Tensor, int8_grouped_gemm, int8_linear, int8_matmul,
                   quantize_to_int8)
from .moe_layer import FP8FlowMoELayer
from .norm import NormOutput, RMSNorm, rmsnorm, rmsnorm_backward, rmsnorm_quantize
from .routing import (ExpertLoadTracker, RoutingPlan, expert_counts, load_balancing_loss, route, route_tokens,
                      router_logits, topk_gating)

__all__ = [
    "FP8FlowMoEConfig",
    "FP8FlowMoECompute",
    "FP8SharedExpertCompute",
    "FP8RecipeConfig",
    "FP8RecipeType",
    "BlockScalingGranularity",
    "quantize_to_fp8",
    "dequantize_from_fp8",
    "scaling_aware_transpose",
    "fused_swiglu_quantize",
    "fused_silu_multiply_quantize",
    "fused_permute_pad",
    "fused_unpermute_unpad",
    "fp8_grouped_gemm",
    "FP8_BLOCK_SIZE",
    "FP8Tensor",
    "PermutedTokens",
    "ExpertWeights",
    "RoutingPlan",
    "route_tokens",
    "topk_gating",
    "load_balancing_loss",
    "route",
    "router_logits",
    "expert_counts",
    "ExpertLoadTracker",
    "FP8FlowMoELayer",
    "GraphedStep",
    "moe_decode",
    "quantize_to_int8",
    "int8_matmul",
    "int8_linear",
    "int8_grouped_gemm",
    "Int8Tensor",
    "Int8Experts",
    "Int8MoECompute",
    "expert_decode",
    "DecodeOutput",
    "RMSNorm",
    "rmsnorm",
    "rmsnorm_quantize",
    "rmsnorm_backward",
    "NormOutput",
    "Activation8",
    "compress_activation",
    "SwigluKept",
    "swiglu_compress",
    "swiglu_backward_8bit",
    "swiglu_8bit",
    "RMSNormKept",
    "rmsnorm_compress",
    "rmsnorm_backward_8bit",
    "rmsnorm_8bit",
    "BalanceOutput",
    "BalanceState",
    "balance_forward",
    "balance_backward",
    "balance_loss",
]
