"""mxfp8gg — MXFP8 grouped GEMM for AMD MI355X (gfx950).

bf16 -> MXFP8 casts, a forward grouped GEMM and a weight-gradient grouped GEMM
over ragged expert groups, the expert FFN's fused SwiGLU casts, the token
routing (decision, dispatch plan, gather, combine), norms, the loss of a linear
layer over a vocabulary and the optimizer step around them, products of e4m3
operands in blocks of 128, log probabilities of tokens and gradient clipping, all
as hand-written HIP kernels in libmxgg.so behind a C ABI (include/mxgg.h).  This
package is the host side: it takes torch tensors, allocates outputs, and calls the library on
the current stream.
"""
from ._lib import MxggError, load as load_library
from .ops import (
    GroupEnds,
    _best_config,
    fused_grouped_fwd,
    fwd_ge,
    grouped_dgrad,
    grouped_mm,
    grouped_mm_swiglu_quant,
    grouped_wgrad,
    offs_to_group_ends,
    padded_token_capacity,
    quant_weight_dual,
    quant_weight_for_dgrad,
    swiglu_backward_quant,
    swiglu_quant,
    to_mxfp8_dim0,
    to_mxfp8_dim1,
    to_mxfp8_dual,
    wgrad_fused,
    wgrad_kernel,
    wgrad_prepare,
    zero_rows_past_groups,
)
from .weight_cache import WeightCastCache
from .autograd import (
    MXFP8ExpertFFN,
    MXFP8GroupedMM,
    MXFP8RoutedExpertFFN,
    moe_ffn,
    moe_ffn_unfused,
    moe_routed_ffn,
    mxfp8_grouped_mm,
)
from .routing import (
    RoutePlan,
    RouteTopK,
    combine,
    combine_score_grad,
    gather_rows,
    gather_to_mxfp8_dual,
    gather_to_mxfp8_dim0,
    route_plan,
    route_topk,
)
from .block import (
    FP8BlockLinear,
    fp8_block_linear,
    fp8_block_mm,
    fp8_block_wgrad,
    to_fp8_block_dim0,
    to_fp8_block_dim1,
    to_fp8_block_weight,
)
from .loss import LinearCrossEntropy, linear_cross_entropy
from .logprob import TokenLogProbs, token_log_probs
from .optim import AdamW, adamw_state, adamw_step, clip_grad_norm_, grad_norm
from .norm import AddRMSNorm, Norm, add_rms_norm, layer_norm, rms_norm, rms_norm_quant
from .torchao_compat import (
    apply,
    triton_mxfp8_grouped_mm,
    triton_mxfp8_wgrad,
    triton_mxfp8_wgrad_v2,
    triton_to_mxfp8_dim0,
    triton_to_mxfp8_dim1,
)

__all__ = [
    "MxggError", "load_library",
    "to_mxfp8_dim0", "to_mxfp8_dim1", "to_mxfp8_dual", "padded_token_capacity",
    "grouped_mm", "grouped_mm_swiglu_quant", "grouped_wgrad", "grouped_dgrad", "quant_weight_for_dgrad",
    "quant_weight_dual", "swiglu_quant", "swiglu_backward_quant",
    "fused_grouped_fwd", "fwd_ge", "wgrad_fused", "wgrad_prepare", "wgrad_kernel",
    "offs_to_group_ends", "zero_rows_past_groups", "GroupEnds",
    "triton_to_mxfp8_dim0", "triton_to_mxfp8_dim1",
    "triton_mxfp8_grouped_mm", "triton_mxfp8_wgrad", "triton_mxfp8_wgrad_v2", "apply",
    "WeightCastCache",
    "MXFP8GroupedMM", "mxfp8_grouped_mm", "MXFP8ExpertFFN", "moe_ffn", "moe_ffn_unfused",
    "route_topk", "RouteTopK", "RoutePlan", "route_plan", "gather_rows", "gather_to_mxfp8_dual", "gather_to_mxfp8_dim0",
    "combine",
    "combine_score_grad", "Norm", "layer_norm", "rms_norm", "add_rms_norm", "AddRMSNorm", "rms_norm_quant",
    "grad_norm", "clip_grad_norm_", "token_log_probs", "TokenLogProbs",
    "to_fp8_block_dim0", "to_fp8_block_dim1", "to_fp8_block_weight", "fp8_block_mm", "fp8_block_wgrad",
    "fp8_block_linear", "FP8BlockLinear",
    "LinearCrossEntropy", "linear_cross_entropy", "AdamW", "adamw_state", "adamw_step", "MXFP8RoutedExpertFFN", "moe_routed_ffn",
]
