"""PyTorch-tensor front end of the fused MXFP4 MoE layer and of the dense feed-forward beside it (tensors only at the
boundary; the work happens behind the C ABI of ``libvkernels_b200.so``)."""
from ._dispatch import OpNotEligible, require, same_gpu_contiguous
from .dense import fused_linear, fused_linear_backward, gated_linear, gated_linear_backward, require_apart
from .moe_fused_mxfp4 import (SITU, SWIGLU, align_em_bound, fused_moe_mxfp4, fused_moe_mxfp4_bf16_into, fused_moe_mxfp4_into,
                              fused_moe_mxfp4_rows_into, PrepackedWeights, prepack_weights,
                              fused_moe_mxfp4_bf16_prepacked_into,
                              kernel_status, moe_act_epilogue, moe_align_block_size, moe_combine,
                              moe_down_preact, moe_gateup_preact, mxfp4_dequant_rows, reserve_workspace,
                              reset_kernel_status, route_align_small, route_topk, router_logits, set_impl)

__all__ = ["OpNotEligible", "require", "same_gpu_contiguous", "SITU", "SWIGLU", "fused_linear", "fused_linear_backward",
           "gated_linear", "gated_linear_backward", "require_apart", "align_em_bound", "fused_moe_mxfp4",
           "fused_moe_mxfp4_bf16_into", "fused_moe_mxfp4_into", "fused_moe_mxfp4_rows_into", "PrepackedWeights", "prepack_weights",
           "fused_moe_mxfp4_bf16_prepacked_into", "kernel_status", "moe_act_epilogue",
           "moe_align_block_size", "moe_combine", "moe_down_preact", "moe_gateup_preact",
           "mxfp4_dequant_rows", "reserve_workspace", "reset_kernel_status", "route_align_small", "route_topk", "router_logits",
           "set_impl"]
