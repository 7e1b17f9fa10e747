"""Quantized fused-MoE ops on gfx950: router (topk_softmax) -> align -> INT4 / MXFP4
grouped GEMM -> combine; and for tuning and serving over them the router's training
step, low-rank adapters and 8-bit activation checkpoints; and the dense gated
feed-forward block beside them, with MXFP4 quantisation and products.

The HIP backend registers inside ``backend_registration_guard``: if the native
library is missing the failure is recorded (``backend_diagnostics()``) and any
call raises — there is no CPU fallback in this package.
"""
from .._backends import Backend
from .._dispatch import backend_registration_guard
from .act_checkpoint import ActCheckpoint, act_checkpoint, act_restore
from .align import moe_align_block_size
from .balance_loss import BalanceLoss, moe_balance_loss, moe_router_backward
from .gated_ffn import gated_ffn, gated_ffn_backward
from .interface import fused_moe_int4_w4a16
from .lora import lora_projection, lora_projection_backward
from .mxfp4_interface import fused_moe_mxfp4
from .mxfp4_linear import Mxfp4, mxfp4_dequantize, mxfp4_linear, mxfp4_quantize
from .sum_reduce import moe_sum_reduce
from .topk_softmax import topk_softmax
from .weights import make_mxfp4_moe_weights, make_w4a16_weights
from .workspace import MoeAlignWorkspace, MoeInt4Workspace, MoeMxfp4Workspace

_KERNELS = ("moe_align_block_size", "moe_sum_reduce", "moe_int4_w4a16", "moe_mxfp4", "topk_softmax")

with backend_registration_guard(_KERNELS, Backend.HIP, source="xkernels_amd.moe.hip_backend"):
    from . import hip_backend

    hip_backend.register_all()

_TUNING = ("moe_balance_loss", "moe_router_backward", "lora_projection", "lora_projection_backward",
           "act_checkpoint", "act_restore")

with backend_registration_guard(_TUNING, Backend.HIP, source="xkernels_amd.moe.hip_tuning"):
    from . import hip_tuning

    hip_tuning.register_all()

_DENSE = ("gated_ffn", "gated_ffn_backward", "mxfp4_quantize", "mxfp4_dequantize", "mxfp4_linear")

with backend_registration_guard(_DENSE, Backend.HIP, source="xkernels_amd.moe.hip_dense"):
    from . import hip_dense

    hip_dense.register_all()

__all__ = [
    "fused_moe_int4_w4a16",
    "fused_moe_mxfp4",
    "moe_align_block_size",
    "moe_sum_reduce",
    "topk_softmax",
    "BalanceLoss",
    "moe_balance_loss",
    "moe_router_backward",
    "lora_projection",
    "lora_projection_backward",
    "ActCheckpoint",
    "act_checkpoint",
    "act_restore",
    "gated_ffn",
    "gated_ffn_backward",
    "Mxfp4",
    "mxfp4_quantize",
    "mxfp4_dequantize",
    "mxfp4_linear",
    "make_w4a16_weights",
    "make_mxfp4_moe_weights",
    "MoeAlignWorkspace",
    "MoeInt4Workspace",
    "MoeMxfp4Workspace",
]
