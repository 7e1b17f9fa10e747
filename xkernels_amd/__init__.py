"""xkernels_amd — MI355X (gfx950) native quantized fused-MoE path of xkernels.

Public ops (same names and signatures as ``xkernels``):
``fused_moe_int4_w4a16``, ``fused_moe_mxfp4``, ``moe_align_block_size``,
``moe_sum_reduce``, ``topk_softmax``; without a counterpart there, for tuning and
serving over the frozen experts: ``moe_balance_loss``, ``moe_router_backward``,
``lora_projection``, ``lora_projection_backward``, ``act_checkpoint``,
``act_restore``; harness: ``find_impl``, ``verify``, ``verify_parity``,
``backend_diagnostics``. The ops run hand-written HIP kernels from
``libxk_moe.so``; they raise if the library is missing or the tensors are not on
the GPU.
"""
from . import registry
from ._backends import Backend
from ._dispatch import backend_diagnostics
from .moe import (
    ActCheckpoint,
    BalanceLoss,
    MoeAlignWorkspace,
    MoeInt4Workspace,
    MoeMxfp4Workspace,
    act_checkpoint,
    act_restore,
    fused_moe_int4_w4a16,
    fused_moe_mxfp4,
    lora_projection,
    lora_projection_backward,
    make_mxfp4_moe_weights,
    make_w4a16_weights,
    moe_align_block_size,
    moe_balance_loss,
    moe_router_backward,
    moe_sum_reduce,
    topk_softmax,
)
from .retrieval import find_impl
from .verify import verify, verify_parity

__version__ = "0.1.0"
__all__ = [
    "Backend", "backend_diagnostics", "registry", "fused_moe_int4_w4a16", "fused_moe_mxfp4",
    "moe_align_block_size", "moe_sum_reduce", "topk_softmax", "make_w4a16_weights", "make_mxfp4_moe_weights",
    "moe_balance_loss", "moe_router_backward", "BalanceLoss", "lora_projection", "lora_projection_backward",
    "act_checkpoint", "act_restore", "ActCheckpoint",
    "MoeAlignWorkspace", "MoeInt4Workspace", "MoeMxfp4Workspace", "find_impl", "verify",
    "verify_parity", "__version__",
]
