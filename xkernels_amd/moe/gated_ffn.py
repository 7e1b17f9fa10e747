"""Public ``gated_ffn`` op and its backward: the dense gated feed-forward block (a shared
expert, or a layer without routed ones) in 16 bits. The reference has no counterpart;
weights are laid out and clamped as ``fused_moe_mxfp4`` has them."""
from __future__ import annotations

import torch

from .._backends import Backend
from .._dispatch import dispatch


def gated_ffn(
    x: torch.Tensor,
    w13: torch.Tensor,
    w2: torch.Tensor,
    *,
    swiglu_limit: float | None = None,
    return_gate_up: bool = False,
    backend: Backend | str = "auto",
):
    """``out = (silu(min(g, L)) * clamp(u, -L, L)) @ w2.T`` with ``g, u`` the halves of ``x @
    w13.T`` and ``L = swiglu_limit`` (None or <= 0: no clamp).

    ``x [M, hidden]`` (rows may lie apart), ``w13 [2 * ispp, hidden]`` (rows ``[gate; up]``),
    ``w2 [hidden, ispp]``, one dtype (bf16 or fp16); ``out [M, hidden]`` of it. fp32 sums; the
    activations between the projections are rounded to the dtype (up to 8 tokens are held as two
    values of it, so a token's last bits depend on whether its call has more). In fp16 an
    activation past 65,504 becomes an infinity, which a ``swiglu_limit`` of up to 255 rules out.
    ``return_gate_up`` adds ``[M, 2 * ispp]`` in fp32, the sums ``g`` and ``u``, which spare the
    backward their product. Rows do not mix: what is not finite in one stays there. No autograd
    graph is recorded (a warning, once, where an input requires a gradient).
    """
    return dispatch("gated_ffn", x, w13, w2, swiglu_limit=swiglu_limit, return_gate_up=return_gate_up,
                    backend=backend)


def gated_ffn_backward(
    grad_out: torch.Tensor,
    x: torch.Tensor,
    w13: torch.Tensor,
    w2: torch.Tensor,
    gate_up: torch.Tensor | None = None,
    *,
    swiglu_limit: float | None = None,
    backend: Backend | str = "auto",
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(grad_x [M, hidden], grad_w13 [2 * ispp, hidden], grad_w2 [hidden, ispp])`` of
    ``gated_ffn`` for ``grad_out [M, hidden]``, in its dtype; ``gate_up`` as the forward
    returned it, else it is computed again. The clamps pass the gradient where ``g <= L``
    and ``|u| <= L``. fp32 sums; the activations and the gradients of ``g`` and ``u`` are rounded
    to the dtype between the products: in fp16 they become infinities past 65,504, lose bits
    below 6e-5 and are 0 below 3e-8, so a loss is scaled as for any training in fp16. Rows of
    an ``x`` that was held in 8 bits come from ``act_restore``.
    """
    return dispatch("gated_ffn_backward", grad_out, x, w13, w2, gate_up, swiglu_limit=swiglu_limit,
                    backend=backend)
