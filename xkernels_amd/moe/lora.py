"""Public ``lora_projection`` op and its backward: low-rank adapters of many requests at
once beside a shared projection, such as a frozen ``fused_moe_int4_w4a16`` one. The
reference has no counterpart."""
from __future__ import annotations

import torch

from .._backends import Backend
from .._dispatch import dispatch
from .act_checkpoint import ActCheckpoint


def lora_projection(
    x: torch.Tensor,
    lora_a: torch.Tensor,
    lora_b: torch.Tensor,
    adapter_ids: torch.Tensor,
    *,
    base: torch.Tensor | None = None,
    scaling: torch.Tensor | None = None,
    return_hidden: bool = False,
    backend: Backend | str = "auto",
):
    """``out[m] = base[m] + scaling[a] * (x[m] @ lora_a[a].T) @ lora_b[a].T``, ``a =
    adapter_ids[m]``; rows with an id outside ``[0, L)`` get ``base[m]`` (zeros without one).

    ``x [M, K]`` and ``base [M, N]`` (rows may lie apart), ``lora_a [L, r, K]``, ``lora_b
    [L, N, r]``, one dtype (bf16 or fp32); ``scaling [L]`` fp32; up to 1,024 adapters of
    rank up to 128 (adapters of smaller ranks filled up with zeros). ``return_hidden``
    adds ``x[m] @ lora_a[a].T`` (fp32 ``[M, r]``), which the backward takes.
    Rows do not mix: what is not finite in one stays there. No autograd graph is recorded
    (a warning, once, where an input requires a gradient).
    """
    return dispatch("lora_projection", x, lora_a, lora_b, adapter_ids, base=base, scaling=scaling,
                    return_hidden=return_hidden, backend=backend)


def lora_projection_backward(
    grad_out: torch.Tensor,
    x: torch.Tensor | ActCheckpoint,
    lora_a: torch.Tensor,
    lora_b: torch.Tensor,
    adapter_ids: torch.Tensor,
    hidden: torch.Tensor,
    *,
    scaling: torch.Tensor | None = None,
    backend: Backend | str = "auto",
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(grad_x [M, K], grad_a [L, r, K], grad_b [L, N, r])`` of ``lora_projection`` in
    ``grad_out``'s dtype; ``grad_x`` is the adapters' part (zeros for rows without one), and
    adapters without rows get zeros. ``x`` as in the forward, or its ``act_checkpoint``;
    ``hidden`` as the forward returned it. The gradient of ``base`` is ``grad_out``.
    """
    return dispatch("lora_projection_backward", grad_out, x, lora_a, lora_b, adapter_ids, hidden,
                    scaling=scaling, backend=backend)
