"""Public ``moe_balance_loss`` and ``moe_router_backward`` ops: the training step of the
router whose forward is ``topk_softmax``. The reference has no counterpart."""
from __future__ import annotations

from typing import NamedTuple

import torch

from .._backends import Backend
from .._dispatch import dispatch


class BalanceLoss(NamedTuple):
    """``loss`` fp32 scalar, ``counts`` int32 ``[E]`` (slots per expert), ``tokens`` int32
    scalar (rows that counted)."""

    loss: torch.Tensor
    counts: torch.Tensor
    tokens: torch.Tensor


def moe_balance_loss(
    gating_output: torch.Tensor,
    topk_ids: torch.Tensor,
    *,
    mask: torch.Tensor | None = None,
    backend: Backend | str = "auto",
) -> BalanceLoss:
    """Load-balancing loss and per-expert counts of a routed batch.

    ``loss = E / (T^2 top_k) * sum_e counts[e] * sum_m softmax(gating_output)[m, e]`` over
    the ``T`` rows that ``mask [M]`` (true: counts) leaves; 1 for a perfectly balanced
    router. ``gating_output [M, E]`` bf16, fp16 or fp32; ``topk_ids [M, top_k]`` as
    ``topk_softmax`` gives them (ids outside ``[0, E)`` count nowhere). Deterministic. No
    autograd graph is recorded (a warning, once, where the logits require a gradient).
    """
    return dispatch("moe_balance_loss", gating_output, topk_ids, mask=mask, backend=backend)


def moe_router_backward(
    gating_output: torch.Tensor,
    topk_ids: torch.Tensor,
    *,
    grad_weights: torch.Tensor | None = None,
    renormalize: bool = True,
    grad_loss: torch.Tensor | None = None,
    counts: torch.Tensor | None = None,
    tokens: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    backend: Backend | str = "auto",
) -> torch.Tensor:
    """Gradient of the logits ``[M, E]`` (in their dtype) in one pass, from ``grad_weights
    [M, top_k]`` (of ``topk_softmax``'s weights, called with the same ``renormalize``),
    ``grad_loss`` (of ``moe_balance_loss``, with its ``counts`` and ``tokens``, or sums of
    them over parts of a batch, int32; the counts are constants) or both. Rows that ``mask``
    leaves out get zeros.
    """
    return dispatch("moe_router_backward", gating_output, topk_ids, grad_weights=grad_weights,
                    renormalize=renormalize, grad_loss=grad_loss, counts=counts, tokens=tokens, mask=mask,
                    backend=backend)
