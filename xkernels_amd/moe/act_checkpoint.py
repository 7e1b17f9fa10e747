"""Public ``act_checkpoint`` and ``act_restore`` ops: activations held in 8 bits for a
backward pass. The reference has no counterpart; the format is MXFP8's (as the MXFP4
experts': blocks of 32 along a row with one e8m0 scale)."""
from __future__ import annotations

from typing import NamedTuple

import torch

from .._backends import Backend
from .._dispatch import dispatch


class ActCheckpoint(NamedTuple):
    """``values`` float8_e4m3fn ``[M, K]``, ``scales`` uint8 e8m0 ``[M, ceil(K / 32)]``:
    value = e4m3 * 2^(byte - 127)."""

    values: torch.Tensor
    scales: torch.Tensor


def act_checkpoint(x: torch.Tensor, *, backend: Backend | str = "auto") -> ActCheckpoint:
    """``x [M, K]`` (bf16, fp16 or fp32) in 8 bits. A block's scale is the least power of two
    with which none of its finite values passes 448; values round to nearest even, off by at
    most 2^-4 of themselves or, the small ones, 2^-17 of the block's largest (2^-137 where
    that largest is below 2^-119: the least scale). Infinities
    and NaN become NaN. No autograd graph is recorded (a warning, once, where ``x`` requires
    a gradient)."""
    return dispatch("act_checkpoint", x, backend=backend)


def act_restore(held: ActCheckpoint, dtype: torch.dtype = torch.bfloat16, *,
                backend: Backend | str = "auto") -> torch.Tensor:
    """The values of a checkpoint in ``dtype`` (bf16, fp16 or fp32)."""
    return dispatch("act_restore", held, dtype, backend=backend)
