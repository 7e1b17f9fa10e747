"""Public ``mxfp4_quantize``, ``mxfp4_dequantize`` and ``mxfp4_linear`` ops: 16- and 32-bit
values to the MXFP4 format of ``fused_moe_mxfp4``'s weights, back, and the product of
two quantised operands. The reference has no counterpart (its MXFP4 weights come
quantised)."""
from __future__ import annotations

from typing import NamedTuple

import torch

from .._backends import Backend
from .._dispatch import dispatch


class Mxfp4(NamedTuple):
    """``codes`` uint8 ``[..., 16 * ceil(K / 32)]`` (e2m1 pairs, low half = even k, the last
    block of a row filled up with zeros), ``scales`` uint8 e8m0 ``[..., ceil(K / 32)]``:
    value = e2m1 * 2^(byte - 127), byte 255 NaN. Where K is a multiple of 32 these are a
    weight and its scales as ``fused_moe_mxfp4`` takes them (which reads byte 255 as 0)."""

    codes: torch.Tensor
    scales: torch.Tensor


def mxfp4_quantize(x: torch.Tensor, *, backend: Backend | str = "auto") -> Mxfp4:
    """``x [..., K]`` (bf16, fp16 or fp32) in 4 bits. A block's scale is the least power of two
    with which none of its values passes 6; values round to nearest even, off by at most a fifth of
    themselves or, below the scale, a quarter of it. A block with an infinity or a NaN becomes
    NaN. K is at most 2^22, a call has fewer than 2^33 values. No autograd graph is recorded (a
    warning, once, where ``x`` requires a gradient)."""
    return dispatch("mxfp4_quantize", x, backend=backend)


def mxfp4_dequantize(held: Mxfp4, dtype: torch.dtype = torch.bfloat16, *, columns: int | None = None,
                     backend: Backend | str = "auto") -> torch.Tensor:
    """The values in ``dtype`` (bf16, fp16 or fp32), ``[..., K]``; ``columns`` gives a K that is
    no multiple of 32. What would pass the type's largest finite value becomes that."""
    return dispatch("mxfp4_dequantize", held, dtype, columns=columns, backend=backend)


def mxfp4_linear(
    x: torch.Tensor | Mxfp4,
    weight: Mxfp4,
    *,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    backend: Backend | str = "auto",
) -> torch.Tensor:
    """``out [M, N] = q(x) @ weight.T + bias`` in fp32 sums, rounded once.

    ``weight`` is ``mxfp4_quantize`` of ``[N, K]``; ``x [M, K]`` (bf16, fp16 or fp32, rows may
    lie apart) is quantised the same way in the call, or comes quantised. ``out_dtype`` bf16,
    fp16 or fp32 (default: ``x``'s, bf16 for a quantised one); ``bias [N]`` of that type. No
    autograd graph is recorded (a warning, once, where an input requires a gradient).
    """
    return dispatch("mxfp4_linear", x, weight, bias=bias, out_dtype=out_dtype, backend=backend)
