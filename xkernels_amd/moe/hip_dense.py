"""HIP backend of the dense block beside the experts: the gated feed-forward block and its
gradients, MXFP4 quantisation and products.

As in ``hip_tuning``: arguments are checked on the host, outputs and scratch are torch
allocations on the tensors' device, the launch goes to torch's current stream of that
device, errors surface as ``RuntimeError`` and CPU tensors are rejected. Nothing
synchronises, so every call may be captured into a HIP graph.
"""
from __future__ import annotations

import torch

from .. import _lib
from .._backends import Backend
from .._dispatch import register
from .hip_backend import _contig, _ptr
from .hip_tuning import _ANY_DT, _bytes, _code, _current_device, _device, _elsewhere, _no_graph, _recording, _rows, \
    _shape, _stream
from .mxfp4_linear import Mxfp4

_FFN_DT = {torch.bfloat16: _lib.XK_DT_BF16, torch.float16: _lib.XK_DT_FP16}
BLOCK = 32
MAX_APART = 2_000_000  # values from row to row that the kernels' offsets hold
LEAST = 2.0 ** -149  # of fp32's positive numbers (a limit of 0 means none)


def _aligned(t: torch.Tensor, n: int = 16) -> torch.Tensor:
    """Contiguous, from an address that the kernels' loads can start at."""
    if not t.is_contiguous():
        return t.contiguous()
    return t if t.data_ptr() % n == 0 else t.clone()


def _aligned_rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``t`` [M, n] as rows of consecutive values that start at 16 bytes (where n is a multiple of 8;
    of other widths the library makes itself such rows), and how far they lie apart."""
    t, ld = _rows(t)
    n = t.shape[1]
    if t.data_ptr() % 16 or (n % 8 == 0 and ld % 8) or ld > max(n, MAX_APART):
        return t.clone(memory_format=torch.contiguous_format), n
    return t, ld


# -------------------------------------------------------------- feed-forward ----

def _ffn_args(op, x, w13, w2, *others):
    if x.dim() != 2 or w13.dim() != 2 or w2.dim() != 2:
        raise RuntimeError(f"{op}: expected x [M, hidden], w13 [2 * ispp, hidden] and w2 [hidden, ispp], got "
                           f"{list(x.shape)}, {list(w13.shape)} and {list(w2.shape)}")
    M, H = x.shape
    I = w2.shape[1]
    _shape(op, "w13", w13, (2 * I, H))
    _shape(op, "w2", w2, (H, I))
    dt = _code(op, x, _FFN_DT)
    for t in (w13, w2, *others):
        if t is not None and t.dtype != x.dtype:
            raise RuntimeError(f"{op}: x is {x.dtype}, another operand {t.dtype}")
    return dt, M, H, I, _aligned(w13), _aligned(w2)


def _limit(op: str, limit: float | None) -> float:
    limit = 0.0 if limit is None else float(limit)
    if limit != limit:
        raise RuntimeError(f"{op}: swiglu_limit is NaN")
    return max(limit, LEAST) if limit > 0 else 0.0


def gated_ffn_hip(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, swiglu_limit: float | None = None,
                  return_gate_up: bool = False):
    op = "gated_ffn"
    i = _device(op, x, w13, w2)
    if i != _current_device():
        return _elsewhere(i, gated_ffn_hip, x, w13, w2, swiglu_limit, return_gate_up)
    if (x.requires_grad or w13.requires_grad or w2.requires_grad) and _recording():
        _no_graph(op)
    dt, M, H, I, w13, w2 = _ffn_args(op, x, w13, w2)
    limit = _limit(op, swiglu_limit)
    xr, ldx = _aligned_rows(x)
    out = x.new_empty((M, H))
    gate_up = x.new_empty((M, 2 * I), dtype=torch.float32) if return_gate_up else None
    nbytes = _bytes("xk_gated_ffn_workspace_bytes", M, H, I)
    ws = x.new_empty(nbytes, dtype=torch.uint8)
    _lib.call("xk_gated_ffn", xr.data_ptr(), dt, ldx, M, H, w13.data_ptr(), w2.data_ptr(), I, limit, out.data_ptr(),
              _ptr(gate_up), ws.data_ptr(), nbytes, _stream(i))
    return (out, gate_up) if return_gate_up else out


def gated_ffn_backward_hip(grad_out: torch.Tensor, x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor,
                           gate_up: torch.Tensor | None = None, swiglu_limit: float | None = None):
    op = "gated_ffn_backward"
    i = _device(op, grad_out, x, w13, w2, gate_up)
    if i != _current_device():
        return _elsewhere(i, gated_ffn_backward_hip, grad_out, x, w13, w2, gate_up, swiglu_limit)
    dt, M, H, I, w13, w2 = _ffn_args(op, x, w13, w2, grad_out)
    _shape(op, "grad_out", grad_out, (M, H))
    _shape(op, "gate_up", gate_up, (M, 2 * I))
    limit = _limit(op, swiglu_limit)
    (gr, ldg), (xr, ldx) = _aligned_rows(grad_out), _aligned_rows(x)
    gu = None if gate_up is None else _contig(gate_up, torch.float32)
    grad_x, grad_w13, grad_w2 = x.new_empty((M, H)), torch.empty_like(w13), torch.empty_like(w2)
    nbytes = _bytes("xk_gated_ffn_backward_workspace_bytes", M, H, I, int(gu is None))
    ws = x.new_empty(nbytes, dtype=torch.uint8)
    _lib.call("xk_gated_ffn_backward", gr.data_ptr(), dt, ldg, xr.data_ptr(), ldx, M, H, w13.data_ptr(),
              w2.data_ptr(), I, _ptr(gu), limit, grad_x.data_ptr(), grad_w13.data_ptr(), grad_w2.data_ptr(),
              ws.data_ptr(), nbytes, _stream(i))
    return grad_x, grad_w13, grad_w2


# --------------------------------------------------------------------- MXFP4 ----

def _check_held(op: str, name: str, held) -> tuple[torch.Tensor, torch.Tensor]:
    c, s = held
    cs, ss = c.shape, s.shape
    if c.dtype != torch.uint8 or s.dtype != torch.uint8 or len(ss) == 0 or cs[:-1] != ss[:-1] or cs[-1] != 16 * ss[-1]:
        raise RuntimeError(f"{op}: {name} must be uint8 codes [..., 16 * blocks] and uint8 scales [..., blocks], got "
                           f"{c.dtype} {list(cs)}, {s.dtype} {list(ss)}")
    return _aligned(c), _aligned(s, 4)


def mxfp4_quantize_hip(x: torch.Tensor) -> Mxfp4:
    op = "mxfp4_quantize"
    i = _device(op, x)
    if i != _current_device():
        return _elsewhere(i, mxfp4_quantize_hip, x)
    if x.requires_grad and _recording():
        _no_graph(op)
    dt = _code(op, x)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise RuntimeError(f"{op}: x must be [..., K], K >= 1, got {list(x.shape)}")
    lead, K = x.shape[:-1], x.shape[-1]
    blocks = -(-K // BLOCK)
    if x.dim() == 2:
        xr, ldx = _rows(x)
    else:
        xr, ldx = x.contiguous(), K
    codes = x.new_empty((*lead, 16 * blocks), dtype=torch.uint8)
    scales = x.new_empty((*lead, blocks), dtype=torch.uint8)
    _lib.call("xk_mxfp4_quantize", xr.data_ptr(), dt, ldx, lead.numel(), K, codes.data_ptr(), scales.data_ptr(),
              _stream(i))
    return Mxfp4(codes, scales)


def mxfp4_dequantize_hip(held: Mxfp4, dtype: torch.dtype = torch.bfloat16, columns: int | None = None) -> torch.Tensor:
    op = "mxfp4_dequantize"
    i = _device(op, *held)
    if i != _current_device():
        return _elsewhere(i, mxfp4_dequantize_hip, held, dtype, columns)
    codes, scales = _check_held(op, "held", held)
    blocks = scales.shape[-1]
    K = blocks * BLOCK if columns is None else int(columns)
    if blocks == 0 or -(-K // BLOCK) != blocks:
        raise RuntimeError(f"{op}: {K} columns in {blocks} blocks of {BLOCK}")
    out = codes.new_empty((*scales.shape[:-1], K), dtype=dtype)
    _lib.call("xk_mxfp4_dequantize", codes.data_ptr(), scales.data_ptr(), scales.shape[:-1].numel(), K,
              _code(op, out), out.data_ptr(), _stream(i))
    return out


def mxfp4_linear_hip(x: torch.Tensor | Mxfp4, weight: Mxfp4, bias: torch.Tensor | None = None,
                     out_dtype: torch.dtype | None = None) -> torch.Tensor:
    op = "mxfp4_linear"
    quantised = isinstance(x, tuple)
    xt, x_scales = x if quantised else (x, None)
    if not isinstance(weight, tuple):
        raise RuntimeError(f"{op}: weight must be an Mxfp4 (codes, scales), got {type(weight).__name__}")
    i = _device(op, xt, x_scales, *weight, bias)
    if i != _current_device():
        return _elsewhere(i, mxfp4_linear_hip, x, weight, bias, out_dtype)
    if (xt.requires_grad or (bias is not None and bias.requires_grad)) and _recording():
        _no_graph(op)
    wc, ws = _check_held(op, "weight", weight)
    if wc.dim() != 2 or xt.dim() != 2:
        raise RuntimeError(f"{op}: expected x [M, K] and a weight [N, K], got {list(xt.shape)} and codes "
                           f"{list(wc.shape)}")
    N, blocks = ws.shape
    if quantised:
        xr, x_scales = _check_held(op, "x", x)
        M, cols, ldx, dt = xr.shape[0], x_scales.shape[1], 0, _lib.XK_DT_NONE
        K = cols * BLOCK
    else:
        dt = _code(op, xt)
        (M, K), (xr, ldx) = xt.shape, _rows(xt)
        cols = -(-K // BLOCK)
    if K == 0 or cols != blocks:
        raise RuntimeError(f"{op}: x has {cols} blocks of {BLOCK} columns, the weight {blocks}")
    if out_dtype is None:
        out_dtype = torch.bfloat16 if quantised else xt.dtype
    out = xr.new_empty((M, N), dtype=out_dtype)
    odt = _code(op, out, _ANY_DT)
    if bias is not None:
        _shape(op, "bias", bias, (N,))
        if bias.dtype != out_dtype:
            raise RuntimeError(f"{op}: bias is {bias.dtype}, the output {out_dtype}")
        bias = bias.contiguous()
    nbytes = _bytes("xk_mxfp4_linear_workspace_bytes", M, K, N)  # 0 for few rows
    scratch = xr.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _lib.call("xk_mxfp4_linear", xr.data_ptr(), dt, ldx, _ptr(x_scales), M, K, wc.data_ptr(), ws.data_ptr(), N,
              _ptr(bias), out.data_ptr(), odt, _ptr(scratch), nbytes, _stream(i))
    return out


def register_all() -> None:
    _lib.load()
    register("gated_ffn", Backend.HIP)(gated_ffn_hip)
    register("gated_ffn_backward", Backend.HIP)(gated_ffn_backward_hip)
    register("mxfp4_quantize", Backend.HIP)(mxfp4_quantize_hip)
    register("mxfp4_dequantize", Backend.HIP)(mxfp4_dequantize_hip)
    register("mxfp4_linear", Backend.HIP)(mxfp4_linear_hip)
