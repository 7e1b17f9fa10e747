"""HIP backend of the ops for tuning and serving over the frozen experts: the
router's training step, low-rank adapters and 8-bit activation checkpoints.

As in ``hip_backend``: arguments are checked on the host, outputs and scratch are
torch allocations on the tensors' device, the launch goes to torch's current stream
of that device, errors surface as ``RuntimeError`` and CPU tensors are rejected.
Nothing synchronises, so every call may be captured into a HIP graph.
"""
from __future__ import annotations

import warnings
from functools import lru_cache

import torch

from .. import _lib
from .._backends import Backend
from .._dispatch import register
from .act_checkpoint import ActCheckpoint
from .balance_loss import BalanceLoss
from .hip_backend import _contig, _need_gpu, _ptr, _raw_stream

_LORA_DT = {torch.bfloat16: _lib.XK_DT_BF16, torch.float32: _lib.XK_DT_FP32}
_ANY_DT = {**_LORA_DT, torch.float16: _lib.XK_DT_FP16}
BLOCK = 32

# the current device's number without torch.cuda's lazy-initialisation checks (the
# tensors at hand are on a device), where this torch has the call
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _device(op: str, first: torch.Tensor, *others: torch.Tensor | None) -> int:
    """The number of the device that all of them are on."""
    i = first.get_device()
    if i < 0:
        _need_gpu(op, first)
    for t in others:
        if t is not None and t.get_device() != i:
            _need_gpu(op, first, t)
    return i


_told: set[str] = set()
_recording = torch.is_grad_enabled


def _no_graph(op: str) -> None:
    """Says, once an op, that a call which autograd would be expected to record (``_recording``, and
    an input requires a gradient) is not. Under no_grad, and in the forward of an
    autograd.Function, which runs without it, there is nothing to say."""
    if op not in _told:
        _told.add(op)
        warnings.warn(f"{op} records no autograd graph: its result carries no gradient to inputs that require one. "
                      "Call it and its backward in a torch.autograd.Function, or under torch.no_grad() if none is "
                      "wanted", RuntimeWarning, stacklevel=5)


def _stream(i: int) -> int:
    return _raw_stream(i) if _raw_stream is not None else torch.cuda.current_stream(i).cuda_stream


def _elsewhere(i: int, fn, *args):
    """``fn(*args)`` with device ``i``, which its tensors are on, as the current one: HIP
    launches on a stream need it."""
    with torch.cuda.device(i):
        return fn(*args)


def _code(op: str, t: torch.Tensor, table=_ANY_DT) -> int:
    dt = table.get(t.dtype)
    if dt is None:
        names = ", ".join(str(d).removeprefix("torch.") for d in table)
        raise RuntimeError(f"{op}: unsupported dtype {t.dtype} ({names})")
    return dt


@lru_cache(maxsize=4096)
def _bytes(query: str, *sizes: int) -> int:
    """A workspace's size, a function of the call's sizes alone."""
    return _lib.query(query, *sizes)


def _ids(op: str, t: torch.Tensor, n: int) -> torch.Tensor:
    """int32, contiguous; 64-bit ids outside [0, n) stay outside."""
    if t.dtype == torch.int32:
        return t if t.is_contiguous() else t.contiguous()
    if t.dtype == torch.int64:
        t = t.clamp(-1, n)
    elif t.dtype not in (torch.int16, torch.int8, torch.uint8):
        raise RuntimeError(f"{op}: ids must be whole numbers, got {t.dtype}")
    return _contig(t, torch.int32)


def _shape(op: str, name: str, t: torch.Tensor | None, want: tuple) -> None:
    if t is not None and t.shape != want:
        raise RuntimeError(f"{op}: {name} must be {list(want)}, got {list(t.shape)}")


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``t`` [M, n] as rows of consecutive values, and how far they lie apart."""
    M, n = t.shape
    if t.is_contiguous():
        return t, n
    if M > 1 and (n == 1 or t.stride(1) == 1) and t.stride(0) >= n:
        return t, t.stride(0)
    return t.contiguous(), n


# ------------------------------------------------------------------- router ----

def _router_args(op, gating_output, topk_ids, mask):
    if gating_output.dim() != 2 or topk_ids.dim() != 2 or topk_ids.shape[0] != gating_output.shape[0]:
        raise RuntimeError(f"{op}: expected gating_output [M, E] and topk_ids [M, top_k], got "
                           f"{list(gating_output.shape)} and {list(topk_ids.shape)}")
    M, E = gating_output.shape
    k = topk_ids.shape[1]
    if not 1 <= k <= E:
        raise RuntimeError(f"{op}: top_k={k} outside [1, E={E}]")
    if mask is not None:
        _shape(op, "mask", mask, (M,))
        mask = _contig(mask if mask.dtype == torch.bool else mask != 0).view(torch.uint8)
    return M, E, k, gating_output.contiguous(), _ids(op, topk_ids, E), mask


def moe_balance_loss_hip(gating_output: torch.Tensor, topk_ids: torch.Tensor,
                         mask: torch.Tensor | None = None) -> BalanceLoss:
    op = "moe_balance_loss"
    i = _device(op, gating_output, topk_ids, mask)
    if i != _current_device():
        return _elsewhere(i, moe_balance_loss_hip, gating_output, topk_ids, mask)
    if gating_output.requires_grad and _recording():
        _no_graph(op)
    dt = _code(op, gating_output)
    M, E, k, g, ids, on = _router_args(op, gating_output, topk_ids, mask)
    loss = g.new_empty((), dtype=torch.float32)
    counts = g.new_empty(E, dtype=torch.int32)
    tokens = g.new_empty((), dtype=torch.int32)
    nbytes = _bytes("xk_moe_balance_loss_workspace_bytes", M, E)  # 0 for small batches
    ws = g.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _lib.call("xk_moe_balance_loss", g.data_ptr(), dt, M, E, ids.data_ptr(), k, _ptr(on), loss.data_ptr(),
              counts.data_ptr(), tokens.data_ptr(), _ptr(ws), nbytes, _stream(i))
    return BalanceLoss(loss, counts, tokens)


def moe_router_backward_hip(gating_output: torch.Tensor, topk_ids: torch.Tensor,
                            grad_weights: torch.Tensor | None = None, renormalize: bool = True,
                            grad_loss: torch.Tensor | None = None, counts: torch.Tensor | None = None,
                            tokens: torch.Tensor | None = None,
                            mask: torch.Tensor | None = None) -> torch.Tensor:
    op = "moe_router_backward"
    i = _device(op, gating_output, topk_ids, grad_weights, grad_loss, counts, tokens, mask)
    if i != _current_device():
        return _elsewhere(i, moe_router_backward_hip, gating_output, topk_ids, grad_weights, renormalize, grad_loss,
                          counts, tokens, mask)
    dt = _code(op, gating_output)
    M, E, k, g, ids, on = _router_args(op, gating_output, topk_ids, mask)
    if grad_weights is None and grad_loss is None:
        raise RuntimeError(f"{op}: neither grad_weights nor grad_loss")
    _shape(op, "grad_weights", grad_weights, (M, k))
    gw = None if grad_weights is None else _contig(grad_weights, torch.float32)
    gl = cn = tk = None
    if grad_loss is not None:
        if counts is None:
            raise RuntimeError(f"{op}: grad_loss needs the counts of moe_balance_loss")
        if tokens is None and mask is not None:
            raise RuntimeError(f"{op}: with a mask, grad_loss needs the tokens of moe_balance_loss")
        _shape(op, "counts", counts, (E,))
        if grad_loss.numel() != 1 or (tokens is not None and tokens.numel() != 1):
            raise RuntimeError(f"{op}: grad_loss and tokens are single numbers")
        gl, cn = _contig(grad_loss, torch.float32), _contig(counts, torch.int32)
        tk = None if tokens is None else _contig(tokens, torch.int32)
    grad = torch.empty_like(g)
    _lib.call("xk_moe_router_backward", g.data_ptr(), dt, M, E, ids.data_ptr(), k, _ptr(on), _ptr(gl), _ptr(cn),
              _ptr(tk), _ptr(gw), int(bool(renormalize)), grad.data_ptr(), _stream(i))
    return grad


# ----------------------------------------------------------------- adapters ----

def _lora_args(op, M, name, cols, axis, lora_a, lora_b, adapter_ids, scaling):
    """Checks the adapters against ``cols`` columns of ``name`` (axis 0: K, 1: N)."""
    if lora_a.dim() != 3 or lora_b.dim() != 3:
        raise RuntimeError(f"{op}: expected lora_a [L, r, K] and lora_b [L, N, r]")
    L, r, K = lora_a.shape
    N = lora_b.shape[1]
    _shape(op, "lora_b", lora_b, (L, N, r))
    _shape(op, "adapter_ids", adapter_ids, (M,))
    _shape(op, "scaling", scaling, (L,))
    if lora_a.dtype != lora_b.dtype:
        raise RuntimeError(f"{op}: lora_a is {lora_a.dtype}, lora_b {lora_b.dtype}")
    if cols != (N if axis else K):
        raise RuntimeError(f"{op}: {name} has {cols} columns, the adapters {N if axis else K}")
    sc = None if scaling is None else _contig(scaling, torch.float32)
    return L, r, K, N, lora_a.contiguous(), lora_b.contiguous(), _ids(op, adapter_ids, L), sc


def lora_projection_hip(x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, adapter_ids: torch.Tensor,
                        base: torch.Tensor | None = None, scaling: torch.Tensor | None = None,
                        return_hidden: bool = False):
    op = "lora_projection"
    i = _device(op, x, lora_a, lora_b, adapter_ids, base, scaling)
    if i != _current_device():
        return _elsewhere(i, lora_projection_hip, x, lora_a, lora_b, adapter_ids, base, scaling, return_hidden)
    if (x.requires_grad or lora_a.requires_grad or lora_b.requires_grad
            or (base is not None and base.requires_grad)) and _recording():
        _no_graph(op)
    dt = _code(op, x, _LORA_DT)
    if x.dim() != 2:
        raise RuntimeError(f"{op}: x must be [M, K], got {list(x.shape)}")
    M, cols = x.shape
    L, r, K, N, a, b, ids, sc = _lora_args(op, M, "x", cols, 0, lora_a, lora_b, adapter_ids, scaling)
    if a.dtype != x.dtype or (base is not None and base.dtype != x.dtype):
        raise RuntimeError(f"{op}: x is {x.dtype}, the adapters {a.dtype}, base {None if base is None else base.dtype}")
    xr, ldx = _rows(x)
    br, ldb = None, N
    if base is not None:
        _shape(op, "base", base, (M, N))
        br, ldb = _rows(base)
    out = x.new_empty((M, N))
    hidden = x.new_empty((M, r), dtype=torch.float32) if return_hidden else None
    nbytes = _bytes("xk_lora_projection_workspace_bytes", M, K, L, r)
    ws = x.new_empty(nbytes, dtype=torch.uint8)
    _lib.call("xk_lora_projection", xr.data_ptr(), dt, ldx, M, K, a.data_ptr(), b.data_ptr(), L, N, r, ids.data_ptr(),
              _ptr(sc), _ptr(br), ldb, out.data_ptr(), _ptr(hidden), ws.data_ptr(), nbytes, _stream(i))
    return (out, hidden) if return_hidden else out


def lora_projection_backward_hip(grad_out: torch.Tensor, x: torch.Tensor | ActCheckpoint, lora_a: torch.Tensor,
                                 lora_b: torch.Tensor, adapter_ids: torch.Tensor, hidden: torch.Tensor,
                                 scaling: torch.Tensor | None = None):
    op = "lora_projection_backward"
    held = isinstance(x, tuple)
    xt, scales = x if held else (x, None)
    i = _device(op, grad_out, xt, scales, lora_a, lora_b, adapter_ids, hidden, scaling)
    if i != _current_device():
        return _elsewhere(i, lora_projection_backward_hip, grad_out, x, lora_a, lora_b, adapter_ids, hidden, scaling)
    dt = _code(op, grad_out, _LORA_DT)
    if grad_out.dim() != 2:
        raise RuntimeError(f"{op}: grad_out must be [M, N], got {list(grad_out.shape)}")
    M, cols = grad_out.shape
    L, r, K, N, a, b, ids, sc = _lora_args(op, M, "grad_out", cols, 1, lora_a, lora_b, adapter_ids, scaling)
    _shape(op, "x", xt, (M, K))
    _shape(op, "hidden", hidden, (M, r))
    if a.dtype != grad_out.dtype or (not held and x.dtype != grad_out.dtype):
        raise RuntimeError(f"{op}: grad_out is {grad_out.dtype}, the adapters {a.dtype}, x {xt.dtype}")
    if held:
        (xr, sr), ldx = _check_held(op, x), K
    else:
        (xr, ldx), sr = _rows(x), None
    gr, ldg = _rows(grad_out)
    h = _contig(hidden, torch.float32)
    grad_x = grad_out.new_empty((M, K))
    grad_a, grad_b = torch.empty_like(a), torch.empty_like(b)
    nbytes = _bytes("xk_lora_projection_backward_workspace_bytes", M, K, N, L, r, dt)
    ws = grad_out.new_empty(nbytes, dtype=torch.uint8)
    _lib.call("xk_lora_projection_backward", gr.data_ptr(), dt, ldg, xr.data_ptr(), ldx, _ptr(sr), M, K, a.data_ptr(),
              b.data_ptr(), L, N, r, ids.data_ptr(), _ptr(sc), h.data_ptr(), grad_x.data_ptr(), grad_a.data_ptr(),
              grad_b.data_ptr(), ws.data_ptr(), nbytes, _stream(i))
    return grad_x, grad_a, grad_b


# -------------------------------------------------------------- checkpoints ----

def _check_held(op: str, held) -> tuple[torch.Tensor, torch.Tensor]:
    v, s = held
    if v.dim() != 2 or v.dtype != torch.float8_e4m3fn or s.dtype != torch.uint8:
        raise RuntimeError(f"{op}: a checkpoint is float8_e4m3fn [M, K] with uint8 scales, got {v.dtype} "
                           f"{list(v.shape)}, {s.dtype}")
    _shape(op, "scales", s, (v.shape[0], -(-v.shape[1] // BLOCK)))
    return v.contiguous(), s.contiguous()


def act_checkpoint_hip(x: torch.Tensor) -> ActCheckpoint:
    op = "act_checkpoint"
    i = _device(op, x)
    if i != _current_device():
        return _elsewhere(i, act_checkpoint_hip, x)
    if x.requires_grad and _recording():
        _no_graph(op)
    dt = _code(op, x)
    if x.dim() != 2 or x.shape[1] == 0:
        raise RuntimeError(f"{op}: x must be [M, K], K >= 1, got {list(x.shape)}")
    M, K = x.shape
    xr, ldx = _rows(x)
    values = x.new_empty((M, K), dtype=torch.float8_e4m3fn)
    scales = x.new_empty((M, -(-K // BLOCK)), dtype=torch.uint8)
    _lib.call("xk_act_checkpoint", xr.data_ptr(), dt, ldx, M, K, values.data_ptr(), scales.data_ptr(), _stream(i))
    return ActCheckpoint(values, scales)


def act_restore_hip(held: ActCheckpoint, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    op = "act_restore"
    i = _device(op, *held)
    if i != _current_device():
        return _elsewhere(i, act_restore_hip, held, dtype)
    v, s = _check_held(op, held)
    M, K = v.shape
    if K == 0:
        raise RuntimeError(f"{op}: no columns")
    out = v.new_empty((M, K), dtype=dtype)
    _lib.call("xk_act_restore", v.data_ptr(), s.data_ptr(), M, K, _code(op, out), out.data_ptr(), _stream(i))
    return out


def register_all() -> None:
    _lib.load()
    register("moe_balance_loss", Backend.HIP)(moe_balance_loss_hip)
    register("moe_router_backward", Backend.HIP)(moe_router_backward_hip)
    register("lora_projection", Backend.HIP)(lora_projection_hip)
    register("lora_projection_backward", Backend.HIP)(lora_projection_backward_hip)
    register("act_checkpoint", Backend.HIP)(act_checkpoint_hip)
    register("act_restore", Backend.HIP)(act_restore_hip)
