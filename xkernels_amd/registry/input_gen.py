"""Seeded input generators for ``verify`` / ``verify_parity``, one per Op Spec.

Recipes follow the reference's registry/input_gen.py:68-159 (same seeds per
tensor, same distributions) so the same (point, seed, device) gives the same
inputs; ``moe_mxfp4`` has no generator upstream and gets one here. The
``topk_softmax`` logits are N(0, 1) in the point's dtype (:203-215).
"""
from __future__ import annotations

from collections.abc import Callable
from typing import Any

import torch

from .dtypes import to_torch_dtype


def _randn(device: str, dtype: torch.dtype, *shape: int, seed: int) -> torch.Tensor:
    g = torch.Generator(device=device).manual_seed(int(seed))
    return torch.randn(*shape, generator=g, device=device, dtype=dtype)


def _moe_sum_reduce(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    dt = to_torch_dtype(p["dtype"])
    y = _randn(device, dt, p["M"], p["top_k"], p["H"], seed=seed)
    w = _randn(device, torch.float32, p["M"], p["top_k"], seed=seed + 1)
    return {"y": y, "w": w, "routed_scaling_factor": 1.0}


def _moe_align_block_size(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    g = torch.Generator(device=device).manual_seed(int(seed))
    E = int(p["num_experts"])
    ids = torch.randint(0, E, (int(p["M"]), int(p["top_k"])), generator=g, device=device,
                        dtype=torch.int32)
    return {"topk_ids": ids, "block_size": int(p["block_size"]), "num_experts": E,
            "truncate": bool(p.get("truncate", True))}


def _moe_int4_w4a16(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    from ..moe.weights import make_w4a16_weights

    dt = to_torch_dtype(p["dtype"])
    M, K, N, E, k = (int(p[x]) for x in ("M", "K", "N", "E", "top_k"))
    gs = int(p.get("group_size", 32))
    A = _randn(device, dt, M, K, seed=seed)
    packed, scale, _ = make_w4a16_weights(E, N, K, gs, device=device, seed=seed + 1)
    g = torch.Generator(device=device).manual_seed(seed + 2)
    ids = torch.randint(0, E, (M, k), generator=g, device=device, dtype=torch.int32)
    w = torch.rand(M, k, generator=g, device=device, dtype=torch.float32)
    return {"A": A, "packed": packed, "scale": scale, "topk_ids": ids, "topk_w": w,
            "group_size": gs, "mul_routed_weight": True}


def _moe_mxfp4(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    from ..moe.weights import make_mxfp4_moe_weights

    dt = to_torch_dtype(p["dtype"])
    M, E, k = int(p["M"]), int(p["E"]), int(p["top_k"])
    hidden, ispp = int(p["hidden"]), int(p["ispp"])
    bias = bool(p.get("bias", False))
    A = _randn(device, dt, M, hidden, seed=seed)
    if "a_scale" in p:  # optional input scale of a sweep point
        A = (A.float() * float(p["a_scale"])).to(dt)
    sc = {k: int(p[k]) for k in ("scale_lo", "scale_hi") if k in p}  # e8m0 bytes [lo, hi)
    wts = make_mxfp4_moe_weights(E, hidden, ispp, with_bias=bias, device=device, seed=seed + 1, **sc)
    g = torch.Generator(device=device).manual_seed(seed + 2)
    ids = torch.stack([torch.randperm(E, generator=g, device=device)[:k] for _ in range(M)]).to(torch.int32)
    logits = torch.randn(M, k, generator=g, device=device, dtype=torch.float32)
    return {"A": A, "w13": wts["w13"], "w13_scale": wts["w13_scale"], "w2": wts["w2"],
            "w2_scale": wts["w2_scale"], "topk_ids": ids, "topk_w": torch.softmax(logits, -1),
            "b13": wts["b13"], "b2": wts["b2"], "swiglu_limit": float(p.get("swiglu_limit", 10.0))}


def _topk_softmax(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    dt = to_torch_dtype(p["dtype"])
    gating = _randn(device, dt, int(p["M"]), int(p["E"]), seed=seed)
    return {"gating_output": gating, "topk": int(p["topk"]), "renormalize": bool(p["renormalize"])}


def _moe_balance_loss(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    z = _randn(device, torch.float32, p["M"], p["E"], seed=seed).to(to_torch_dtype(p["dtype"]))
    g = torch.Generator(device=device).manual_seed(seed + 1)
    mask = torch.rand(int(p["M"]), generator=g, device=device) >= p["padded"] if p["padded"] else None
    return {"gating_output": z, "topk_ids": torch.topk(z.float(), int(p["top_k"]), dim=1).indices.int(), "mask": mask}


def _moe_router_backward(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    a = _moe_balance_loss({**p, "padded": 0.0}, seed, device)
    ids = a["topk_ids"]
    return {"gating_output": a["gating_output"], "topk_ids": ids,
            "grad_weights": _randn(device, torch.float32, *ids.shape, seed=seed + 2),
            "renormalize": bool(p["renormalize"]), "grad_loss": torch.ones((), device=device),
            "counts": torch.bincount(ids.flatten().long(), minlength=int(p["E"])).int()}


def _lora_projection(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    dt = to_torch_dtype(p["dtype"])
    M, K, N, L, r = (int(p[x]) for x in ("M", "K", "N", "L", "r"))
    g = torch.Generator(device=device).manual_seed(seed + 3)
    return {"x": _randn(device, torch.float32, M, K, seed=seed).to(dt),
            "lora_a": (_randn(device, torch.float32, L, r, K, seed=seed + 1) / K ** 0.5).to(dt),
            "lora_b": (_randn(device, torch.float32, L, N, r, seed=seed + 2) / r ** 0.5).to(dt),
            "adapter_ids": torch.randint(-1, L, (M,), generator=g, device=device, dtype=torch.int32),
            "base": _randn(device, torch.float32, M, N, seed=seed + 4).to(dt),
            "scaling": torch.rand(L, generator=g, device=device) + 0.5}


def _lora_projection_backward(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    f = _lora_projection(p, seed, device)
    hidden = _randn(device, torch.float32, int(p["M"]), int(p["r"]), seed=seed + 5)
    x = _held(f["x"]) if p.get("held") else f["x"]
    return {"grad_out": f["base"], "x": x, "lora_a": f["lora_a"], "lora_b": f["lora_b"],
            "adapter_ids": f["adapter_ids"], "hidden": hidden, "scaling": f["scaling"]}


def _held(x: torch.Tensor):
    """Any valid checkpoint: the values' own e4m3 rounding with scales of 1."""
    from ..moe.act_checkpoint import ActCheckpoint

    scales = torch.full((x.shape[0], -(-x.shape[1] // 32)), 127, dtype=torch.uint8, device=x.device)
    return ActCheckpoint(x.to(torch.float8_e4m3fn), scales)


def _act_checkpoint(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    return {"x": (8 * _randn(device, torch.float32, int(p["M"]), int(p["K"]), seed=seed)).to(to_torch_dtype(p["dtype"]))}


def _act_restore(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    x = _randn(device, torch.float32, int(p["M"]), int(p["K"]), seed=seed)
    return {"held": _held(x), "dtype": to_torch_dtype(p["dtype"])}


def _gated_ffn(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    dt = to_torch_dtype(p["dtype"])
    M, H, I = (int(p[x]) for x in ("M", "hidden", "ispp"))
    return {"x": _randn(device, torch.float32, M, H, seed=seed).to(dt),
            "w13": (_randn(device, torch.float32, 2 * I, H, seed=seed + 1) / H ** 0.5).to(dt),
            "w2": (_randn(device, torch.float32, H, I, seed=seed + 2) / I ** 0.5).to(dt),
            "swiglu_limit": float(p["limit"]) if p.get("limit") else None}


def _gated_ffn_backward(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    f = _gated_ffn(p, seed, device)
    M, dt = int(p["M"]), f["x"].dtype
    gate_up = _randn(device, torch.float32, M, f["w13"].shape[0], seed=seed + 4) if p.get("kept") else None
    grad = _randn(device, torch.float32, M, f["x"].shape[1], seed=seed + 3).to(dt)
    return {"grad_out": grad, "x": f["x"], "w13": f["w13"], "w2": f["w2"], "gate_up": gate_up,
            "swiglu_limit": f["swiglu_limit"]}


def _mxfp4(rows: int, K: int, seed: int, device: str):
    """Any valid codes, with scales about 1."""
    from ..moe.mxfp4_linear import Mxfp4

    g = torch.Generator(device=device).manual_seed(seed)
    nb = -(-K // 32)
    return Mxfp4(torch.randint(0, 256, (rows, 16 * nb), generator=g, device=device, dtype=torch.uint8),
                 torch.randint(124, 129, (rows, nb), generator=g, device=device, dtype=torch.uint8))


def _mxfp4_dequantize(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    return {"held": _mxfp4(int(p["M"]), int(p["K"]), seed, device), "dtype": to_torch_dtype(p["dtype"])}


def _mxfp4_linear(p: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    dt = to_torch_dtype(p["dtype"])
    M, K, N = (int(p[x]) for x in ("M", "K", "N"))
    bias = _randn(device, torch.float32, N, seed=seed + 2).to(dt) if p.get("bias") else None
    return {"x": (_randn(device, torch.float32, M, K, seed=seed) / K ** 0.5).to(dt),
            "weight": _mxfp4(N, K, seed + 1, device), "bias": bias}


_GENERATORS: dict[str, Callable[[dict, int, str], dict[str, Any]]] = {
    "moe_sum_reduce@1.0.0": _moe_sum_reduce,
    "moe_align_block_size@1.0.0": _moe_align_block_size,
    "moe_int4_w4a16@1.0.0": _moe_int4_w4a16,
    "moe_mxfp4@1.0.0": _moe_mxfp4,
    "topk_softmax@1.0.0": _topk_softmax,
    "moe_balance_loss@1.0.0": _moe_balance_loss,
    "moe_router_backward@1.0.0": _moe_router_backward,
    "lora_projection@1.0.0": _lora_projection,
    "lora_projection_backward@1.0.0": _lora_projection_backward,
    "act_checkpoint@1.0.0": _act_checkpoint,
    "act_restore@1.0.0": _act_restore,
    "gated_ffn@1.0.0": _gated_ffn,
    "gated_ffn_backward@1.0.0": _gated_ffn_backward,
    "mxfp4_quantize@1.0.0": _act_checkpoint,
    "mxfp4_dequantize@1.0.0": _mxfp4_dequantize,
    "mxfp4_linear@1.0.0": _mxfp4_linear,
}


def has_generator(op_id: str) -> bool:
    return op_id in _GENERATORS


def register_input_gen(op_id: str, fn) -> None:
    _GENERATORS[op_id] = fn


def generate_inputs(op_id: str, point: dict[str, Any], seed: int, device: str) -> dict[str, Any]:
    if op_id not in _GENERATORS:
        raise KeyError(f"no input generator for {op_id!r}; have {sorted(_GENERATORS)}")
    return _GENERATORS[op_id](point, seed, device)


def supported_op_ids() -> list[str]:
    return sorted(_GENERATORS)
