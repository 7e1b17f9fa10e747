"""Plain torch (fp32) forms of the dense block's ops: the REFERENCE backend that the test
harness registers for them. TEST INFRASTRUCTURE, as the rest of this package. Written from
the ops' definitions (the reference has no counterpart); pinned by tests/test_dense_host.py
against 64-bit forms and autograd."""
from __future__ import annotations

import torch

BLOCK = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _clamped(gu, I, limit):
    g, u = gu[:, :I], gu[:, I:]
    if limit is None or limit <= 0:
        return g, u, torch.ones_like(g), torch.ones_like(u)
    return g.clamp(max=limit), u.clamp(-limit, limit), (g <= limit).float(), (u.abs() <= limit).float()


def gated_ffn_ref(x, w13, w2, swiglu_limit=None, return_gate_up=False):
    gu = x.float() @ w13.float().t()
    g, u, _, _ = _clamped(gu, w2.shape[1], swiglu_limit)
    out = ((g * torch.sigmoid(g) * u) @ w2.float().t()).to(x.dtype)
    return (out, gu) if return_gate_up else out


def gated_ffn_backward_ref(grad_out, x, w13, w2, gate_up=None, swiglu_limit=None):
    dt = x.dtype
    dy, x, w13, w2 = (t.float() for t in (grad_out, x, w13, w2))
    gu = x @ w13.t() if gate_up is None else gate_up.float()
    g, u, on_g, on_u = _clamped(gu, w2.shape[1], swiglu_limit)
    s = torch.sigmoid(g)
    dh = dy @ w2
    d = torch.cat((dh * u * s * (1 + g * (1 - s)) * on_g, dh * g * s * on_u), 1)
    return (d @ w13).to(dt), (d.t() @ x).to(dt), (dy.t() @ (g * s * u)).to(dt)


def mxfp4_quantize_ref(x):
    """``(codes, scales)``."""
    K = x.shape[-1]
    b = torch.nn.functional.pad(x.float(), (0, -K % BLOCK)).reshape(*x.shape[:-1], -1, BLOCK)
    fine = torch.isfinite(b).all(-1)
    b = torch.where(fine.unsqueeze(-1), b, 0.0)
    m, k = torch.frexp(b.abs().amax(-1))
    e = torch.where(m > 0, k - 3 + (m > 0.75).int(), -127).clamp(min=-127)
    v = torch.ldexp(b, -e.unsqueeze(-1))
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 2).clamp(min=-1))
    q = (torch.round(v / step) * step).abs().contiguous()
    code = torch.searchsorted(torch.tensor(GRID, device=x.device), q).to(torch.uint8)
    code = torch.where(torch.signbit(b), code + 8, code).reshape(*x.shape[:-1], -1, 2)
    return code[..., 0] | code[..., 1] << 4, torch.where(fine, e + 127, 255).to(torch.uint8)


def _values(codes, scales):
    """In 64 bits, whole blocks."""
    grid = torch.tensor(GRID, dtype=torch.float64, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).int().reshape(*scales.shape, BLOCK)
    v = torch.where(c > 7, -grid[c & 7], grid[c & 7]) * torch.exp2(scales.double() - 127).unsqueeze(-1)
    v = torch.where(scales.unsqueeze(-1) == 255, float("nan"), v)
    return v.reshape(*scales.shape[:-1], -1)


def mxfp4_dequantize_ref(held, dtype=torch.bfloat16, columns=None):
    top = torch.finfo(dtype).max
    return _values(*held)[..., :columns].clamp(-top, top).to(dtype)


def mxfp4_linear_ref(x, weight, bias=None, out_dtype=None):
    quantised = isinstance(x, tuple)
    dt = out_dtype or (torch.bfloat16 if quantised else x.dtype)
    y = _values(*(x if quantised else mxfp4_quantize_ref(x))).float() @ _values(*weight).float().t()
    return (y if bias is None else y + bias.float()).to(dt)


DENSE_REFERENCES = {
    "gated_ffn": gated_ffn_ref,
    "gated_ffn_backward": gated_ffn_backward_ref,
    "mxfp4_quantize": mxfp4_quantize_ref,
    "mxfp4_dequantize": mxfp4_dequantize_ref,
    "mxfp4_linear": mxfp4_linear_ref,
}
