"""64-bit forms of the dense block's ops, and bounds of what their kernels may be off, from
the arithmetic: half a step of the type for each rounding to it, ``gamma(n)`` for fp32 sums
of n terms, and for the activation its derivative (at most 1.1, the second one at most 0.5)
times what its argument is off."""
from __future__ import annotations

import torch

from tests._tuning_ref import F32, gamma, half_step

# (64-bit forms of the feed-forward block stay on their inputs' device)
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _tiny(dtype: torch.dtype) -> float:
    """Half of the least step, by which values near zero may be off."""
    return torch.finfo(dtype).smallest_normal * half_step(dtype)


def _clamped(g, u, limit):
    if limit is None:
        return g, u, torch.ones_like(g), torch.ones_like(u)
    return g.clamp(max=limit), u.clamp(-limit, limit), (g <= limit).double(), (u.abs() <= limit).double()


def ffn_ref(x, w13, w2, limit=None, pair=False):
    """``(out, gate_up, bound of out, bound of gate_up)``; ``pair``: the activations are held with what
    their rounding left, rounded itself (off by a half step of a half step), in a sum of twice the terms."""
    e, tiny = half_step(x.dtype), _tiny(x.dtype)
    x, w13, w2 = (t.double() for t in (x, w13, w2))
    H, I = w2.shape
    gu, off = x @ w13.t(), gamma(H) * (x.abs() @ w13.abs().t())
    gc, uc, _, _ = _clamped(gu[:, :I], gu[:, I:], limit)
    s = torch.sigmoid(gc)
    h = gc * s * uc
    h_off = 1.1 * uc.abs() * off[:, :I] + (gc * s).abs() * off[:, I:] + (gc.abs() + 16) * F32 * h.abs()
    h_off = h_off * (1 + e) + (e * e if pair else e) * h.abs() + tiny
    out, n = h @ w2.t(), 2 * I if pair else I
    return out, gu, (h_off * (1 + gamma(n)) + gamma(n) * (1 + e) * h.abs()) @ w2.abs().t(), off


def ffn_grad_ref(dy, x, w13, w2, limit=None):
    """``((dx, dW13, dW2), (their bounds))``."""
    e, tiny = half_step(x.dtype), _tiny(x.dtype)
    dy, x, w13, w2 = (t.double() for t in (dy, x, w13, w2))
    H, I = w2.shape
    M = x.shape[0]
    gu, off = x @ w13.t(), gamma(H) * (x.abs() @ w13.abs().t())
    g, u = gu[:, :I], gu[:, I:]
    gc, uc, on_g, on_u = _clamped(g, u, limit)
    # a sum next to the limit may fall on its other side
    near = torch.zeros_like(gu) if limit is None else \
        (torch.cat(((g - limit).abs(), (u.abs() - limit).abs()), 1) <= 2 * off).double()
    og, ou = off[:, :I], off[:, I:]
    s = torch.sigmoid(gc)
    silu, slope = gc * s, s * (1 + gc * (1 - s))
    dh, dh_off = dy @ w2, gamma(H) * (dy.abs() @ w2.abs())
    rel = (gc.abs() + 32) * F32
    dg, du, h = dh * uc * slope, dh * silu, silu * uc
    dg_off = dh_off * (uc * slope).abs() + dh.abs() * (ou * slope.abs() + 0.5 * uc.abs() * og) + \
        rel * dh.abs() * uc.abs() * (s + (gc * s).abs())
    du_off = dh_off * silu.abs() + dh.abs() * 1.1 * og + rel * du.abs()
    h_off = 1.1 * uc.abs() * og + silu.abs() * ou + rel * h.abs()
    d = torch.cat((dg * on_g, du * on_u), 1)
    d_off = torch.cat((dg_off, du_off), 1)
    d_off = d_off * (1 + e) + e * d.abs() + near * torch.cat((dg.abs(), du.abs()), 1) + tiny
    h_off = h_off * (1 + e) + e * h.abs() + tiny
    grads = d @ w13, d.t() @ x, dy.t() @ h
    bounds = ((d_off + gamma(2 * I) * (d.abs() + d_off)) @ w13.abs(),
              (d_off + gamma(M) * (d.abs() + d_off)).t() @ x.abs(),
              dy.abs().t() @ (h_off + gamma(M) * (h.abs() + h_off)))
    return grads, bounds


def mxfp4_ref(x: torch.Tensor):
    """``(values in 64 bits [..., K], scale bytes)`` by search: for each block the least exponent
    with which nothing passes 6, for each value the nearest of the grid (the even code of two);
    a block that is not finite is NaN with byte 255."""
    x = x.double().cpu()
    K = x.shape[-1]
    nb = -(-K // 32)
    b = torch.nn.functional.pad(x.reshape(-1, K), (0, nb * 32 - K)).view(-1, nb, 32)
    fine = torch.isfinite(b).all(-1)
    b = torch.where(fine.unsqueeze(-1), b, 0.0)
    exps = torch.arange(-127, 128, dtype=torch.float64)
    fits = b.abs().amax(-1, keepdim=True) * torch.exp2(-exps) <= 6.0
    e = exps[fits.int().argmax(-1)]
    v = b.abs() * torch.exp2(-e).unsqueeze(-1)
    at = torch.searchsorted(GRID, v.contiguous()).clamp(1, 7)
    down, up = v - GRID[at - 1], GRID[at] - v
    code = torch.where((down < up) | ((down == up) & ((at - 1) % 2 == 0)), at - 1, at)
    q = torch.copysign(GRID[code], b) * torch.exp2(e).unsqueeze(-1)
    q = torch.where(fine.unsqueeze(-1), q, float("nan"))
    scales = torch.where(fine, e + 127, 255.0).to(torch.uint8)
    return q.view(-1, nb * 32)[:, :K].reshape(x.shape), scales.view(*x.shape[:-1], nb)


def mxfp4_values(held) -> torch.Tensor:
    """The values of codes and scales in 64 bits, whole blocks."""
    c, s = (t.cpu() for t in held)
    n = torch.stack((c & 15, c >> 4), -1).int().reshape(*s.shape, 32)
    v = torch.where(n > 7, -GRID[n & 7], GRID[n & 7]) * torch.exp2(s.double() - 127).unsqueeze(-1)
    return torch.where(s.unsqueeze(-1) == 255, float("nan"), v).reshape(*s.shape[:-1], -1)


def linear_ref(xv, wv, bias=None):
    """``(out, bound)`` of values in 64 bits."""
    out, off = xv @ wv.t(), gamma(xv.shape[1]) * (xv.abs() @ wv.abs().t())
    return (out, off) if bias is None else (out + bias.double().cpu(), off + F32 * (out.abs() + off))
