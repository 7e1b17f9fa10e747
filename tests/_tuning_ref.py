"""64-bit forms of the tuning ops, and bounds of what their kernels may be off,
from the arithmetic: an output rounding of half a step (``finfo.eps / 2``), fp32
sums of n terms (n + 32) * 2^-23 of the sum of magnitudes (twice the half step per
addition, for a matrix unit's own order and rounding), and 2^-16 for an operand
held as a bf16 pair (its two roundings leave 2^-17)."""
from __future__ import annotations

import torch

F32 = 2.0 ** -23


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def gamma(n: int) -> float:
    return (n + 32) * F32


def pair(dtype: torch.dtype) -> float:
    return 2.0 ** -16 if dtype == torch.bfloat16 else 0.0


def check(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, msg: str = ""):
    """``|got - want| <= half a step of the output + (1 + half a step) * bound``, the bound
    being that of the value before its last rounding; the type's least step beside."""
    got64, want, bound = got.detach().double().cpu(), want.cpu(), bound.cpu()
    assert got64.shape == want.shape, (got64.shape, want.shape, msg)
    u = half_step(got.dtype)
    lim = u * want.abs() + (1 + u) * bound + torch.finfo(got.dtype).smallest_normal * 2 * u
    bad = ~((got64 - want).abs() <= lim)
    if bad.any():
        i = int(bad.reshape(-1).nonzero()[0])
        raise AssertionError(f"{msg}: {int(bad.sum())}/{bad.numel()} values out of bounds; first at {i}: got "
                             f"{got64.reshape(-1)[i]:.9g} want {want.reshape(-1)[i]:.9g} bound {lim.reshape(-1)[i]:.3g}")


# ----------------------------------------------------------------- adapters ----

def lora_ref(x, a, b, ids, base=None, scaling=None):
    """``(out, hidden, bound of out, bound of hidden)`` in 64 bits (on the CPU)."""
    dt = x.dtype
    x, a, b, ids = x.double().cpu(), a.double().cpu(), b.double().cpu(), ids.cpu()
    L, r, K = a.shape
    M, N = x.shape[0], b.shape[1]
    sc = torch.ones(L, dtype=torch.float64) if scaling is None else scaling.double().cpu()
    out = torch.zeros(M, N, dtype=torch.float64) if base is None else base.double().cpu().clone()
    mag = out.abs()
    hidden = torch.zeros(M, r, dtype=torch.float64)
    bh, bo = torch.zeros(M, r, dtype=torch.float64), torch.zeros(M, N, dtype=torch.float64)
    for i in range(L):
        m = torch.nonzero(ids == i).flatten()
        h = x[m] @ a[i].t()
        hb = gamma(K) * (x[m].abs() @ a[i].abs().t())
        hidden[m], bh[m] = h, hb
        out[m] += sc[i] * (h @ b[i].t())
        size = sc[i].abs() * (h.abs() @ b[i].abs().t())
        bo[m] = sc[i].abs() * (hb @ b[i].abs().t()) + (pair(dt) + gamma(r) + 4 * F32) * size + 2 * F32 * (mag[m] + size)
    return out, hidden, bo, bh


def lora_grad_ref(dy, x, a, b, ids, hidden, scaling=None):
    """``((dx, dA, dB), (their bounds))``; x already in the values that the call reads."""
    dt = dy.dtype
    dy, x, a, b = (t.double().cpu() for t in (dy, x, a, b))
    hidden, ids = hidden.double().cpu(), ids.cpu()
    L, r, K = a.shape
    M, N = dy.shape
    sc = torch.ones(L, dtype=torch.float64) if scaling is None else scaling.double().cpu()
    dx, dxb = torch.zeros(M, K, dtype=torch.float64), torch.zeros(M, K, dtype=torch.float64)
    da, dab = torch.zeros(L, r, K, dtype=torch.float64), torch.zeros(L, r, K, dtype=torch.float64)
    db, dbb = torch.zeros(L, N, r, dtype=torch.float64), torch.zeros(L, N, r, dtype=torch.float64)
    for i in range(L):
        m = torch.nonzero(ids == i).flatten()
        n = m.numel()
        s = sc[i].abs()
        g = sc[i] * (dy[m] @ b[i])
        gb = (gamma(N) + 2 * F32) * s * (dy[m].abs() @ b[i].abs())
        dx[m] = g @ a[i]
        dxb[m] = gb @ a[i].abs() + (pair(dt) + gamma(r)) * (g.abs() @ a[i].abs())
        da[i] = g.t() @ x[m]
        dab[i] = gb.t() @ x[m].abs() + (pair(dt) + gamma(n)) * (g.abs().t() @ x[m].abs())
        u = sc[i] * hidden[m]
        db[i] = dy[m].t() @ u
        dbb[i] = (pair(dt) + gamma(n) + 2 * F32) * (dy[m].abs().t() @ u.abs())
    return (dx, da, db), (dxb, dab, dbb)


# ------------------------------------------------------------------- router ----

def softmax_delta(z: torch.Tensor) -> float:
    """Relative bound of a probability in fp32: the argument's rounding (its size times
    half a step), the exponential's few steps, the sum's terms."""
    f = z[torch.isfinite(z)]
    spread = float(f.max() - f.min()) if f.numel() else 0.0
    return (2 * spread + z.shape[1] + 32) * F32


def balance_ref(z, ids, mask=None):
    """``(loss, counts, tokens)`` in 64 bits."""
    z, ids = z.double().cpu(), ids.long().cpu()
    M, E = z.shape
    on = torch.ones(M, dtype=torch.bool) if mask is None else mask.cpu().bool()
    sel = ids[on]
    sel = sel[(sel >= 0) & (sel < E)]
    counts = torch.bincount(sel.flatten(), minlength=E)
    T, k = int(on.sum()), ids.shape[1]
    if T == 0:
        return torch.zeros((), dtype=torch.float64), counts, 0
    p = torch.softmax(z[on], 1)
    return E / (T * T * k) * (counts.double() @ p.sum(0)), counts, T


def router_grad_ref(z, ids, grad_weights=None, renorm=True, grad_loss=None, counts=None, mask=None):
    """``(grad, bound)`` in 64 bits; ids of one row may repeat, ids out of range have no slot."""
    delta = softmax_delta(z.double().cpu())
    z, ids = z.double().cpu(), ids.long().cpu()
    M, E = z.shape
    k = ids.shape[1]
    on = torch.ones(M, dtype=torch.bool) if mask is None else mask.cpu().bool()
    T = int(on.sum())
    p = torch.softmax(z, 1)
    grad, bound = torch.zeros_like(z), torch.zeros_like(z)
    if grad_loss is not None and T:
        f = float(grad_loss) * E / (T * T * k)
        c = counts.double().cpu()
        c = c - c.mean()
        mean_off = F32 * (E + 4) * counts.double().cpu().mean()  # the mean's own sum in 32 bits
        pc = (p @ c).unsqueeze(1)
        grad += f * p * (c - pc)
        size = (c - pc).abs() + c.abs() + (p @ c.abs()).unsqueeze(1)
        bound += abs(f) * p * ((3 * delta + 16 * F32) * size + 4 * mean_off)
    if grad_weights is not None:
        u = grad_weights.double().cpu()
        valid = ((ids >= 0) & (ids < E)).double()
        safe = ids.clamp(0, E - 1)
        pj = p.gather(1, safe) * valid
        if renorm:
            total = pj.sum(1, keepdim=True)
            w = torch.where(total > 0, pj / total.clamp(min=1e-300), 0.0) * valid
            mean = (w * u).sum(1, keepdim=True)
            slot, size = w * (u - mean), w * (u.abs() + (w * u.abs()).sum(1, keepdim=True))
        else:
            slot, size = pj * u * valid, pj * u.abs() * valid
            q = slot.sum(1, keepdim=True)
            grad -= p * q
            bound += (3 * delta + (k + 16) * F32) * p * (pj * u.abs()).sum(1, keepdim=True)
        grad.scatter_add_(1, safe, slot)
        bound.scatter_add_(1, safe, (4 * delta + (2 * k + 16) * F32) * size)
    grad[~on], bound[~on] = 0.0, 0.0
    return grad, bound


# -------------------------------------------------------------- checkpoints ----

def e4m3_grid() -> torch.Tensor:
    """All non-negative finite e4m3 values, ascending: 2^-9 steps below 2^-6, then 8 a binade."""
    sub = torch.arange(8, dtype=torch.float64) * 2.0 ** -9
    norm = torch.cat([(1 + torch.arange(8, dtype=torch.float64) / 8) * 2.0 ** e for e in range(-6, 9)])
    return torch.cat([sub, norm])[:-1]  # the last code is NaN


def checkpoint_ref(x: torch.Tensor):
    """``(restored values in 64 bits, scale bytes)``, by search: for each block the least
    exponent, for each value the nearest grid value (the even code of two)."""
    x = x.double().cpu()
    M, K = x.shape
    nb = -(-K // 32)
    grid = e4m3_grid()
    padded = torch.zeros(M, nb * 32, dtype=torch.float64)
    padded[:, :K] = x
    blocks = padded.view(M, nb, 32)
    fine = torch.isfinite(blocks)
    amax = torch.where(fine, blocks.abs(), 0.0).amax(-1)
    exps = torch.arange(-127, 128, dtype=torch.float64)
    fits = amax.unsqueeze(-1) * torch.exp2(-exps) <= 448.0
    e = exps[fits.int().argmax(-1)]
    v = torch.where(fine, blocks, 0.0) * torch.exp2(-e).unsqueeze(-1)
    at = torch.searchsorted(grid, v.abs().contiguous()).clamp(1, grid.numel() - 1)
    lo, hi = grid[at - 1], grid[at]
    down, up = v.abs() - lo, hi - v.abs()
    code = torch.where((down < up) | ((down == up) & ((at - 1) % 2 == 0)), at - 1, at)
    q = torch.copysign(grid[code], v) * torch.exp2(e).unsqueeze(-1)
    q = torch.where(fine, q, float("nan"))
    return q.reshape(M, -1)[:, :K], (e + 127).to(torch.uint8)
