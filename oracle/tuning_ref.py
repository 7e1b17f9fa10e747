"""Plain torch (fp32) forms of the ops for tuning and serving over the frozen experts:
the REFERENCE backend that the test harness registers for them. TEST
INFRASTRUCTURE, as the rest of this package. Written from the ops' definitions (the
reference has no counterpart); pinned by tests/test_tuning_host.py against 64-bit
forms and autograd."""
from __future__ import annotations

import torch

BLOCK, E4M3_MAX = 32, 448.0


def _rows_on(M, mask, device):
    return torch.ones(M, dtype=torch.bool, device=device) if mask is None else mask.bool()


def moe_balance_loss_ref(gating_output, topk_ids, mask=None):
    """``(loss, counts, tokens)``."""
    M, E = gating_output.shape
    on = _rows_on(M, mask, gating_output.device)
    ids = topk_ids[on].long().flatten()
    counts = torch.bincount(ids[(ids >= 0) & (ids < E)], minlength=E)
    T, k = int(on.sum()), topk_ids.shape[1]
    p = torch.softmax(gating_output[on].float(), 1).sum(0, dtype=torch.float64)
    loss = E / (T * T * k) * (counts.double() @ p) if T else p.new_zeros(())
    return loss.float(), counts.int(), torch.tensor(T, dtype=torch.int32, device=gating_output.device)


def moe_router_backward_ref(gating_output, topk_ids, grad_weights=None, renormalize=True, grad_loss=None,
                            counts=None, tokens=None, mask=None):
    M, E = gating_output.shape
    z, ids = gating_output.float(), topk_ids.long()
    on = _rows_on(M, mask, z.device)
    p = torch.softmax(z, 1)
    grad = torch.zeros_like(p)
    T = M if tokens is None else int(tokens)
    if grad_loss is not None and T:
        c = counts.float() - counts.float().mean()
        grad += float(grad_loss) * E / (T * T * ids.shape[1]) * p * (c - (p @ c).unsqueeze(1))
    if grad_weights is not None:
        valid = (ids >= 0) & (ids < E)
        at = ids.clamp(0, E - 1)
        u = torch.where(valid, grad_weights.float(), 0.0)
        if renormalize:
            w = torch.softmax(z.gather(1, at).masked_fill(~valid, float("-inf")), 1).nan_to_num()
            grad.scatter_add_(1, at, w * (u - (w * u).sum(1, keepdim=True)))
        else:
            du = torch.zeros_like(p).scatter_add_(1, at, u)
            grad += p * (du - (p * du).sum(1, keepdim=True))
    return torch.where(on.unsqueeze(1), grad, 0.0).to(gating_output.dtype)


def lora_projection_ref(x, lora_a, lora_b, adapter_ids, base=None, scaling=None, return_hidden=False):
    M, (L, r, _), N = x.shape[0], lora_a.shape, lora_b.shape[1]
    out = torch.zeros(M, N, device=x.device) if base is None else base.to(torch.float32, copy=True)
    hidden = torch.zeros(M, r, device=x.device)
    for i in range(L):
        m = torch.nonzero(adapter_ids == i).flatten()
        hidden[m] = x[m].float() @ lora_a[i].float().t()
        out[m] += (1.0 if scaling is None else scaling[i]) * (hidden[m] @ lora_b[i].float().t())
    out = out.to(x.dtype)
    return (out, hidden) if return_hidden else out


def lora_projection_backward_ref(grad_out, x, lora_a, lora_b, adapter_ids, hidden, scaling=None):
    x = act_restore_ref(x, grad_out.dtype).float() if isinstance(x, tuple) else x.float()
    gx = torch.zeros(x.shape, device=x.device)
    ga, gb = torch.zeros(lora_a.shape, device=x.device), torch.zeros(lora_b.shape, device=x.device)
    for i in range(lora_a.shape[0]):
        m = torch.nonzero(adapter_ids == i).flatten()
        dy = grad_out[m].float() * (1.0 if scaling is None else scaling[i])
        g = dy @ lora_b[i].float()
        gx[m], ga[i], gb[i] = g @ lora_a[i].float(), g.t() @ x[m], dy.t() @ hidden[m].float()
    return gx.to(grad_out.dtype), ga.to(lora_a.dtype), gb.to(lora_b.dtype)


def act_checkpoint_ref(x):
    """``(values float8_e4m3fn, scales uint8)``."""
    M, K = x.shape
    b = torch.nn.functional.pad(x.float(), (0, -K % BLOCK)).view(M, -1, BLOCK)
    fine = torch.isfinite(b)
    m, k = torch.frexp(torch.where(fine, b.abs(), 0.0).amax(-1))
    e = torch.where(m > 0, k - 9 + (m > E4M3_MAX / 512).int(), -127).clamp(min=-127)
    q = torch.where(fine, torch.ldexp(b, -e.unsqueeze(-1)), float("nan")).to(torch.float8_e4m3fn)
    return q.view(M, -1)[:, :K].contiguous(), (e + 127).to(torch.uint8)


def act_restore_ref(held, dtype=torch.bfloat16):
    values, scales = held
    powers = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, 1)[:, : values.shape[1]]
    top = torch.finfo(dtype).max
    return (values.double() * powers).clamp(-top, top).to(dtype)


TUNING_REFERENCES = {
    "moe_balance_loss": moe_balance_loss_ref,
    "moe_router_backward": moe_router_backward_ref,
    "lora_projection": lora_projection_ref,
    "lora_projection_backward": lora_projection_backward_ref,
    "act_checkpoint": act_checkpoint_ref,
    "act_restore": act_restore_ref,
}
