"""What tuning and serving over the frozen MoE layer costs: the router's training
step, low-rank adapters beside a shared projection and their gradients, and
activation checkpoints in 8 bits.

A case is a dict of plain values with an ``op``:

* ``router``      balance loss, per-expert counts and the gradient of the logits
* ``adapter``     adapters of many requests beside a shared projection
* ``adapter-grad`` the gradients of the same (input and both weights), the input
  held as it is or in 8 bits
* ``checkpoint``  activations to 8 bits and back

``listed()`` names the fixed cases, ``draw(rng)`` gives further ones of the same
ranges, ``prepare`` makes a case's inputs on the GPU, ``run`` is one pass: through
the library where ``own`` is set, else in plain torch operations in 32 bits.
``exact`` is the same result in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
E4M3_MAX = 448.0


def router(M, E, top_k, dtype="bf16", renormalize=True, padded=0.0):
    """``padded``: the share of rows that are padding (masked out)."""
    return {"op": "router", "M": M, "E": E, "top_k": top_k, "dtype": dtype, "renormalize": renormalize,
            "padded": padded}


def adapter(M, K, N, adapters, rank, dtype="bf16", layout="requests", bare=0.0):
    """``layout``: rows of one request lie together (``requests``), or every row is
    a request of its own (``mixed``); ``bare``: the share of requests without an
    adapter."""
    return {"op": "adapter", "M": M, "K": K, "N": N, "adapters": adapters, "rank": rank, "dtype": dtype,
            "layout": layout, "bare": bare}


def adapter_grad(M, K, N, adapters, rank, dtype="bf16", layout="requests", bare=0.0, held="as is"):
    """``held``: the input ``as is``, or in ``8 bits``."""
    return {**adapter(M, K, N, adapters, rank, dtype, layout, bare), "op": "adapter-grad", "held": held}


def checkpoint(M, K, dtype="bf16"):
    return {"op": "checkpoint", "M": M, "K": K, "dtype": dtype}


def listed() -> list[dict]:
    return [
        # the router of one short sequence, fp32 logits
        {"name": "router-m200", **router(200, 48, 8, "fp32")},
        # a training batch of 8,192 tokens whose sequences are padded
        {"name": "router-m8192", **router(8192, 256, 8, "bf16", padded=0.1)},
        # a large batch on a 384-expert router
        {"name": "router-m65536", **router(65536, 384, 8, "bf16", renormalize=False)},
        # one user's decode step with an adapter beside the gate/up projection
        {"name": "adapter-m1", **adapter(1, 7168, 4096, 8, 16, layout="mixed")},
        # a decode batch of 64 users over 32 adapters, some without one
        {"name": "adapter-m64", **adapter(64, 7168, 4096, 32, 16, layout="mixed", bare=0.2)},
        # prompts of several users in one batch
        {"name": "adapter-m4096", **adapter(4096, 7168, 4096, 8, 32, bare=0.1)},
        # a large prefill batch beside the down projection, high rank
        {"name": "adapter-m16384", **adapter(16384, 2048, 7168, 8, 64)},
        # a small tuning step of two adapters, ragged sizes
        {"name": "grad-m300", **adapter_grad(300, 2880, 2880, 2, 8, bare=0.1)},
        # a tuning step of four adapters, activations kept as they are
        {"name": "grad-m8192", **adapter_grad(8192, 7168, 4096, 4, 16)},
        # a large tuning step of one adapter from 8-bit activations
        {"name": "grad-m16384-8bit", **adapter_grad(16384, 7168, 2048, 1, 32, held="8 bits")},
        # checkpoints of a short sequence
        {"name": "checkpoint-m100", **checkpoint(100, 2880)},
        # checkpoints of a large training batch
        {"name": "checkpoint-m16384", **checkpoint(16384, 7168)},
    ]


def _log(rng, lo, hi) -> int:
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng) -> int:
    """A projection's width: a model's, any multiple of 8, or an odd one."""
    kind = rng.random()
    if kind < 0.4:
        return rng.choice([1024, 2048, 2880, 4096, 7168])
    n = _log(rng, 256, 7168)
    return max(8, n // 8 * 8) if kind < 0.85 else n | 1


def draw(rng) -> dict:
    op = rng.choice(["router", "adapter", "adapter", "adapter-grad", "adapter-grad", "checkpoint"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if op == "router":
        E = rng.choice([8, 48, 64, 100, 256, 384])
        return router(_log(rng, 1, 65536), E, rng.choice([1, 2, 4, 6, 8]), rng.choice(["bf16", "fp16", "fp32"])
                      if E < 200 else "bf16", rng.random() < 0.7, rng.choice([0.0, 0.1, 0.5]))
    if op == "checkpoint":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return checkpoint(_log(rng, 1, 16384 if dtype != "fp32" else 8192), _width(rng), dtype)
    rank = rng.choice([4, 8, 12, 16, 16, 32, 32, 64])
    adapters = _log(rng, 1, min(32, 512 // rank))
    K, N = _width(rng), _width(rng)
    layout, bare = rng.choice(["requests", "mixed"]), rng.choice([0.0, 0.1, 0.4])
    if op == "adapter":
        return adapter(_log(rng, 1, 8192 if dtype == "bf16" else 4096), K, N, adapters, rank, dtype, layout, bare)
    return adapter_grad(_log(rng, 1, 8192 if dtype == "bf16" else 4096), K, N, adapters, rank, dtype, layout, bare,
                        rng.choice(["as is", "8 bits"]))


# ------------------------------------------------------------------- inputs ---

def _adapter_ids(c, g):
    M, dev = c["M"], "cuda"
    n = M if c["layout"] == "mixed" else max(1, min(M, 2 * c["adapters"]))
    which = torch.randint(0, c["adapters"], (n,), generator=g, device=dev, dtype=torch.int32)
    which[torch.rand(n, generator=g, device=dev) < c["bare"]] = -1
    if c["layout"] == "mixed":
        return which
    ends = torch.sort(torch.randint(0, M + 1, (n - 1,), generator=g, device=dev)).values  # ragged, some empty
    return which[torch.bucketize(torch.arange(M, device=dev), ends, right=True)].contiguous()


def _blocks(x):
    """[M, K] -> [M, blocks, 32], the last block filled up with zeros."""
    M, K = x.shape
    return torch.nn.functional.pad(x, (0, -K % 32)).view(M, -1, 32)


def _to_8_bits(x):
    """Values in e4m3 and one power of two for each 32 of a row, the least with
    which none of them passes 448; infinities and NaN become NaN and do not count."""
    b = _blocks(x.float())
    fine = torch.isfinite(b)
    amax = torch.where(fine, b.abs(), 0.0).amax(-1)
    m, k = torch.frexp(amax)
    e = torch.where(amax > 0, k - 9 + (m > 0.875).int(), -127).clamp(-127, 127)
    q = torch.where(fine, torch.ldexp(b, -e.unsqueeze(-1)), float("nan")).to(torch.float8_e4m3fn)
    return q.view(x.shape[0], -1)[:, : x.shape[1]].contiguous(), (e + 127).to(torch.uint8)


def _from_8_bits(q, scales):
    """fp32 values."""
    e = scales.int().unsqueeze(-1) - 127
    return torch.ldexp(_blocks(q.float()), e).view(q.shape[0], -1)[:, : q.shape[1]]


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, M, dt = c["op"], c["M"], DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": c}
    if op == "router":
        E, k = c["E"], c["top_k"]
        popularity = 0.5 * randn(E)
        s["logits"] = (1.5 * randn(M, E) + popularity).to(dt)
        s["ids"] = torch.topk(s["logits"].float(), k, dim=1).indices.to(torch.int32)
        s["grad_weights"] = randn(M, k) / M
        s["grad_loss"] = torch.full((), 0.01, device="cuda")
        s["mask"] = torch.rand(M, generator=g, device="cuda") >= c["padded"] if c["padded"] else None
        return s
    if op == "checkpoint":
        # channels of different magnitude, as activations have them
        s["x"] = (randn(M, c["K"]) * torch.exp(randn(c["K"]))).to(dt)
        return s
    K, N, L, r = c["K"], c["N"], c["adapters"], c["rank"]
    s["a"] = (randn(L, r, K) / math.sqrt(K)).to(dt)
    s["b"] = (randn(L, N, r) / math.sqrt(r)).to(dt)
    s["scaling"] = torch.rand(L, generator=g, device="cuda") * 1.5 + 0.5
    s["ids"] = _adapter_ids(c, g)
    s["x"] = randn(M, K).to(dt)
    if op == "adapter":
        s["base"] = randn(M, N).to(dt)
        return s
    s["grad"] = (randn(M, N) / 64).to(dt)
    s["hidden"] = _rows_times(s["x"].float(), s["a"].float(), s["ids"])
    if c["held"] == "8 bits":
        s["x"] = _to_8_bits(s["x"])
    return s


# --------------------------------------------------------------- plain forms ---

def _router_plain(s):
    c, z, ids, mask = s["case"], s["logits"].float(), s["ids"].long(), s["mask"]
    M, E, k = c["M"], c["E"], c["top_k"]
    on = torch.ones(M, 1, device=z.device) if mask is None else mask.float().unsqueeze(1)
    ez = torch.exp(z - z.amax(1, keepdim=True))
    p = ez / ez.sum(1, keepdim=True)
    chosen = torch.zeros(M, E, device=z.device).scatter_add_(1, ids, on.expand(M, k))
    counts = chosen.sum(0, dtype=torch.float64)
    tokens = on.sum(dtype=torch.float64).clamp(min=1.0)
    factor = E / (tokens * tokens * k)
    loss = (factor * (counts * (p * on).sum(0, dtype=torch.float64)).sum()).float()
    over = (counts - counts.mean()).float()
    grad = (factor * s["grad_loss"]).float() * p * (over - (p * over).sum(1, keepdim=True))
    pj, u = p.gather(1, ids), s["grad_weights"]
    if c["renormalize"]:
        w = pj / pj.sum(1, keepdim=True)
        grad.scatter_add_(1, ids, w * (u - (w * u).sum(1, keepdim=True)))
    else:
        grad -= p * (pj * u).sum(1, keepdim=True)
        grad.scatter_add_(1, ids, pj * u)
    return loss, counts.int(), (grad * on).to(s["logits"].dtype)


def _wide(h, ids, L):
    """[M, r] -> [M, L * r]: row m's values in its adapter's columns, zeros elsewhere."""
    mine = ids.unsqueeze(1) == torch.arange(L, device=h.device, dtype=ids.dtype)
    return torch.where(mine.unsqueeze(2), h.unsqueeze(1), 0.0).view(h.shape[0], -1)


def _rows_times(x, a, ids):
    """``x[m] @ a[ids[m]].T``: every adapter's products, of which a row keeps its own."""
    L, r, K = a.shape
    h = (x @ a.reshape(L * r, K).t()).view(-1, L, r)
    mine = ids.unsqueeze(1) == torch.arange(L, device=x.device, dtype=ids.dtype)
    return torch.where(mine.unsqueeze(2), h, 0.0).sum(1)


def _adapter_plain(s):
    a, b, ids, L = s["a"].float(), s["b"].float(), s["ids"], s["case"]["adapters"]
    h = _rows_times(s["x"].float(), a, ids)
    delta = _wide(h, ids, L) @ (b * s["scaling"].view(L, 1, 1)).transpose(1, 2).reshape(-1, b.shape[1])
    return (s["base"].float() + delta).to(s["base"].dtype)


def _adapter_grad_plain(s):
    a, b, ids, grad = s["a"].float(), s["b"].float(), s["ids"], s["grad"].float()
    (L, r, K), N, dt = a.shape, b.shape[1], s["a"].dtype
    x = s["x"].float() if torch.is_tensor(s["x"]) else _from_8_bits(*s["x"])
    bs = (b * s["scaling"].view(L, 1, 1)).transpose(1, 2).contiguous()  # [L, r, N]
    g = _wide(_rows_times(grad, bs, ids), ids, L)  # [M, L * r]
    grad_x = g @ a.view(L * r, K)
    grad_a = (g.t() @ x).view(L, r, K)
    grad_b = (_wide(s["hidden"], ids, L).t() @ grad).view(L, r, N) * s["scaling"].view(L, 1, 1)
    return grad_x.to(dt), grad_a.to(dt), grad_b.transpose(1, 2).contiguous().to(dt)


def _checkpoint_plain(s):
    q, scales = _to_8_bits(s["x"])
    return _from_8_bits(q, scales).to(s["x"].dtype), scales


def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        import xkernels_amd as xk
        if op == "router":
            loss, counts, tokens = xk.moe_balance_loss(s["logits"], s["ids"], mask=s["mask"])
            grad = xk.moe_router_backward(s["logits"], s["ids"], grad_weights=s["grad_weights"],
                                          renormalize=c["renormalize"], grad_loss=s["grad_loss"], counts=counts,
                                          tokens=tokens, mask=s["mask"])
            return loss, counts, grad
        if op == "adapter":
            return xk.lora_projection(s["x"], s["a"], s["b"], s["ids"], base=s["base"], scaling=s["scaling"])
        if op == "adapter-grad":
            x = s["x"] if torch.is_tensor(s["x"]) else xk.ActCheckpoint(*s["x"])
            return xk.lora_projection_backward(s["grad"], x, s["a"], s["b"], s["ids"], s["hidden"],
                                               scaling=s["scaling"])
        held = xk.act_checkpoint(s["x"])
        return xk.act_restore(held, s["x"].dtype), held.scales
    if op == "router":
        return _router_plain(s)
    if op == "adapter":
        return _adapter_plain(s)
    if op == "adapter-grad":
        return _adapter_grad_plain(s)
    return _checkpoint_plain(s)


# --------------------------------------------------------------------- work ---

def work(c) -> dict:
    op, M, size = c["op"], c["M"], SIZES[c["dtype"]]
    if op == "router":
        E, k = c["E"], c["top_k"]
        # the logits for the loss, and again for the gradient, which needs its sums
        return {"bytes": 3 * M * E * size + M * k * (4 + 4) + M * bool(c["padded"]), "flops": 20.0 * M * E}
    K = c["K"]
    if op == "checkpoint":
        return {"bytes": 2 * (M * K * (size + 1) + M * -(-K // 32)), "flops": 4.0 * M * K}
    N, L, r = c["N"], c["adapters"], c["rank"]
    used = L * (1.0 - (1.0 - 1.0 / L) ** (M if c["layout"] == "mixed" else min(M, 2 * L)))
    rows = M * (1.0 - c["bare"])
    if op == "adapter":
        return {"bytes": M * (K + 2 * N) * size + used * r * (K + N) * size + M * 4, "flops": 2.0 * rows * r * (K + N)}
    held = K * size if c["held"] == "as is" else K + -(-K // 32)
    return {"bytes": M * (N * size + held + K * size + r * 4 + 4) + (used + L) * r * (K + N) * size,
            "flops": 4.0 * rows * r * (K + N)}


# ------------------------------------------------------------------- 64 bits ---

def _e4m3(v):
    """64-bit values of at most 448 to the nearest e4m3 value, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def _exact_8_bits(x):
    """The restored values in 64 bits, and the scale bytes."""
    b = _blocks(x.double())
    amax = b.abs().amax(-1)
    e = torch.ceil(torch.log2(amax / E4M3_MAX)).clamp(-127, 127)
    e = torch.where(amax > torch.exp2(e) * E4M3_MAX, e + 1, e)
    e = torch.where(amax <= torch.exp2(e - 1) * E4M3_MAX, e - 1, e).clamp(-127, 127)
    e = e.unsqueeze(-1)
    return (_e4m3(b * torch.exp2(-e)) * torch.exp2(e)).view(x.shape[0], -1)[:, : x.shape[1]], e


def exact(c, seed):
    s = prepare(c, seed)
    op, M = c["op"], c["M"]
    if op == "router":
        z, ids, E, k = s["logits"].double(), s["ids"].long(), c["E"], c["top_k"]
        on = torch.arange(M, device=z.device) if s["mask"] is None else torch.nonzero(s["mask"]).flatten()
        grad = torch.zeros_like(z)
        if on.numel() == 0:
            return z.new_zeros(()), None, grad
        p, ids, u = torch.softmax(z[on], 1), ids[on], s["grad_weights"][on].double()
        counts = torch.bincount(ids.flatten(), minlength=E).double()
        factor = E / (on.numel() ** 2 * k)
        loss = factor * (counts @ p.sum(0))
        d = p * (counts - (p @ counts).unsqueeze(1)) * factor * s["grad_loss"].double()
        if c["renormalize"]:
            w = torch.softmax(z[on].gather(1, ids), 1)
            d.scatter_add_(1, ids, w * (u - (w * u).sum(1, keepdim=True)))
        else:
            dp = torch.zeros_like(p).scatter_add_(1, ids, u)
            d += p * (dp - (dp * p).sum(1, keepdim=True))
        grad[on] = d
        return loss, None, grad
    if op == "checkpoint":
        return _exact_8_bits(s["x"])[0], None
    L, ids = c["adapters"], s["ids"]
    if op == "adapter":
        y = s["base"].double()
        for i in range(L):
            m = torch.nonzero(ids == i).flatten()
            y[m] += s["scaling"][i].double() * (s["x"][m].double() @ s["a"][i].double().t()) @ s["b"][i].double().t()
        return y
    if torch.is_tensor(s["x"]):
        x = s["x"].double()
    else:
        q, scales = s["x"]
        powers = torch.exp2(scales.double() - 127).repeat_interleave(32, 1)[:, : q.shape[1]]
        x = q.double() * powers
    grad_x = torch.zeros(M, c["K"], dtype=torch.float64, device="cuda")
    grad_a = torch.zeros(s["a"].shape, dtype=torch.float64, device="cuda")
    grad_b = torch.zeros(s["b"].shape, dtype=torch.float64, device="cuda")
    for i in range(L):
        m = torch.nonzero(ids == i).flatten()
        dy = s["grad"][m].double() * s["scaling"][i].double()
        g = dy @ s["b"][i].double()
        grad_x[m] = g @ s["a"][i].double()
        grad_a[i] = g.t() @ x[m]
        grad_b[i] = dy.t() @ s["hidden"][m].double()
    return grad_x, grad_a, grad_b
