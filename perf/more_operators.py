"""What the dense gated feed-forward block beside the routed experts costs, in
training and in serving, and the way of its weights into 4 bits: quantisation and
the product of quantised operands.

A case is a dict of plain values with an ``op``:

* ``ffn``        the block's forward
* ``ffn-train``  its training step: the forward, which keeps the projections' sums,
                 and the gradients of the input and of all weights
* ``quantise``   values to 4 bits (MXFP4) and back
* ``product``    16- or 32-bit activations, quantised in the call, times quantised weights

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
LIMIT = 10.0  # the clamp of the experts' SwiGLU


def ffn(M, hidden, ispp, dtype="bf16", clamp=False):
    return {"op": "ffn", "M": M, "hidden": hidden, "ispp": ispp, "dtype": dtype, "clamp": clamp}


def ffn_train(M, hidden, ispp, dtype="bf16", clamp=False):
    return {**ffn(M, hidden, ispp, dtype, clamp), "op": "ffn-train"}


def quantise(M, K, dtype="bf16"):
    return {"op": "quantise", "M": M, "K": K, "dtype": dtype}


def product(M, K, N, dtype="bf16", bias=False):
    return {"op": "product", "M": M, "K": K, "N": N, "dtype": dtype, "bias": bias}


def listed() -> list[dict]:
    return [
        # one user's decode step through the shared expert
        {"name": "ffn-m1", **ffn(1, 7168, 2048)},
        # a decode batch of 64 users, clamped as the MXFP4 experts are
        {"name": "ffn-m64", **ffn(64, 4096, 2048, clamp=True)},
        # prompts of several users in one batch
        {"name": "ffn-m4096", **ffn(4096, 7168, 2048)},
        # a short training batch, no size a multiple of a tile
        {"name": "train-m1023", **ffn_train(1023, 1001, 333, "fp16", clamp=True)},
        # a tuning step of ordinary sizes
        {"name": "train-m2000", **ffn_train(2000, 2880, 2880)},
        # a large training batch
        {"name": "train-m8192", **ffn_train(8192, 7168, 2048)},
        # a small matrix, fp32, the last block of a row short
        {"name": "quantise-m300", **quantise(300, 1000, "fp32")},
        # the weights of four experts' gate and up projections, one after the other
        {"name": "quantise-m16384", **quantise(16384, 7168)},
        # one user's decode step
        {"name": "product-m1", **product(1, 7168, 4096)},
        # a decode batch, ragged sizes, with a bias
        {"name": "product-m77", **product(77, 2880, 2881, "fp16", bias=True)},
        # a prefill batch through the gate/up projection
        {"name": "product-m4096", **product(4096, 7168, 4096)},
        # a large prefill batch through the down projection
        {"name": "product-m16384", **product(16384, 2048, 7168)},
    ]


def _log(rng, lo, hi) -> int:
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo=256, hi=7168) -> int:
    """A projection's width: a model's, any multiple of 8, or an odd one."""
    kind = rng.random()
    if kind < 0.4:
        return rng.choice([w for w in (512, 1024, 2048, 2880, 4096, 7168) if lo <= w <= hi])
    n = _log(rng, lo, hi)
    return max(8, n // 8 * 8) if kind < 0.8 else min(hi, n | 1)


def draw(rng) -> dict:
    op = rng.choice(["ffn", "ffn", "ffn-train", "ffn-train", "quantise", "product", "product"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "quantise":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return quantise(_log(rng, 1, 16384 if dtype != "fp32" else 8192), _width(rng, 33), dtype)
    if op == "product":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return product(_log(rng, 1, 8192), _width(rng), _width(rng, 128), dtype, rng.random() < 0.3)
    make = ffn if op == "ffn" else ffn_train
    return make(_log(rng, 1, 8192 if op == "ffn" else 4096), _width(rng), _width(rng, 64, 4096), dtype,
                rng.random() < 0.5)


# ------------------------------------------------------------------- 4 bits ---

def _blocks(x):
    """[M, K] -> [M, blocks, 32], the last block filled up with zeros."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).view(x.shape[0], -1, 32)


def _to_4_bits(x):
    """``(values, scales)``: what e2m1 holds of each value over its block's scale, [M,
    blocks, 32], and the e8m0 bytes, the least power of two with which none passes 6."""
    b = _blocks(x.float())
    m, k = torch.frexp(b.abs().amax(-1))  # m in [0.5, 1)
    e = torch.where(m > 0, k - 3 + (m > 0.75).int(), -127).clamp(min=-127)
    v = torch.ldexp(b, -e.unsqueeze(-1))
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 2).clamp(min=-1))
    return torch.round(v / step) * step, (e + 127).to(torch.uint8)


def _pack(values):
    """e2m1 codes, two a byte, the even place in the low half: [M, blocks * 16]."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=values.device)
    code = torch.searchsorted(grid, values.abs().contiguous()).to(torch.uint8)
    code = torch.where(values < 0, code + 8, code).view(values.shape[0], -1, 2)
    return code[..., 0] | code[..., 1] << 4


def _unpack(codes):
    """[M, blocks * 16] bytes -> [M, blocks, 32] values."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                        device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1)
    return grid[c.int()].view(codes.shape[0], -1, 32)


def _scaled(values, scales, K):
    """fp32 [M, K]."""
    return torch.ldexp(values, scales.int().unsqueeze(-1) - 127).view(values.shape[0], -1)[:, :K]


# ------------------------------------------------------------------- inputs ---

def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, M, dt = c["op"], c["M"], DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def activations(n):  # channels of different magnitude, as activations have them
        return (randn(M, n) * torch.exp(0.5 * randn(n))).to(dt)

    s = {"case": c}
    if op == "quantise":
        # weights or activations whose rows and channels differ in magnitude
        s["x"] = (randn(M, c["K"]) * torch.exp(randn(c["K"])) * torch.exp(randn(M, 1))).to(dt)
        return s
    if op == "product":
        K, N = c["K"], c["N"]
        s["x"] = activations(K)
        values, s["scales"] = _to_4_bits(randn(N, K) / math.sqrt(K))
        s["codes"] = _pack(values)
        s["bias"] = randn(N).to(dt) if c["bias"] else None
        return s
    H, I = c["hidden"], c["ispp"]
    s["x"] = activations(H)
    s["w13"] = (2.0 * randn(2 * I, H) / math.sqrt(H)).to(dt)
    s["w2"] = (randn(H, I) / math.sqrt(I)).to(dt)
    s["limit"] = LIMIT if c["clamp"] else None
    if op == "ffn-train":
        s["grad"] = (randn(M, H) / 16).to(dt)
    return s


# --------------------------------------------------------------- plain forms ---

def _gated(gu, I, limit):
    """``(g, u)`` clamped, ``sigmoid(g)``, and where the clamps let a gradient pass."""
    g, u = gu[:, :I], gu[:, I:]
    if limit is None:
        on_g = on_u = 1.0
    else:
        on_g, on_u = g <= limit, u.abs() <= limit
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g, u, 1.0 / (1.0 + torch.exp(-g)), on_g, on_u


def _ffn_plain(s):
    dt, I = s["x"].dtype, s["case"]["ispp"]
    x, w13, w2 = s["x"].float(), s["w13"].float(), s["w2"].float()
    g, u, sig, on_g, on_u = _gated(x @ w13.t(), I, s["limit"])
    h = g * sig * u
    out = (h @ w2.t()).to(dt)
    if s["case"]["op"] == "ffn":
        return out
    grad = s["grad"].float()
    dh = grad @ w2
    dg = dh * u * sig * (1.0 + g * (1.0 - sig)) * on_g
    du = dh * g * sig * on_u
    d = torch.cat((dg, du), 1)
    return out, (d @ w13).to(dt), (d.t() @ x).to(dt), (grad.t() @ h).to(dt)


def _product_plain(s):
    c, K = s["case"], s["case"]["K"]
    y = _scaled(*_to_4_bits(s["x"]), K) @ _scaled(_unpack(s["codes"]), s["scales"], K).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[c["dtype"]])


def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        import xkernels_amd as xk
        if op == "ffn":
            return xk.gated_ffn(s["x"], s["w13"], s["w2"], swiglu_limit=s["limit"])
        if op == "ffn-train":
            out, gate_up = xk.gated_ffn(s["x"], s["w13"], s["w2"], swiglu_limit=s["limit"], return_gate_up=True)
            return (out, *xk.gated_ffn_backward(s["grad"], s["x"], s["w13"], s["w2"], gate_up,
                                                swiglu_limit=s["limit"]))
        if op == "product":
            return xk.mxfp4_linear(s["x"], xk.Mxfp4(s["codes"], s["scales"]), bias=s["bias"])
        held = xk.mxfp4_quantize(s["x"])
        return xk.mxfp4_dequantize(held, s["x"].dtype, columns=c["K"]), held.scales
    if op == "product":
        return _product_plain(s)
    if op == "quantise":
        values, scales = _to_4_bits(s["x"])
        return _scaled(values, scales, c["K"]).to(s["x"].dtype), scales
    return _ffn_plain(s)


# --------------------------------------------------------------------- work ---

def work(c) -> dict:
    op, M, size = c["op"], c["M"], SIZES[c["dtype"]]
    if op == "quantise":
        K, nb = c["K"], -(-c["K"] // 32)
        return {"bytes": 2 * M * (K * size + 17 * nb), "flops": 4.0 * M * K}
    if op == "product":
        K, N, nb = c["K"], c["N"], -(-c["K"] // 32)
        return {"bytes": M * (K + N) * size + N * 17 * nb + N * size * bool(c["bias"]), "flops": 2.0 * M * N * K}
    H, I = c["hidden"], c["ispp"]
    if op == "ffn":
        return {"bytes": (2 * M * H + 3 * H * I) * size, "flops": 6.0 * M * H * I}
    return {"bytes": (4 * M * H + 6 * H * I) * size, "flops": 18.0 * M * H * I}


# ------------------------------------------------------------------- 64 bits ---

def _exact_4_bits(x):
    """``(values in 64 bits [M, K], scale bytes)`` by comparison with every border."""
    M, K = x.shape
    b = _blocks(x.double())
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax / 6.0)).clamp(-127, 127)
    e = torch.where(amax > 6.0 * torch.exp2(e), e + 1, e)
    e = torch.where(amax <= 6.0 * torch.exp2(e - 1), e - 1, e).clamp(-127, 127)
    v = b.abs() * torch.exp2(-e)
    q = torch.zeros_like(v)
    # a value passes to the next of the grid past the middle, or at it where the next is even
    for low, high, even in ((0, 0.5, 0), (0.5, 1, 1), (1, 1.5, 0), (1.5, 2, 1), (2, 3, 0), (3, 4, 1), (4, 6, 0)):
        middle = (low + high) / 2
        q = torch.where(v >= middle if even else v > middle, high, q)
    q = torch.where(b < 0, -q, q) * torch.exp2(e)
    return q.view(M, -1)[:, :K], (e.squeeze(-1) + 127).to(torch.uint8)


def exact(c, seed):
    s = prepare(c, seed)
    op = c["op"]
    if op == "quantise":
        return _exact_4_bits(s["x"])[0], None
    if op == "product":
        w = _unpack(s["codes"]).double() * torch.exp2(s["scales"].double() - 127).unsqueeze(-1)
        y = _exact_4_bits(s["x"])[0] @ w.view(c["N"], -1)[:, : c["K"]].t()
        return y if s["bias"] is None else y + s["bias"].double()
    x, w13, w2 = (s[k].double().requires_grad_(op == "ffn-train") for k in ("x", "w13", "w2"))
    g, u = (x @ w13.t()).chunk(2, 1)
    if s["limit"] is not None:
        g, u = torch.clamp(g, max=s["limit"]), torch.clamp(u, -s["limit"], s["limit"])
    out = (torch.nn.functional.silu(g) * u) @ w2.t()
    if op == "ffn":
        return out
    return (out.detach(), *torch.autograd.grad(out, (x, w13, w2), s["grad"].double()))
