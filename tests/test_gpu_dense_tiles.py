"""The dense block's products in every tile and every way of cutting k, for each type, epilogue and form of the
call that is a kernel of its own, against their 64-bit forms."""
from __future__ import annotations

import pytest
import torch

import xkernels_amd as xk
from oracle.dense_ref import _values
from tests._dense_ref import ffn_grad_ref, ffn_ref
from tests._dense_sizes import FFN, MXFP4
from tests._tuning_ref import F32, gamma, half_step

pytestmark = pytest.mark.gpu
BF, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _check(got, want, bound, what):
    """As _tuning_ref.check, on the tensors' device."""
    assert got.shape == want.shape, what
    u = half_step(got.dtype)
    limit = u * want.abs() + (1 + u) * bound + torch.finfo(got.dtype).smallest_normal * 2 * u
    off = (got.double() - want).abs()
    bad = ~(off <= limit)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, {float((off / limit).nan_to_num().max()):.3g} of it"


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


@pytest.mark.parametrize("dt", [BF, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("M,H,I", FFN)
def test_feed_forward(M, H, I, dt, dev):
    """A step with the sums kept, and its gradients again with them recomputed: the same bits."""
    g = torch.Generator(device="cuda").manual_seed(M)
    x = (_randn(g, M, H) * torch.exp(0.5 * _randn(g, H))).to(dt)
    w13 = (2 * _randn(g, 2 * I, H) / H ** 0.5).to(dt)
    w2, dy = (_randn(g, H, I) / I ** 0.5).to(dt), (_randn(g, M, H) / 16).to(dt)
    limit = 6.0 if (M + H + I) % 2 else None
    out, gu = xk.gated_ffn(x, w13, w2, swiglu_limit=limit, return_gate_up=True)
    want, gu_want, bound, gu_bound = ffn_ref(x, w13, w2, limit)
    _check(gu, gu_want, gu_bound, "gate_up")
    _check(out, want, bound, "out")
    del want, gu_want, bound, gu_bound
    got = xk.gated_ffn_backward(dy, x, w13, w2, gu, swiglu_limit=limit)
    want, bounds = ffn_grad_ref(dy, x, w13, w2, limit)
    for name, p, q, b in zip(("grad_x", "grad_w13", "grad_w2"), got, want, bounds):
        _check(p, q, b, name)
    again = xk.gated_ffn_backward(dy, x, w13, w2, swiglu_limit=limit)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("M,K,N", MXFP4)
def test_mxfp4(M, K, N, dev):
    """Each type of output, with a bias and without; operands quantised in the call and before it."""
    g = torch.Generator(device="cuda").manual_seed(M)
    x = (_randn(g, M, K) * torch.exp(_randn(g, K))).to(BF)
    xq, w = xk.mxfp4_quantize(x), xk.mxfp4_quantize(_randn(g, N, K) / K ** 0.5)
    xv, wv = _values(*xq), _values(*w)
    want, off = xv @ wv.t(), gamma(K) * (xv.abs() @ wv.abs().t())
    for out in (BF, FP16, FP32):
        y = xk.mxfp4_linear(x, w, out_dtype=out)
        _check(y, want, off, out)
        assert torch.equal(xk.mxfp4_linear(xq, w, out_dtype=out), y)
        bias = _randn(g, N).to(out)
        sum_ = want + bias.double()
        _check(xk.mxfp4_linear(xq, w, bias=bias, out_dtype=out), sum_, off + F32 * (sum_.abs() + off), (out, "bias"))


@pytest.mark.parametrize("M", [12, 40, 300])
def test_mxfp4_scales_far_apart_on_both_sides(M, dev):
    """Rows of x and of the weight over all of fp32's range: what fp32 holds is right, what passes its largest value an
    infinity of the result's sign, and nothing NaN (K = 32: one block, so that no sum passes through an infinity)."""
    K, N = 32, 70
    g = torch.Generator(device="cuda").manual_seed(M)
    x = _randn(g, M, K) * torch.logspace(-37, 37, M, device="cuda").unsqueeze(1)
    w = xk.mxfp4_quantize(_randn(g, N, K) * torch.logspace(-37, 37, N, device="cuda").unsqueeze(1))
    xv, wv = _values(*xk.mxfp4_quantize(x)), _values(*w)
    want, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    y = xk.mxfp4_linear(x, w)
    top, inside = torch.finfo(FP32).max, size <= torch.finfo(FP32).max
    assert (want.abs() > 2 * top).any() and inside.any() and not y.isnan().any()
    over = want.abs() > 2 * top
    assert torch.equal(y[over], (want[over].sign() * float("inf")).float())
    _check(y[inside], want[inside], gamma(K) * size[inside] + 40 * 2.0 ** -149, "inside")  # (each sum off by a least step)
