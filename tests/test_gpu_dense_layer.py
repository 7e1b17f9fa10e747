"""The dense block together with the framework's own ops, as a program uses them: a training
step of a shared expert through torch's autograd, its input held in 8 bits; then that expert
and routed ones from 16 bits into MXFP4, and a serving step of both."""
from __future__ import annotations

import pytest
import torch

import xkernels_amd as xk
from oracle.torch_ref import moe_mxfp4_ref
from tests._dense_ref import ffn_grad_ref, ffn_ref, linear_ref, mxfp4_ref, mxfp4_values
from tests._tuning_ref import check
from xkernels_amd import verify, verify_parity

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
OPS = ["gated_ffn", "gated_ffn_backward", "mxfp4_quantize", "mxfp4_dequantize", "mxfp4_linear"]


@pytest.mark.parametrize("op", OPS)
def test_verify_hip_card(op, dev):
    r = verify(f"{op}.hip@1.0.0", arch="amd_cdna4", measure_perf=True)
    assert r["compiled"], r["artifacts"]
    assert r["correctness"]["passed"], r["correctness"]
    assert r["determinism_check"] and r["perf"]["ms"] > 0


@pytest.mark.parametrize("op", OPS)
def test_verify_parity_hip_vs_reference(op, dev):
    r = verify_parity(f"{op}@1.0.0", archs=["amd_cdna4"])
    assert r["n_runnable"] == 2, r["errors"]
    assert r["agree"] is True, r["diverging"]


class SharedExpert(torch.autograd.Function):
    """The block with its input held in 8 bits for the weights' gradients."""

    @staticmethod
    def forward(ctx, x, w13, w2, limit):
        out, gate_up = xk.gated_ffn(x, w13, w2, swiglu_limit=limit, return_gate_up=True)
        ctx.held, ctx.limit = xk.act_checkpoint(x), limit
        ctx.save_for_backward(w13, w2, gate_up)
        return out

    @staticmethod
    def backward(ctx, grad):
        w13, w2, gate_up = ctx.saved_tensors
        x = xk.act_restore(ctx.held, grad.dtype)
        return (*xk.gated_ffn_backward(grad, x, w13, w2, gate_up, swiglu_limit=ctx.limit), None)


def _weights(H, I, seed):
    g = torch.Generator().manual_seed(seed)
    return ((2 * torch.randn(2 * I, H, generator=g) / H ** 0.5).to(BF).cuda(),
            (torch.randn(H, I, generator=g) / I ** 0.5).to(BF).cuda())


@pytest.mark.parametrize("M", [7, 300])
def test_training_step(M, dev):
    H, I, limit = 256, 192, 3.0
    w13, w2 = _weights(H, I, 1)
    g = torch.Generator().manual_seed(M)
    x, dy = (torch.randn(M, H, generator=g).to(BF).cuda() for _ in range(2))
    leaves = [t.clone().requires_grad_() for t in (x, w13, w2)]
    y = SharedExpert.apply(*leaves, limit)
    want, _, bound, _ = ffn_ref(x, w13, w2, limit)
    check(y, want, bound)
    got = torch.autograd.grad(y, leaves, dy)
    # x itself gives the sums and thereby d and h; dW13 takes x as it was held
    ref, bounds = ffn_grad_ref(dy, x, w13, w2, limit)
    check(got[0], ref[0], bounds[0])
    check(got[2], ref[2], bounds[2])
    held = xk.act_restore(xk.act_checkpoint(x), BF)
    assert torch.equal(got[1], xk.gated_ffn_backward(dy, held, w13, w2, xk.gated_ffn(
        x, w13, w2, swiglu_limit=limit, return_gate_up=True)[1], swiglu_limit=limit)[1])
    # each held value is off by at most 2^-4 of itself or 2^-17 of its block's largest
    off = x.abs().double() * 2.0 ** -4 + x.abs().double().amax() * 2.0 ** -17
    gu = x.double() @ w13.double().t()
    a, b = gu.chunk(2, 1)
    s = torch.sigmoid(a.clamp(max=limit))
    dh = dy.double() @ w2.double()
    slope = (s * (1 + a.clamp(max=limit) * (1 - s))).abs()
    size = torch.cat((dh.abs() * b.abs().clamp(max=limit) * slope, dh.abs() * (a.clamp(max=limit) * s).abs()), 1)
    check(got[1], ref[1], bounds[1] * 1.1 + 1.02 * size.t() @ off)


def test_captured_while_an_eager_graph_lives(dev):
    """The step's backward captured while an eager graph of the same leaves waits for its own."""
    H, I, M = 128, 96, 40
    w13, w2 = _weights(H, I, 2)
    x, dy = torch.randn(M, H, device="cuda").to(BF), torch.randn(M, H, device="cuda").to(BF)
    leaves = [t.clone().requires_grad_() for t in (x, w13, w2)]
    eager = SharedExpert.apply(*leaves, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        xk.gated_ffn_backward(dy, x, w13, w2)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, gate_up = xk.gated_ffn(x, w13, w2, return_gate_up=True)
        grads = xk.gated_ffn_backward(dy, x, w13, w2, gate_up)
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x.copy_(torch.randn(M, H, device="cuda", generator=g))
        graph.replay()
        now = xk.gated_ffn_backward(dy, x, w13, w2)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(grads, now)) and torch.equal(out, xk.gated_ffn(x, w13, w2))
    got = torch.autograd.grad(eager, leaves, dy)
    assert all(t.isfinite().all() for t in got)


@pytest.mark.parametrize("M", [1, 5, 90])
def test_serving_step(M, dev):
    """Routed experts and a shared one, all quantised from 16 bits."""
    H, I, E, k = 256, 64, 8, 2
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, H, generator=g).to(BF)
    e13 = (torch.randn(E, 2 * I, H, generator=g) / 8).to(BF)
    e2 = (torch.randn(E, H, I, generator=g) / 8).to(BF)
    q13, q2 = xk.mxfp4_quantize(e13.cuda()), xk.mxfp4_quantize(e2.cuda())
    for q, w in ((q13, e13), (q2, e2)):
        want, scales = mxfp4_ref(w)
        assert torch.equal(mxfp4_values(q), want) and torch.equal(q.scales.cpu(), scales)
    w, ids = xk.topk_softmax(torch.randn(M, E, generator=g).cuda(), k)
    routed = xk.fused_moe_mxfp4(x.cuda(), *q13, *q2, ids, w)
    want = moe_mxfp4_ref(x, *(t.cpu() for t in (*q13, *q2)), ids.cpu(), w.cpu())
    torch.testing.assert_close(routed.cpu().float(), want.float(), rtol=2e-2, atol=2e-2)

    w13, w2 = _weights(H, I, 3)
    s13, s2 = xk.mxfp4_quantize(w13), xk.mxfp4_quantize(w2)
    gu = xk.mxfp4_linear(x.cuda(), s13)
    want, bound = linear_ref(mxfp4_ref(x)[0], mxfp4_values(s13))
    check(gu, want, bound)
    h = torch.nn.functional.silu(gu[:, :I]) * gu[:, I:]
    shared = xk.mxfp4_linear(h, s2)
    want, bound = linear_ref(mxfp4_ref(h)[0], mxfp4_values(s2))
    check(shared, want, bound)
    assert (routed + shared).isfinite().all()
    # the block of the values that the codes stand for, on values that they stand for
    x8 = xk.mxfp4_dequantize(xk.mxfp4_quantize(x.cuda()))
    out, kept = xk.gated_ffn(x8, xk.mxfp4_dequantize(s13), xk.mxfp4_dequantize(s2), return_gate_up=True)
    torch.testing.assert_close(kept.float(), gu.float(), rtol=2.0 ** -7, atol=2.0 ** -7)
