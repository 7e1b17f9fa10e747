"""The gated feed-forward block and its gradients against their 64-bit forms."""
from __future__ import annotations

import pytest
import torch

import xkernels_amd as xk
from tests._dense_ref import ffn_grad_ref, ffn_ref
from tests._tuning_ref import check

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _nan_in_free_memory():
    """What the allocator hands out next holds NaN: scratch that is read before it is written shows."""
    if torch.cuda.is_available():
        for n in (1 << 12, 1 << 18, 1 << 22, 1 << 25):
            torch.full((n,), float("nan"), device="cuda")


BF, FP16 = torch.bfloat16, torch.float16


def _inputs(M, H, I, dt, seed=0, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, H, generator=g) * torch.exp(0.5 * torch.randn(H, generator=g))).to(dt)
    w13 = (scale * torch.randn(2 * I, H, generator=g) / H ** 0.5).to(dt)
    w2 = (torch.randn(H, I, generator=g) / I ** 0.5).to(dt)
    dy = (torch.randn(M, H, generator=g) / 16).to(dt)
    return tuple(t.cuda() for t in (x, w13, w2, dy))


SIZES = [(1, 64, 32), (1, 7168, 256), (2, 33, 7), (3, 8, 1), (16, 256, 128), (17, 1, 40), (33, 520, 65), (64, 1024, 136),
         (100, 1001, 333), (129, 136, 130), (200, 72, 1000), (300, 640, 256), (513, 320, 264), (1023, 200, 96)]


@pytest.mark.parametrize("dt", [BF, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("M,H,I", SIZES)
def test_forward(M, H, I, dt, dev):
    x, w13, w2, _ = _inputs(M, H, I, dt, M)
    limit = 2.5 if M % 2 else None
    out, gu = xk.gated_ffn(x, w13, w2, swiglu_limit=limit, return_gate_up=True)
    want, gu_want, bound, gu_bound = ffn_ref(x, w13, w2, limit)
    assert gu.dtype == torch.float32
    check(gu, gu_want, gu_bound, "gate_up")
    check(out, want, bound, "out")
    assert torch.equal(out, xk.gated_ffn(x, w13, w2, swiglu_limit=limit))


@pytest.mark.parametrize("dt", [BF, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("M,H,I", SIZES)
@pytest.mark.parametrize("recompute", [False, True])
def test_backward(M, H, I, dt, recompute, dev):
    x, w13, w2, dy = _inputs(M, H, I, dt, M + 1)
    limit = None if M % 2 else 2.5
    gu = None if recompute else xk.gated_ffn(x, w13, w2, swiglu_limit=limit, return_gate_up=True)[1]
    got = xk.gated_ffn_backward(dy, x, w13, w2, gu, swiglu_limit=limit)
    want, bounds = ffn_grad_ref(dy, x, w13, w2, limit)
    for name, p, q, b in zip(("grad_x", "grad_w13", "grad_w2"), got, want, bounds):
        check(p, q, b, name)


# Sizes at which every tile and every way of cutting k is taken by one of the six products: 256 x 256 and
# 256 x 224 tiles, two 128 x 128 ones to a CU, slices of all tiles and of a last round's.
LARGE = [(2048, 2304, 3584), (8000, 1800, 1030), (2100, 4096, 2000), (4064, 1024, 3584), (4096, 7168, 256), (900, 2880, 1440),
         (4090, 2080, 4100)]


@pytest.mark.parametrize("M,H,I", LARGE)
def test_large(M, H, I, dev):
    x, w13, w2, dy = _inputs(M, H, I, BF, M)
    out, gu = xk.gated_ffn(x, w13, w2, swiglu_limit=6.0, return_gate_up=True)
    want, gu_want, bound, gu_bound = ffn_ref(x, w13, w2, 6.0)
    check(gu, gu_want, gu_bound, "gate_up")
    check(out, want, bound, "out")
    del want, gu_want, bound, gu_bound
    got = xk.gated_ffn_backward(dy, x, w13, w2, gu, swiglu_limit=6.0)
    want, bounds = ffn_grad_ref(dy, x, w13, w2, 6.0)
    for name, p, q, b in zip(("grad_x", "grad_w13", "grad_w2"), got, want, bounds):
        check(p, q, b, name)
    again = xk.gated_ffn_backward(dy, x, w13, w2, gu, swiglu_limit=6.0)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("dt", [BF, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("M,H,I", [(1, 1024, 2048), (2, 520, 65), (7, 96, 1001), (8, 256, 4100), (3, 8, 1)])
def test_few_tokens_keep_what_rounding_leaves(M, H, I, dt, dev):
    x, w13, w2, _ = _inputs(M, H, I, dt, M + 2)
    want, _, bound, _ = ffn_ref(x, w13, w2, 8.0, pair=True)
    check(xk.gated_ffn(x, w13, w2, swiglu_limit=8.0), want, bound, "out")


# Rows of a few values, with lengths a little past whole chunks of 64: the tile's columns are many rows of the
# operand, and nothing behind its last row may be read, let alone count.
@pytest.mark.parametrize("M,H,I", [(65, 8, 8), (129, 8, 24), (66, 24, 8), (193, 16, 33), (321, 40, 72), (130, 65, 65)])
def test_narrow(M, H, I, dev):
    x, w13, w2, dy = _inputs(M, H, I, BF, M)
    want, bounds = ffn_grad_ref(dy, x, w13, w2, None)
    padded = []
    for t in (x, w13, w2, dy):  # each before a stretch of NaN
        held = torch.full((t.numel() + 4096,), float("nan"), dtype=t.dtype, device=t.device)
        held[:t.numel()] = t.reshape(-1)
        padded.append(held[:t.numel()].view_as(t))
    x, w13, w2, dy = padded
    for name, p, q, b in zip(("grad_x", "grad_w13", "grad_w2"), xk.gated_ffn_backward(dy, x, w13, w2), want, bounds):
        check(p, q, b, name)


def test_gradient_against_differences(dev):
    """The gradients against differences of the 64-bit form along random directions."""
    x, w13, w2, dy = _inputs(40, 96, 48, BF, 5)
    got = xk.gated_ffn_backward(dy, x, w13, w2)
    args = [t.double().cpu() for t in (x, w13, w2)]
    g = torch.Generator().manual_seed(1)

    def value(a):
        gu = a[0] @ a[1].t()
        return ((torch.nn.functional.silu(gu[:, :48]) * gu[:, 48:]) @ a[2].t() * dy.double().cpu()).sum()

    _, bounds = ffn_grad_ref(dy, x, w13, w2)
    for n in range(3):
        step = torch.randn(args[n].shape, generator=g, dtype=torch.float64)
        plus, minus = list(args), list(args)
        plus[n], minus[n] = args[n] + 1e-5 * step, args[n] - 1e-5 * step
        slope = (value(plus) - value(minus)) / 2e-5
        mine = got[n].double().cpu()
        off = ((bounds[n].cpu() + 2.0 ** -8 * mine.abs()) * step.abs()).sum() + 1e-6 * slope.abs() + 1e-6
        assert abs((mine * step).sum() - slope) <= off


def test_no_tokens(dev):
    x, w13, w2, dy = _inputs(4, 64, 32, BF)
    out, gu = xk.gated_ffn(x[:0], w13, w2, return_gate_up=True)
    assert out.shape == (0, 64) and gu.shape == (0, 64)
    for keep in (None, gu):
        gx, g13, g2 = xk.gated_ffn_backward(dy[:0], x[:0], w13, w2, keep)
        assert gx.shape == (0, 64) and not g13.any() and not g2.any()


@pytest.mark.parametrize("M", [5, 70])
def test_rows_apart_and_odd_addresses(M, dev):
    H, I = 200, 72
    x, w13, w2, dy = _inputs(M, H, I, BF, 3)
    want = xk.gated_ffn(x, w13, w2)
    grads = xk.gated_ffn_backward(dy, x, w13, w2)

    def placed(t, ld, first):  # rows ld apart, from `first` values into a buffer of NaN
        buf = torch.full((t.shape[0] * ld + first + 8,), float("nan"), dtype=t.dtype, device=t.device)
        v = buf[first:first + t.shape[0] * ld].view(t.shape[0], ld)[:, :t.shape[1]]
        v.copy_(t)
        return v

    for ld, first in ((208, 0), (208, 8), (203, 0), (216, 3)):
        xs, dys = placed(x, ld, first), placed(dy, ld, first)
        assert torch.equal(xk.gated_ffn(xs, w13, w2), want)
        assert all(torch.equal(p, q) for p, q in zip(xk.gated_ffn_backward(dys, xs, w13, w2), grads))
    w13o, w2o = placed(w13, H, 1), placed(w2, I, 5)
    assert torch.equal(xk.gated_ffn(x, w13o, w2o), want)
    assert torch.equal(xk.gated_ffn(x.t().contiguous().t(), w13, w2), want)


@pytest.mark.parametrize("M,H,I", [(9, 64, 32), (150, 136, 200), (9, 33, 17)])
def test_what_is_not_finite_stays_in_its_row(M, H, I, dev):
    x, w13, w2, dy = _inputs(M, H, I, BF, 4)
    want = xk.gated_ffn(x, w13, w2)
    gx = xk.gated_ffn_backward(dy, x, w13, w2)[0]
    bad = x.clone()
    bad[2, H // 2], bad[7, 0] = float("nan"), float("inf")
    out = xk.gated_ffn(bad, w13, w2)
    bgx = xk.gated_ffn_backward(dy, bad, w13, w2)[0]
    keep = torch.ones(M, dtype=torch.bool)
    keep[2] = keep[7] = False
    assert torch.equal(out[keep], want[keep]) and torch.equal(bgx[keep], gx[keep])
    assert out[2].isnan().all() and bgx[2].isnan().all() and not out[7].isfinite().all()


def test_limits(dev):
    """Sums on, just under and just over the limit: clamped there, the gradient passed up to it."""
    L = 10.03  # between two bf16 values, 10 and 10.0625
    over = [9.0, 10.0, 10.028, 10.032, 10.05, 10.1, 30.0]
    H, I = 16, 8
    for sign in (1.0, -1.0):
        for gate in (True, False):
            # x = (a, b) in two bf16 parts, so that the sum lies anywhere
            v = torch.tensor(over, dtype=torch.float64) * sign
            a = v.to(BF)
            b = (v - a.double()).to(BF)
            x = torch.zeros(len(over), H, dtype=BF)
            x[:, 0], x[:, 1], x[:, 2] = a, b, 1.0
            w13 = torch.zeros(2 * I, H, dtype=BF)
            mine, other = (slice(0, I), slice(I, 2 * I)) if gate else (slice(I, 2 * I), slice(0, I))
            w13[mine, 0], w13[mine, 1], w13[other, 2] = 1.0, 1.0, 2.0
            w2 = torch.eye(H, I, dtype=BF)
            dy = torch.ones(len(over), H, dtype=BF)
            x, w13, w2, dy = (t.cuda() for t in (x, w13, w2, dy))
            out, gu = xk.gated_ffn(x, w13, w2, swiglu_limit=L, return_gate_up=True)
            want, gw, bound, _ = ffn_ref(x, w13, w2, L)
            check(out, want, bound)
            past = (gu[:, mine].double() > L) if gate else gu[:, mine].double().abs() > L
            assert torch.equal(past, gw[:, mine] > L if gate else gw[:, mine].abs() > L)
            for keep in (gu, None):
                got = xk.gated_ffn_backward(dy, x, w13, w2, keep, swiglu_limit=L)
                ref, bounds = ffn_grad_ref(dy, x, w13, w2, L)
                for p, q, bd in zip(got, ref, bounds):
                    check(p, q, bd)


@pytest.mark.parametrize("M,H,I", [(1, 256, 64), (40, 136, 72), (300, 264, 200)])
def test_captured(M, H, I, dev):
    """Captured once, replayed with new inputs between eager calls."""
    x, w13, w2, dy = _inputs(M, H, I, BF, 6)

    def step():
        out, gu = xk.gated_ffn(x, w13, w2, swiglu_limit=3.0, return_gate_up=True)
        return (out, *xk.gated_ffn_backward(dy, x, w13, w2, gu, swiglu_limit=3.0))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        for t, n in zip((x, w13, w2, dy), _inputs(M, H, I, BF, 100 + seed)):
            t.copy_(n)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, eager)), seed


def test_two_streams(dev):
    """Two calls at once do not share anything."""
    sets = [_inputs(200, 264, 136, BF, s) for s in (1, 2)]
    want = [(xk.gated_ffn(x, a, b), *xk.gated_ffn_backward(dy, x, a, b)) for x, a, b, dy in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for st, (x, a, b, dy) in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append((xk.gated_ffn(x, a, b), *xk.gated_ffn_backward(dy, x, a, b)))
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert all(torch.equal(s, t) for s, t in zip(p, q))


def test_past_32_bits(dev):
    """Rows behind 2^31 bytes of every long operand: the last ones as in a batch of their own, and the
    weights' gradients of those alone."""
    M, H, I, last = 540_000, 2048, 24, 300
    _, w13, w2, dy = _inputs(1, H, I, BF, 7)
    x = torch.zeros(M, H, dtype=BF, device="cuda")
    dys = torch.zeros(M, H, dtype=BF, device="cuda")
    xe, _, _, dye = _inputs(last, H, I, BF, 8)
    x[-last:], dys[-last:] = xe, dye
    out, gu = xk.gated_ffn(x, w13, w2, return_gate_up=True)
    want, _, bound, _ = ffn_ref(xe, w13, w2)
    check(out[-last:], want, bound)
    assert not out[:-last].any()
    got = xk.gated_ffn_backward(dys, x, w13, w2, gu)
    ref, bounds = ffn_grad_ref(dye, xe, w13, w2)
    check(got[0][-last:], ref[0], bounds[0])
    assert not got[0][:-last].any()
    for p, q, b in zip(got[1:], ref[1:], bounds[1:]):  # (the other rows' terms are zeros)
        check(p, q, b)


def test_refusals(dev):
    x, w13, w2, dy = _inputs(4, 64, 32, BF)
    gu = torch.zeros(4, 64, device="cuda")
    bad = [lambda: xk.gated_ffn(x.float(), w13.float(), w2.float()), lambda: xk.gated_ffn(x, w13.half(), w2),
           lambda: xk.gated_ffn(x[0], w13, w2), lambda: xk.gated_ffn(x[:, :32], w13, w2),
           lambda: xk.gated_ffn(x, w13[:63], w2), lambda: xk.gated_ffn(x, w13, w2[:, :31]),
           lambda: xk.gated_ffn(x, w13, w2.cpu()), lambda: xk.gated_ffn(x, w13, w2, swiglu_limit=float("nan")),
           lambda: xk.gated_ffn_backward(dy[:3], x, w13, w2), lambda: xk.gated_ffn_backward(dy.half(), x, w13, w2),
           lambda: xk.gated_ffn_backward(dy, x, w13, w2, gu[:, :32]),
           lambda: xk.gated_ffn_backward(dy, x, w13, w2, gu[:3])]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()


def test_no_graph_is_said(dev, monkeypatch):
    from xkernels_amd.moe import hip_tuning

    monkeypatch.setattr(hip_tuning, "_told", set())
    x, w13, w2, _ = _inputs(4, 64, 32, BF)
    with pytest.warns(RuntimeWarning, match="gated_ffn records no autograd graph"):
        out = xk.gated_ffn(x, w13.requires_grad_(), w2)
    assert not out.requires_grad
