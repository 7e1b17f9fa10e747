"""MXFP4 quantisation, its way back and the product of quantised operands against their
64-bit forms."""
from __future__ import annotations

import pytest
import torch

import xkernels_amd as xk
from tests._dense_ref import GRID, linear_ref, mxfp4_ref, mxfp4_values
from tests._tuning_ref import check, gamma

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _nan_in_free_memory():
    """What the allocator hands out next holds NaN: scratch that is read before it is written shows."""
    if torch.cuda.is_available():
        for n in (1 << 12, 1 << 18, 1 << 22, 1 << 25):
            torch.full((n,), float("nan"), device="cuda")


BF, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF, FP16, FP32]
IDS = ["bf16", "fp16", "fp32"]


def _values(shape, dt, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(spread * torch.randn(shape[-1], generator=g))
    return x.to(dt).cuda()


def _same(held, want, scales):
    got = mxfp4_values(held)[..., : want.shape[-1]]
    assert torch.equal(held.scales.cpu(), scales)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33), (7, 100), (64, 2880), (33, 1001), (2, 3, 64), (96,),
                                   (4, 1, 50), (300, 7168)])
def test_quantize(shape, dt, dev):
    x = _values(shape, dt, 1, 3.0)
    held = xk.mxfp4_quantize(x)
    want, scales = mxfp4_ref(x)
    assert isinstance(held, xk.Mxfp4) and held.codes.shape == (*shape[:-1], 16 * scales.shape[-1])
    _same(held, want, scales)
    K = shape[-1]
    codes = torch.stack((held.codes & 15, held.codes >> 4), -1).reshape(*shape[:-1], -1)
    assert not codes[..., K:].any()  # the last block's rest
    for out in TYPES:
        back = xk.mxfp4_dequantize(held, out, columns=K)
        top = torch.finfo(out).max
        assert back.dtype == out
        torch.testing.assert_close(back.double().cpu(), want.clamp(-top, top).to(out).double(), rtol=0, atol=0,
                                   equal_nan=True)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_every_border(dt, dev):
    """Each grid value, the middles and their neighbours, both signs, under several scales; and each
    largest value around the step to the next scale."""
    mid = (GRID[1:] + GRID[:-1]) / 2
    e = torch.finfo(dt).eps
    v = torch.cat([GRID, mid, mid * (1 - e), mid * (1 + e)])
    v = torch.cat([v, -v])
    rows = []
    for exp in (-14, -3, 0, 9):
        for chunk in v.split(31):
            row = torch.zeros(32, dtype=torch.float64)
            row[: chunk.numel()], row[31] = chunk, 6.0
            rows.append(row * 2.0 ** exp)
        for top in (6.0, 6.0 * (1 + e), 6.0 * (1 - e), 8.0, 8 * (1 - e), 4.0, 7.0, 5.0):
            row = torch.linspace(-1, 1, 32, dtype=torch.float64)
            row[5] = top
            rows.append(row * 2.0 ** exp)
    x = torch.stack(rows).to(dt).cuda()
    _same(xk.mxfp4_quantize(x), *mxfp4_ref(x))


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_extremes(dt, dev):
    f = torch.finfo(dt)
    x = torch.zeros(12, 64, dtype=dt)
    x[1, 3], x[2, 40], x[3, 0] = f.max, -f.max, f.smallest_normal
    x[4, 7] = f.smallest_normal * f.eps  # the least denormal
    x[5, :] = torch.tensor(f.smallest_normal, dtype=dt) * 3
    x[6, 1], x[7, 33], x[8, 63] = float("inf"), float("-inf"), float("nan")
    x[9, 0], x[9, 1] = f.max, f.smallest_normal
    x[10, :] = -0.0
    x[11, 31], x[11, 32] = float("nan"), 2.0
    x = x.cuda()
    held = xk.mxfp4_quantize(x)
    want, scales = mxfp4_ref(x)
    _same(held, want, scales)
    top = f.max
    back = xk.mxfp4_dequantize(held, dt).double().cpu()
    assert torch.equal(back.nan_to_num(), want.clamp(-top, top).to(dt).double().nan_to_num())
    assert torch.equal(back.isnan(), want.isnan())


def test_every_byte_back(dev):
    """All codes under all scales, in fp32."""
    codes = torch.arange(256, dtype=torch.uint8).view(16, 16).repeat(256, 1).cuda()
    scales = torch.arange(256, dtype=torch.uint8).repeat_interleave(16).view(-1, 1).cuda()
    want = mxfp4_values((codes, scales))
    top = torch.finfo(FP32).max
    got = xk.mxfp4_dequantize(xk.Mxfp4(codes, scales), FP32).double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(), want.clamp(-top, top).nan_to_num())


def test_quantize_rows_apart(dev):
    for dt in TYPES:
        x = _values((40, 101), dt, 2)
        want = xk.mxfp4_quantize(x)
        buf = torch.full((40, 150), float("nan"), dtype=dt, device="cuda")
        for first in (0, 1, 16):
            buf[:, first:first + 101] = x
            got = xk.mxfp4_quantize(buf[:, first:first + 101])
            assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
        got = xk.mxfp4_quantize(x.t().contiguous().t())
        assert torch.equal(got.codes, want.codes)
    assert xk.mxfp4_quantize(x[:0]).codes.shape == (0, 64)
    assert xk.mxfp4_dequantize(xk.mxfp4_quantize(x[:0])).shape == (0, 128)


SIZES = [(1, 32, 1), (1, 7168, 130), (2, 33, 5), (3, 100, 17), (16, 256, 64), (17, 2880, 65), (40, 300, 129), (64, 512, 96),
         (65, 128, 33), (77, 288, 2881), (128, 1024, 128), (200, 1001, 200), (300, 640, 513), (1000, 96, 260)]


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear(M, K, N, dt, dev):
    x = _values((M, K), dt, M)
    held = xk.mxfp4_quantize(_values((N, K), BF, N) / K ** 0.5)
    bias = _values((N,), dt, 3) if M % 2 else None
    y = xk.mxfp4_linear(x, held, bias=bias)
    xv, wv = mxfp4_ref(x)[0], mxfp4_values(held)[:, :K]
    want, bound = linear_ref(xv, wv, bias)
    assert y.dtype == dt
    check(y, want, bound)
    xq = xk.mxfp4_quantize(x)
    assert torch.equal(xk.mxfp4_linear(xq, held, bias=bias, out_dtype=dt), y)
    if bias is None:
        assert xk.mxfp4_linear(xq, held).dtype == BF
        for out in TYPES:
            check(xk.mxfp4_linear(x, held, out_dtype=out), want, bound)


@pytest.mark.parametrize("M,K,N", [(4096, 2048, 4096), (8000, 520, 7160), (2500, 1024, 5200), (1000, 7168, 1024), (4090, 512, 4100)])
def test_linear_large(M, K, N, dev):
    """Every tile and way of cutting k."""
    x, w = xk.mxfp4_quantize(_values((M, K), BF, 1)), xk.mxfp4_quantize(_values((N, K), BF, 2) / K ** 0.5)
    xv, wv = mxfp4_values(x).cuda(), mxfp4_values(w).cuda()
    want = xv @ wv.t()
    check(xk.mxfp4_linear(x, w), want, gamma(K) * (xv.abs() @ wv.abs().t()))


def test_linear_far_scales(dev):
    """Rows whose scales are far apart, up to the least and the largest, in fp32."""
    M, K, N = 40, 192, 70
    x = _values((M, K), FP32, 1) * torch.logspace(-36, 36, M, device="cuda").unsqueeze(1)
    w = _values((N, K), FP32, 2)
    held = xk.mxfp4_quantize(w)
    want, bound = linear_ref(mxfp4_ref(x)[0], mxfp4_values(held))
    check(xk.mxfp4_linear(x, held), want, bound)


@pytest.mark.parametrize("M,K,N", [(9, 160, 40), (70, 64, 200), (3, 2000, 33)])
def test_linear_not_finite(M, K, N, dev):
    """A NaN or infinity makes its row NaN, a NaN block of the weight its column, nothing else; the
    bytes behind a row's last scale do not matter."""
    x, w = _values((M, K), BF, 1), _values((N, K), BF, 2)
    held = xk.mxfp4_quantize(w)
    want = xk.mxfp4_linear(x, held)
    bad = x.clone()
    bad[1, K - 1], bad[2, 0] = float("nan"), float("-inf")
    w[5, 7], w[N - 1, K - 1] = float("inf"), float("nan")
    got = xk.mxfp4_linear(bad, xk.mxfp4_quantize(w))
    rows, cols = torch.ones(M, dtype=torch.bool), torch.ones(N, dtype=torch.bool)
    rows[1] = rows[2] = cols[5] = cols[N - 1] = False
    assert torch.equal(got[rows][:, cols], want[rows][:, cols])
    assert got[~rows].isnan().all() and got[:, ~cols].isnan().all()


def test_past_32_bits(dev):
    """Rows behind 2^31 values and 2^31 bytes of codes: the last ones as in a batch of their own."""
    M, K, N, last = 1_100_000, 4096, 40, 200
    x = torch.zeros(M, K, dtype=BF, device="cuda")
    end = _values((last, K), BF, 1)
    x[-last:] = end
    q, qe = xk.mxfp4_quantize(x), xk.mxfp4_quantize(end)
    assert torch.equal(q.codes[-last:], qe.codes) and torch.equal(q.scales[-last:], qe.scales)
    back = xk.mxfp4_dequantize(q)
    assert torch.equal(back[-last:], xk.mxfp4_dequantize(qe)) and not back[:-last].any()
    del back
    w = xk.mxfp4_quantize(_values((N, K), BF, 2))
    want, bound = linear_ref(mxfp4_values(qe), mxfp4_values(w))
    for a in (x, q):
        y = xk.mxfp4_linear(a, w, out_dtype=BF)
        check(y[-last:], want, bound)
        assert not y[:-last].any()


def test_linear_odd_addresses(dev):
    x, held = _values((30, 224), BF, 1), xk.mxfp4_quantize(_values((50, 224), BF, 2))
    want = xk.mxfp4_linear(x, held)
    buf = torch.zeros(30 * 231 + 1, dtype=BF, device="cuda")[1:].view(30, 231)
    buf[:, 2:226] = x
    assert torch.equal(xk.mxfp4_linear(buf[:, 2:226], held), want)
    codes = torch.zeros(held.codes.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(held.codes.shape)
    scales = torch.zeros(held.scales.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(held.scales.shape)
    codes.copy_(held.codes), scales.copy_(held.scales)
    assert torch.equal(xk.mxfp4_linear(x, xk.Mxfp4(codes, scales)), want)
    assert torch.equal(xk.mxfp4_dequantize(xk.Mxfp4(codes, scales)), xk.mxfp4_dequantize(held))
    assert xk.mxfp4_linear(x[:0], held).shape == (0, 50)


@pytest.mark.parametrize("M", [1, 20, 200])
def test_captured(M, dev):
    x, w = _values((M, 288), BF, 1), _values((100, 288), BF, 2)

    def step():
        held = xk.mxfp4_quantize(w)
        return xk.mxfp4_linear(x, held), xk.mxfp4_dequantize(held)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for seed in range(4):
        x.copy_(_values((M, 288), BF, 10 + seed)), w.copy_(_values((100, 288), BF, 20 + seed))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(kept, eager)), seed


def test_refusals(dev):
    x, held = _values((4, 64), BF), xk.mxfp4_quantize(_values((8, 64), BF))
    c, s = held
    bad = [lambda: xk.mxfp4_quantize(x.double()), lambda: xk.mxfp4_quantize(x[:, :0]),
           lambda: xk.mxfp4_dequantize(held, torch.float64), lambda: xk.mxfp4_dequantize(held, columns=32),
           lambda: xk.mxfp4_dequantize(held, columns=65), lambda: xk.mxfp4_dequantize(xk.Mxfp4(c, s[:, :1])),
           lambda: xk.mxfp4_dequantize(xk.Mxfp4(c.int(), s)), lambda: xk.mxfp4_linear(x[:, :32], held),
           lambda: xk.mxfp4_linear(x[0], held), lambda: xk.mxfp4_linear(x.double(), held),
           lambda: xk.mxfp4_linear(x, xk.Mxfp4(c, s[:4])), lambda: xk.mxfp4_linear(x, held, bias=x[0, :8].float()),
           lambda: xk.mxfp4_linear(x, held, bias=x[0, :7]), lambda: xk.mxfp4_linear(x, held, out_dtype=torch.int32),
           lambda: xk.mxfp4_linear(x.cpu(), held), lambda: xk.mxfp4_linear(x, xk.Mxfp4(c[:0], s[:0]))]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
