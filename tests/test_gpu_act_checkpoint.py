"""act_checkpoint and act_restore on the GPU, bit for bit against a search over the
e4m3 values in 64 bits."""
from __future__ import annotations

import pytest
import torch

import xkernels_amd as xk
from tests._tuning_ref import checkpoint_ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check(x):
    held = xk.act_checkpoint(x)
    M, K = x.shape
    assert held.values.dtype == torch.float8_e4m3fn and held.values.shape == (M, K)
    assert held.scales.dtype == torch.uint8 and held.scales.shape == (M, -(-K // 32))
    want, scales = checkpoint_ref(x)
    assert torch.equal(held.scales.cpu(), scales)
    exact = held.values.cpu().double() * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)[:, :K]
    assert torch.equal(exact.isnan(), want.isnan())
    assert torch.equal(exact.nan_to_num(), want.nan_to_num())
    for dt in DTYPES:
        got = xk.act_restore(held, dt)
        lim = torch.finfo(dt).max
        ref = want.clamp(-lim, lim).to(dt)  # (clamp keeps NaN)
        assert torch.equal(got.cpu().isnan(), ref.isnan())
        assert torch.equal(got.cpu().nan_to_num(), ref.nan_to_num()), dt
    return held


@pytest.mark.parametrize("M,K", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 48), (7, 100), (16, 256), (100, 2880), (9, 7168),
                                 (300, 16), (64, 17)])
@pytest.mark.parametrize("dt", DTYPES)
def test_bits(M, K, dt, dev):
    g = torch.Generator().manual_seed(M + K)
    x = (torch.randn(M, K, generator=g) * torch.exp(2 * torch.randn(K, generator=g))).to(dt).cuda()
    _check(x)


def test_every_value_and_tie(dev):
    """All e4m3 values, the middles between neighbours and their next fp32 values, at many scales."""
    from tests._tuning_ref import e4m3_grid
    grid = e4m3_grid().float()
    mid = (grid[1:] + grid[:-1]) / 2
    near = torch.cat([mid, torch.nextafter(mid, torch.tensor(1e9)), torch.nextafter(mid, torch.tensor(0.0)), grid])
    near = torch.cat([near, -near])
    n = -(-near.numel() // 31)
    rows = torch.zeros(n, 32)
    rows[:, 1:].reshape(-1)
    body = torch.zeros(n * 31)
    body[: near.numel()] = near
    rows[:, 1:] = body.view(n, 31)
    rows[:, 0] = 448.0  # every block's scale is 1
    for e in (0, 1, -30, 90, -110):
        _check((rows * 2.0 ** e).cuda())


@pytest.mark.parametrize("dt", DTYPES)
def test_extremes(dt, dev):
    f = torch.finfo(dt)
    x = torch.zeros(10, 64, dtype=dt)
    x[0, 3] = f.max
    x[1, :] = f.smallest_normal
    x[2, 5], x[2, 40] = f.smallest_normal * f.eps, -f.smallest_normal * f.eps  # the least steps
    x[3, 1], x[3, 2] = float("inf"), 3.0
    x[4, 1], x[4, 33] = float("nan"), -2.0
    x[5] = float("-inf")
    x[6, 0], x[6, 1:32] = f.max, 1.0
    x[7] = -0.0
    x[8, 0] = f.min
    _check(x.cuda())


def test_rows_apart_and_unaligned(dev):
    x = torch.randn(40, 96).bfloat16().cuda()
    want = xk.act_checkpoint(x)
    for off in (16, 5):
        wide = torch.full((40, 160), float("nan"), dtype=torch.bfloat16, device="cuda")
        wide[:, off:off + 96] = x
        got = xk.act_checkpoint(wide[:, off:off + 96])
        assert torch.equal(got.values.view(torch.uint8), want.values.view(torch.uint8))
        assert torch.equal(got.scales, want.scales)
    t = xk.act_checkpoint(x.t().contiguous().t())
    assert torch.equal(t.values.view(torch.uint8), want.values.view(torch.uint8))


def test_empty(dev):
    held = xk.act_checkpoint(torch.empty(0, 40, device="cuda"))
    assert held.values.shape == (0, 40) and held.scales.shape == (0, 2)
    assert xk.act_restore(held).shape == (0, 40)


def test_more_than_32_bits_of_values(dev):
    """Rows past 2^31 values: the last ones as the first."""
    M, K = 70000, 32768
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    row = torch.randn(K).bfloat16().cuda()
    x[0], x[-1] = row, row
    held = xk.act_checkpoint(x)
    assert torch.equal(held.values[0].view(torch.uint8), held.values[-1].view(torch.uint8))
    assert held.values[-1].view(torch.uint8).any()
    back = xk.act_restore(held)
    assert torch.equal(back[0], back[-1]) and not back[1].any() and not back[-2].any()
