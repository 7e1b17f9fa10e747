"""The dense block's ops at values where their kernels' ways part: weights that are not finite."""
from __future__ import annotations

import pytest
import torch

import xkernels_amd as xk

pytestmark = pytest.mark.gpu
BF, FP16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dt", [BF, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("M", [1, 3, 8, 9, 16, 17])
def test_infinities_of_w2(M, dt, dev):
    """An infinity in w2 makes its column an infinity of the activation's sign, whatever rounding left of that; a
    NaN, or two infinities that meet with different signs, make a NaN. Other columns stay."""
    H, I = 64, 48
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, H, generator=g).to(dt).cuda()
    w13 = (torch.randn(2 * I, H, generator=g) / 4).to(dt).cuda()
    w2 = (torch.randn(H, I, generator=g) / 4).to(dt).cuda()
    before, gu = xk.gated_ffn(x, w13, w2, return_gate_up=True)
    h = torch.nn.functional.silu(gu[:, :I].double()) * gu[:, I:].double()
    assert (h.abs() > 1e-6).all()  # (none that the type holds as 0)
    inf = float("inf")
    w2[3, 7], w2[20, 0], w2[40, 11], w2[63, 5], w2[63, 6] = inf, -inf, float("nan"), inf, -inf
    out = xk.gated_ffn(x, w13, w2).double()
    assert torch.equal(out[:, 3], h[:, 7].sign() * inf) and torch.equal(out[:, 20], h[:, 0].sign() * -inf)
    assert out[:, 40].isnan().all()
    both = h[:, 5].sign() * inf + h[:, 6].sign() * -inf
    assert torch.equal(out[:, 63].isnan(), both.isnan()) and torch.equal(out[:, 63].nan_to_num(), both.nan_to_num())
    rest = [c for c in range(H) if c not in (3, 20, 40, 63)]
    assert torch.equal(out[:, rest], before[:, rest].double())
