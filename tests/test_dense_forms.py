"""What the dense block's documentation says of its numbers, held against the forms that the kernels are
tested with, on the CPU."""
from __future__ import annotations

import ctypes

import torch

import xkernels_amd as xk
from oracle import dense_ref as o


def test_mxfp4_error():
    """A value is off by at most a fifth of itself (5 of the scale becomes 4) or, below the scale, by a
    quarter of that."""
    x = torch.linspace(-6, 6, 31 * 4001).view(-1, 31)
    x = torch.cat((x, torch.full((x.shape[0], 1), 6.0)), 1)  # (each block's scale is 1)
    codes, scales = o.mxfp4_quantize_ref(x)
    assert (scales == 127).all()
    off, size = (o._values(codes, scales) - x.double()).abs(), x.double().abs()
    assert (off <= torch.where(size < 1, 0.25, size / 5) * (1 + 1e-12)).all()
    row = torch.zeros(1, 32)
    row[0, :4] = torch.tensor([6.0, 5.0, 2.5, 1.25])
    assert o._values(*o.mxfp4_quantize_ref(row))[0, :4].tolist() == [6.0, 4.0, 2.0, 1.0]
    assert "off by at most a fifth of" in " ".join(xk.mxfp4_quantize.__doc__.split())


def test_the_least_limits_still_clamp():
    """A limit that fp32 would hold as 0, which means none."""
    from xkernels_amd.moe.hip_dense import _limit

    for limit in (5e-324, 1e-50, 2.0 ** -150, 2.0 ** -149, 1e-40, 7.0):
        assert 0 < ctypes.c_float(_limit("gated_ffn", limit)).value <= max(limit, 2.0 ** -149) * 1.001
    assert [_limit("gated_ffn", v) for v in (None, 0.0, -1.0, -5e-324)] == [0.0] * 4
