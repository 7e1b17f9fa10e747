"""What the dense block's documentation says of its numbers, held against the forms that the kernels are
tested with, on the CPU."""
from __future__ import annotations

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
