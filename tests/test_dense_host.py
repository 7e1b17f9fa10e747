"""The dense block's ops without a GPU: the C entry points reject bad arguments before any
launch, the size queries take any numbers, the Python ops reject CPU tensors; the oracle
against the 64-bit forms that the GPU tests compare with, and those against autograd."""
from __future__ import annotations

import pytest
import torch

import xkernels_amd as xk
from oracle import dense_ref as o
from tests._dense_ref import GRID, ffn_grad_ref, ffn_ref, linear_ref, mxfp4_ref, mxfp4_values
from xkernels_amd import _dispatch, _lib, verify
from xkernels_amd.registry import all_cards, all_specs, cost_model, input_gen, load_shape_sweep, reference_callable

P = 0x1000  # a pointer that no refused call follows
BF, FP32, FP16 = _lib.XK_DT_BF16, _lib.XK_DT_FP32, _lib.XK_DT_FP16
INVALID, WORKSPACE = _lib.XK_ERR_INVALID, _lib.XK_ERR_WORKSPACE
NAMES = ("gated_ffn", "gated_ffn_backward", "mxfp4_quantize", "mxfp4_dequantize", "mxfp4_linear")
OPS = [f"{k}@1.0.0" for k in NAMES]


def _rc(name, *args):
    return getattr(_lib.load(), name)(*args)


def test_registered():
    for name in NAMES:
        assert xk.Backend.HIP in _dispatch.registered_backends(name) and name in xk.__all__


@pytest.mark.parametrize("op", OPS)
def test_registry(op):
    assert {"HIP", "REFERENCE"} <= set(all_cards()[op])
    for p in load_shape_sweep(all_specs()[op].shape_sweep):
        flops, nbytes = cost_model.cost_model(op, p)
        assert flops > 0 and nbytes > 0
        assert callable(reference_callable(op)) and input_gen.generate_inputs(op, p, 7, "cpu")
    r = verify(op.replace("@", ".reference@"), arch="any")
    assert r["compiled"] and r["correctness"]["passed"], r
    if not torch.cuda.is_available():
        r = verify(op.replace("@", ".hip@"), arch="amd_cdna4")
        assert r["compiled"] is False and "device" in r["artifacts"]["error"]


@pytest.mark.parametrize("op", OPS)
def test_oracle_leaves_its_inputs_alone(op):
    for p in load_shape_sweep(all_specs()[op].shape_sweep):
        f = input_gen.generate_inputs(op, p, 3, "cpu")
        flat = [t for v in f.values() for t in (v if isinstance(v, tuple) else (v,)) if torch.is_tensor(t)]
        before = [t.clone() for t in flat]
        reference_callable(op)(**f)
        assert all(torch.equal(t, b) for t, b in zip(flat, before)), p


# ------------------------------------------------------------------ refusals ----

def _ffn(dtype=BF, ldx=64, M=8, H=64, I=32, x=P, w13=P, w2=P, out=P, gu=None, ws=P, ws_bytes=1 << 40):
    return _rc("xk_gated_ffn", x, dtype, ldx, M, H, w13, w2, I, 0.0, out, gu, ws, ws_bytes, None)


BAD = [dict(dtype=FP32), dict(dtype=7), dict(M=-1), dict(M=1 << 29), dict(H=0), dict(I=0), dict(H=1000001),
       dict(I=500001), dict(M=(1 << 29) - 1, H=1000000, ldx=1000000), dict(x=None), dict(w13=None), dict(w2=None),
       dict(x=P + 8), dict(w13=P + 2), dict(w2=P + 8), dict(ldx=63), dict(ldx=68), dict(ldx=2000008), dict(ws=P + 16)]


@pytest.mark.parametrize("kw", BAD + [dict(out=None)])
def test_ffn_refuses(kw):
    assert _ffn(**kw) == INVALID and _lib.last_error()


def test_ffn_workspace():
    assert _ffn(ws=None) == WORKSPACE and _ffn(ws_bytes=16) == WORKSPACE
    assert _ffn(M=0, x=None, out=None, ws=None) == _lib.XK_OK


def _grad(dtype=BF, ldg=64, ldx=64, M=8, H=64, I=32, dy=P, x=P, w13=P, w2=P, gu=None, gx=P, g13=P, g2=P, ws=P,
          ws_bytes=1 << 40):
    return _rc("xk_gated_ffn_backward", dy, dtype, ldg, x, ldx, M, H, w13, w2, I, gu, 0.0, gx, g13, g2, ws, ws_bytes,
               None)


@pytest.mark.parametrize("kw", BAD + [dict(dy=None), dict(gx=None), dict(g13=None), dict(g2=None), dict(dy=P + 4),
                                      dict(ldg=60), dict(ldg=65), dict(ldg=3000000)])
def test_ffn_backward_refuses(kw):
    assert _grad(**kw) == INVALID and _lib.last_error()


def test_ffn_backward_workspace():
    assert _grad(ws_bytes=64) == WORKSPACE
    need = [_lib.query("xk_gated_ffn_backward_workspace_bytes", 4096, 512, 256, r) for r in (0, 1)]
    assert need[1] >= need[0] + 4096 * 512 * 4


@pytest.mark.parametrize("args", [(P, 7, 32, 4, 32, P, P), (P, BF, 32, -1, 32, P, P), (P, BF, 32, 4, 0, P, P),
                                  (P, BF, 32, 1 << 40, 32, P, P), (P, BF, 32, 1 << 28, 32, P, P), (P, BF, 1 << 23, 4, (1 << 22) + 1, P, P),
                                  (None, BF, 32, 4, 32, P, P), (P, BF, 32, 4, 32, None, P), (P, BF, 32, 4, 32, P, None),
                                  (P, BF, 31, 4, 32, P, P)])
def test_quantize_refuses(args):
    assert _rc("xk_mxfp4_quantize", *args, None) == INVALID and _lib.last_error()


@pytest.mark.parametrize("args", [(P, P, 4, 32, 9, P), (P, P, -4, 32, BF, P), (P, P, 1 << 28, 1, BF, P), (P, P, 4, 0, BF, P), (None, P, 4, 32, BF, P),
                                  (P, None, 4, 32, BF, P), (P, P, 4, 32, BF, None)])
def test_dequantize_refuses(args):
    assert _rc("xk_mxfp4_dequantize", *args, None) == INVALID and _lib.last_error()


def _linear(x=P, dtype=BF, ldx=64, xs=None, M=40, K=64, wc=P, ws=P, N=32, bias=None, out=P, odt=BF, scratch=P,
            scratch_bytes=1 << 40):
    return _rc("xk_mxfp4_linear", x, dtype, ldx, xs, M, K, wc, ws, N, bias, out, odt, scratch, scratch_bytes, None)


@pytest.mark.parametrize("kw", [dict(dtype=5), dict(odt=-1), dict(M=-1), dict(M=1 << 29), dict(K=0), dict(K=1000001),
                                dict(N=0), dict(N=1000001), dict(M=(1 << 29) - 1, N=1000000), dict(M=1 << 28, N=1), dict(x=None), dict(wc=None),
                                dict(ws=None), dict(out=None), dict(ldx=63), dict(wc=P + 8), dict(ws=P + 2),
                                dict(xs=P + 1, dtype=-1), dict(xs=P, x=P + 4), dict(scratch=P + 128)])
def test_linear_refuses(kw):
    assert _linear(**kw) == INVALID and _lib.last_error()


def test_linear_workspace():
    assert _linear(scratch=None) == WORKSPACE and _linear(scratch_bytes=1) == WORKSPACE
    assert _lib.query("xk_mxfp4_linear_workspace_bytes", 16, 4096, 4096) == 0  # one launch


def test_size_queries_take_any_numbers():
    for bad in (-1, 0, 1 << 62):
        assert _lib.query("xk_gated_ffn_workspace_bytes", 8, bad, 8) == 0
        assert _lib.query("xk_gated_ffn_backward_workspace_bytes", 8, 8, bad, 1) == 0
        assert _lib.query("xk_mxfp4_linear_workspace_bytes", 8, bad, 8) == 0
    assert _lib.query("xk_gated_ffn_workspace_bytes", 0, 64, 64) == 0
    assert _lib.query("xk_gated_ffn_backward_workspace_bytes", 0, 64, 64, 0) == 0


def test_workspaces_are_not_larger_than_they_need_be():
    """Aligned sizes of large batches: the activations, no copies, no slices of k."""
    M, H, I = 8192, 4096, 2048
    assert _lib.query("xk_gated_ffn_workspace_bytes", M, H, I) == M * I * 2
    assert _lib.query("xk_gated_ffn_backward_workspace_bytes", M, H, I, 0) == M * I * 6
    assert _lib.query("xk_mxfp4_linear_workspace_bytes", M, H, 4096) == M * H // 2 + M * H // 32


def test_ops_refuse_cpu_tensors():
    x, w13, w2 = torch.randn(4, 8).bfloat16(), torch.randn(12, 8).bfloat16(), torch.randn(8, 6).bfloat16()
    held = xk.Mxfp4(*o.mxfp4_quantize_ref(torch.randn(3, 8)))
    calls = [lambda: xk.gated_ffn(x, w13, w2, backend="hip"), lambda: xk.gated_ffn_backward(x, x, w13, w2, backend="hip"),
             lambda: xk.mxfp4_quantize(x, backend="hip"), lambda: xk.mxfp4_dequantize(held, backend="hip"),
             lambda: xk.mxfp4_linear(x, held, backend="hip"), lambda: xk.mxfp4_linear(held, held, backend="hip")]
    for call in calls:
        with pytest.raises(RuntimeError, match="device"):
            call()


# ------------------------------------------------------------- the 64-bit forms ----

@pytest.mark.parametrize("limit", [None, 0.8])
def test_ffn_forms_against_autograd(limit):
    g = torch.Generator().manual_seed(0)
    x, w13, w2, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((9, 7), (10, 7), (7, 5), (9, 7)))
    args = [t.clone().requires_grad_() for t in (x, w13, w2)]
    a, b = (args[0] @ args[1].t()).chunk(2, 1)
    if limit:
        a, b = a.clamp(max=limit), b.clamp(-limit, limit)
    y = (torch.nn.functional.silu(a) * b) @ args[2].t()
    out, gu, _, _ = ffn_ref(x, w13, w2, limit)
    torch.testing.assert_close(out, y.detach())
    torch.testing.assert_close(gu, x @ w13.t())
    want = torch.autograd.grad(y, args, dy)
    for p, q in zip(ffn_grad_ref(dy, x, w13, w2, limit)[0], want):
        torch.testing.assert_close(p, q)
    x, w13, w2, dy = (t.float() for t in (x, w13, w2, dy))
    got, kept = o.gated_ffn_ref(x, w13, w2, limit, True)
    torch.testing.assert_close(got.double(), out, rtol=1e-5, atol=1e-5)
    for keep in (None, kept):
        for p, q in zip(o.gated_ffn_backward_ref(dy, x, w13, w2, keep, limit), want):
            torch.testing.assert_close(p.double(), q, rtol=1e-4, atol=1e-5)


def test_mxfp4_forms():
    x = torch.tensor([[6.0, 0.25, -0.75, 2.5, 5.0, 3.5, -1.25] + [0.0] * 25, [6.5, 1.0, 0.5] + [0.0] * 29,
                      [float("inf")] + [1.0] * 31])
    q, s = mxfp4_ref(x)
    assert s.tolist() == [[127], [128], [255]] and q[2].isnan().all()
    assert q[0, :7].tolist() == [6.0, 0.0, -1.0, 2.0, 4.0, 4.0, -1.0]  # ties to the even code
    assert q[1, :3].tolist() == [6.0, 1.0, 0.0]  # 3.25, 0.5 and 0.25 of the scale 2
    codes = torch.arange(16, dtype=torch.uint8)
    held = (codes[::2] | codes[1::2] << 4).repeat(2).view(1, 16), torch.tensor([[127]], dtype=torch.uint8)
    assert mxfp4_values(held)[0, :16].tolist() == [*GRID.tolist(), *(-GRID).tolist()]


def test_mxfp4_oracle():
    x = torch.randn(40, 100, generator=torch.Generator().manual_seed(1)) * torch.logspace(-44, 38, 40).unsqueeze(1)
    x[3, 5], x[7, 99], x[9] = float("nan"), float("-inf"), 0.0
    held = o.mxfp4_quantize_ref(x)
    want, scales = mxfp4_ref(x)
    assert torch.equal(held[1], scales)
    got = mxfp4_values(held)[:, :100]
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(o.mxfp4_dequantize_ref(held, torch.float32, 100).double(), want, rtol=0, atol=0,
                               equal_nan=True)
    a, w = torch.randn(6, 64), o.mxfp4_quantize_ref(torch.randn(5, 64))
    want, _ = linear_ref(mxfp4_ref(a)[0], mxfp4_values(w), a[0, :5])
    torch.testing.assert_close(o.mxfp4_linear_ref(a, w, a[0, :5]).double(), want, rtol=1e-5, atol=1e-5)


def test_linear_weight_without_scales_is_refused():
    codes = torch.zeros(8, 32, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="Mxfp4"):
        xk.mxfp4_linear(torch.zeros(2, 64), codes, backend="hip")
