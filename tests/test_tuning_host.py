"""Refusals of the tuning ops without a GPU: the C entry points reject bad arguments
before any launch, the size queries take any numbers, the Python ops reject CPU
tensors; and the 64-bit forms that the GPU tests compare with, against autograd."""
from __future__ import annotations

import pytest
import torch

import xkernels_amd as xk
from tests._tuning_ref import balance_ref, checkpoint_ref, e4m3_grid, lora_grad_ref, lora_ref, router_grad_ref
from xkernels_amd import _dispatch, _lib, verify
from xkernels_amd.registry import all_cards, all_specs, cost_model, input_gen, load_shape_sweep, reference_callable

P = 0x1000  # a pointer that no refused call follows
BF, FP32, FP16 = _lib.XK_DT_BF16, _lib.XK_DT_FP32, _lib.XK_DT_FP16
INVALID, WORKSPACE = _lib.XK_ERR_INVALID, _lib.XK_ERR_WORKSPACE


def _rc(name, *args):
    return getattr(_lib.load(), name)(*args)


def test_registered():
    for name in ("moe_balance_loss", "moe_router_backward", "lora_projection", "lora_projection_backward",
                 "act_checkpoint", "act_restore"):
        assert xk.Backend.HIP in _dispatch.registered_backends(name)
        assert name in xk.__all__


OPS = [f"{k}@1.0.0" for k in ("moe_balance_loss", "moe_router_backward", "lora_projection",
                              "lora_projection_backward", "act_checkpoint", "act_restore")]


@pytest.mark.parametrize("op", OPS)
def test_registry(op):
    assert {"HIP", "REFERENCE"} <= set(all_cards()[op])
    points = load_shape_sweep(all_specs()[op].shape_sweep)
    for p in points:
        flops, nbytes = cost_model.cost_model(op, p)
        assert flops > 0 and nbytes > 0
        a, b = (input_gen.generate_inputs(op, p, 7, "cpu") for _ in range(2))
        assert callable(reference_callable(op)) and a.keys() == b.keys()
    r = verify(op.replace("@", ".reference@"), arch="any")
    assert r["compiled"] and r["correctness"]["passed"], r
    if not torch.cuda.is_available():
        r = verify(op.replace("@", ".hip@"), arch="amd_cdna4")
        assert r["compiled"] is False and "device" in r["artifacts"]["error"]


def test_oracle_against_the_64_bit_forms():
    from oracle import tuning_ref as o

    f = input_gen.generate_inputs(OPS[2], load_shape_sweep("lora_projection")[3], 1, "cpu")
    out, hidden, bound, _ = lora_ref(*(f[k] for k in ("x", "lora_a", "lora_b", "adapter_ids", "base", "scaling")))
    got, gh = o.lora_projection_ref(**f, return_hidden=True)
    torch.testing.assert_close(got.double(), out, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(gh.double(), hidden, rtol=1e-5, atol=1e-5)
    f = input_gen.generate_inputs(OPS[3], load_shape_sweep("lora_projection_backward")[2], 1, "cpu")
    want, _ = lora_grad_ref(f["grad_out"], f["x"], f["lora_a"], f["lora_b"], f["adapter_ids"], f["hidden"], f["scaling"])
    for p, q in zip(o.lora_projection_backward_ref(**f), want):
        torch.testing.assert_close(p.double(), q, rtol=1e-5, atol=1e-4)
    f = input_gen.generate_inputs(OPS[0], load_shape_sweep("moe_balance_loss")[1], 1, "cpu")
    loss, counts, T = balance_ref(f["gating_output"], f["topk_ids"], f["mask"])
    got = o.moe_balance_loss_ref(**f)
    torch.testing.assert_close(got[0].double(), loss, rtol=1e-6, atol=0)
    assert torch.equal(got[1].long(), counts) and int(got[2]) == T
    for renorm in (True, False):
        f = input_gen.generate_inputs(OPS[1], load_shape_sweep("moe_router_backward")[0], 1, "cpu")
        f["renormalize"] = renorm
        f["topk_ids"][3, 1] = -1
        want, _ = router_grad_ref(f["gating_output"], f["topk_ids"], f["grad_weights"], renorm, 1.0, f["counts"])
        torch.testing.assert_close(o.moe_router_backward_ref(**f).double(), want, rtol=1e-4, atol=1e-7)
    x = torch.randn(9, 70) * 100
    x[2, 3], x[4, 60] = float("inf"), float("nan")
    want, scales = checkpoint_ref(x)
    held = o.act_checkpoint_ref(x)
    assert torch.equal(held[1], scales)
    torch.testing.assert_close(o.act_restore_ref(held, torch.float32).double(), want, rtol=0, atol=0, equal_nan=True)


def _balance(dtype=BF, M=800, E=16, k=2, logits=P, ids=P, loss=P, counts=P, tokens=P, ws=P, ws_bytes=1 << 40):
    return _rc("xk_moe_balance_loss", logits, dtype, M, E, ids, k, None, loss, counts, tokens, ws, ws_bytes, None)


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(M=-1), dict(E=0), dict(E=1 << 25), dict(k=0), dict(k=17),
                                dict(M=1 << 29, k=8), dict(logits=None), dict(ids=None), dict(loss=None),
                                dict(counts=None), dict(tokens=None), dict(ws=P + 8)])
def test_balance_loss_refuses(kw):
    assert _balance(**kw) == INVALID and _lib.last_error()


@pytest.mark.parametrize("kw", [dict(ws=None), dict(ws_bytes=16)])
def test_balance_loss_workspace(kw):
    assert _balance(**kw) == WORKSPACE


def _grad(dtype=BF, M=8, E=16, k=2, logits=P, ids=P, gl=P, counts=P, gw=P, out=P):
    return _rc("xk_moe_router_backward", logits, dtype, M, E, ids, k, None, gl, counts, None, gw, 1, out, None)


@pytest.mark.parametrize("kw", [dict(dtype=-1), dict(M=-2), dict(k=0), dict(gl=None, gw=None), dict(counts=None),
                                dict(logits=None), dict(ids=None), dict(out=None)])
def test_router_backward_refuses(kw):
    assert _grad(**kw) == INVALID and _lib.last_error()


def _lora(dtype=BF, ldx=64, M=8, K=64, L=2, N=32, r=8, x=P, a=P, b=P, ids=P, base=P, ldb=32, out=2 * P, ws=P,
          ws_bytes=1 << 40):
    return _rc("xk_lora_projection", x, dtype, ldx, M, K, a, b, L, N, r, ids, None, base, ldb, out, None, ws,
               ws_bytes, None)


@pytest.mark.parametrize("kw", [dict(dtype=FP16), dict(M=-1), dict(K=0), dict(N=0), dict(L=0), dict(L=1025), dict(r=0),
                                dict(r=129), dict(x=None), dict(a=None), dict(b=None), dict(ids=None),
                                dict(out=None), dict(ldx=63), dict(ldb=31), dict(out=P, ldb=33), dict(ws=P + 4)])
def test_lora_refuses(kw):
    assert _lora(**kw) == INVALID and _lib.last_error()


@pytest.mark.parametrize("kw", [dict(ws=None), dict(ws_bytes=16)])
def test_lora_workspace(kw):
    assert _lora(**kw) == WORKSPACE


def _lora_grad(dtype=BF, ldg=32, ldx=64, scales=None, M=8, K=64, L=2, N=32, r=8, dy=P, x=P, a=P, b=P, ids=P, h=P,
               gx=P, ga=P, gb=P, ws=P, ws_bytes=1 << 40):
    return _rc("xk_lora_projection_backward", dy, dtype, ldg, x, ldx, scales, M, K, a, b, L, N, r, ids, None, h, gx, ga,
               gb, ws, ws_bytes, None)


@pytest.mark.parametrize("kw", [dict(dtype=FP16), dict(M=-1), dict(L=0), dict(r=129), dict(dy=None), dict(x=None),
                                dict(a=None), dict(b=None), dict(ids=None), dict(h=None), dict(gx=None),
                                dict(ga=None), dict(gb=None), dict(ldg=31), dict(ldx=63), dict(scales=P, ldx=72),
                                dict(ws=P + 8)])
def test_lora_backward_refuses(kw):
    assert _lora_grad(**kw) == INVALID and _lib.last_error()


def test_lora_backward_workspace():
    assert _lora_grad(ws_bytes=64) == WORKSPACE


@pytest.mark.parametrize("args", [(P, 7, 32, 4, 32, P, P), (P, BF, 32, -1, 32, P, P), (P, BF, 32, 4, 0, P, P),
                                  (None, BF, 32, 4, 32, P, P), (P, BF, 32, 4, 32, None, P), (P, BF, 31, 4, 32, P, P)])
def test_checkpoint_refuses(args):
    assert _rc("xk_act_checkpoint", *args, None) == INVALID and _lib.last_error()


@pytest.mark.parametrize("args", [(P, P, 4, 32, 9, P), (P, P, -4, 32, BF, P), (P, None, 4, 32, BF, P),
                                  (P, P, 4, 32, BF, None)])
def test_restore_refuses(args):
    assert _rc("xk_act_restore", *args, None) == INVALID and _lib.last_error()


def test_size_queries_take_any_numbers():
    for bad in (-1, 0, 1 << 62):
        assert _lib.query("xk_lora_projection_workspace_bytes", 8, bad, 2, 8) == 0
        assert _lib.query("xk_lora_projection_workspace_bytes", 8, 64, 2, bad) == 0
        assert _lib.query("xk_lora_projection_backward_workspace_bytes", 8, 64, 64, bad, 8, BF) == 0
        assert _lib.query("xk_moe_balance_loss_workspace_bytes", 8, bad) == 0
    assert _lib.query("xk_moe_balance_loss_workspace_bytes", 256, 512) == 0  # one workgroup needs none
    assert _lib.query("xk_moe_balance_loss_workspace_bytes", 257, 512) > 0
    assert _lib.query("xk_lora_projection_workspace_bytes", 8, 64, 2, 8) > 0
    assert _lib.query("xk_lora_projection_backward_workspace_bytes", 0, 64, 64, 2, 8, BF) > 0


def test_ops_refuse_cpu_tensors():
    z, ids = torch.randn(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    x, a, b = torch.randn(4, 8), torch.randn(2, 4, 8), torch.randn(2, 6, 4)
    calls = [lambda: xk.moe_balance_loss(z, ids, backend="hip"),
             lambda: xk.moe_router_backward(z, ids, grad_weights=torch.randn(4, 2), backend="hip"),
             lambda: xk.lora_projection(x, a, b, ids[:, 0], backend="hip"),
             lambda: xk.lora_projection_backward(torch.randn(4, 6), x, a, b, ids[:, 0], torch.randn(4, 4), backend="hip"),
             lambda: xk.act_checkpoint(x, backend="hip"),
             lambda: xk.act_restore(xk.ActCheckpoint(x.to(torch.float8_e4m3fn), ids[:, :1].to(torch.uint8)), backend="hip")]
    for call in calls:
        with pytest.raises(RuntimeError, match="device"):
            call()


# ------------------------------------------------------------ the 64-bit forms ----

def test_lora_forms_against_autograd():
    g = torch.Generator().manual_seed(0)
    x, a, b = (torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((9, 7), (3, 2, 7), (3, 5, 2)))
    ids, sc = torch.tensor([0, 2, 2, -1, 0, 5, 2, 0, 0]), torch.tensor([0.5, 2.0, 3.0], dtype=torch.float64)
    dy = torch.randn(9, 5, generator=g, dtype=torch.float64)
    rows = [m for m in range(9) if 0 <= ids[m] < 3]
    y = torch.stack([sc[ids[m]] * (x[m] @ a[ids[m]].t()) @ b[ids[m]].t() if m in rows else x.new_zeros(5) for m in range(9)])
    want = torch.autograd.grad((y * dy).sum(), (x, a, b))
    out, hidden, _, _ = lora_ref(x.detach(), a.detach(), b.detach(), ids, None, sc)
    torch.testing.assert_close(out, y.detach())
    got, _ = lora_grad_ref(dy, x.detach(), a.detach(), b.detach(), ids, hidden, sc)
    for p, q in zip(got, want):
        torch.testing.assert_close(p, q)


@pytest.mark.parametrize("renorm", [True, False])
def test_router_forms_against_autograd(renorm):
    g = torch.Generator().manual_seed(1)
    z = torch.randn(6, 10, generator=g, dtype=torch.float64, requires_grad=True)
    ids = torch.topk(z.detach(), 3, dim=1).indices
    u = torch.randn(6, 3, generator=g, dtype=torch.float64)
    mask = torch.tensor([1, 1, 0, 1, 1, 1], dtype=torch.bool)
    loss, counts, T = balance_ref(z.detach(), ids, mask)
    p = torch.softmax(z, 1)
    w = p.gather(1, ids)
    w = w / w.sum(1, keepdim=True) if renorm else w
    L = 10 / (T * T * 3) * (counts.double() @ p[mask].sum(0))
    torch.testing.assert_close(L.detach(), loss)
    want, = torch.autograd.grad(0.3 * L + (w * u)[mask].sum(), z)
    got, _ = router_grad_ref(z.detach(), ids, u, renorm, torch.tensor(0.3, dtype=torch.float64), counts, mask)
    torch.testing.assert_close(got, want)


def test_checkpoint_form():
    grid = e4m3_grid()
    assert grid.numel() == 127 and grid[-1] == 448 and grid[1] == 2.0 ** -9
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(codes, grid)
    x = torch.tensor([[448.0, 1.0, -1.0625, 0.0, 17.0] + [0.0] * 27, [449.0, 3.0] + [0.0] * 30])
    q, s = checkpoint_ref(x)
    assert s.tolist() == [[127], [128]]
    assert q[0, :5].tolist() == [448.0, 1.0, -1.0, 0.0, 16.0]  # ties to the even code
    assert q[1, :2].tolist() == [448.0, 3.0]  # 449 is 224.5 scaled: 224


@pytest.mark.parametrize("kw", [dict(M=1 << 29), dict(K=1000001, ldx=1 << 24), dict(N=1000001, ldb=1 << 24)])
def test_lora_refuses_what_no_grid_holds(kw):
    assert _lora(**kw) == INVALID and "bad sizes" in _lib.last_error()
    grad = {{"ldb": "ldg"}.get(k, k): v for k, v in kw.items()}
    assert _lora_grad(**grad) == INVALID and "bad sizes" in _lib.last_error()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_oracle_takes_8_bits_as_restored(dt):
    """A largest value whose 8-bit neighbour passes the type's range: finite gradients."""
    from oracle import tuning_ref as o

    x = torch.ones(2, 40, dtype=dt)
    x[0, 5] = torch.finfo(dt).max
    held = o.act_checkpoint_ref(x)
    rest = (torch.ones(1, 3, 40, dtype=dt), torch.ones(1, 8, 3, dtype=dt), torch.zeros(2, dtype=torch.int32),
            torch.ones(2, 3))
    dy = torch.full((2, 8), 2.0 ** -9, dtype=dt)
    got = o.lora_projection_backward_ref(dy, held, *rest)
    want = o.lora_projection_backward_ref(dy, o.act_restore_ref(held, dt), *rest)
    assert all(torch.isfinite(t).all() for t in got) and all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("op", OPS)
def test_oracle_leaves_its_inputs_alone(op):
    """fp32 inputs, which a cast to fp32 does not copy, and every other point of the sweep."""
    points = load_shape_sweep(all_specs()[op].shape_sweep)
    for p in points + [{**q, "dtype": "fp32"} for q in points]:
        f = input_gen.generate_inputs(op, p, 3, "cpu")
        flat = [t for v in f.values() for t in (v if isinstance(v, tuple) else (v,)) if torch.is_tensor(t)]
        before = [t.clone() for t in flat]
        out = reference_callable(op)(**f)
        assert all(torch.equal(t.view(torch.uint8) if t.dim() else t, b.view(torch.uint8) if b.dim() else b)
                   for t, b in zip(flat, before)), p
        outs = [out] if torch.is_tensor(out) else list(out)
        assert not {t.data_ptr() for t in outs if t.numel()} & {t.data_ptr() for t in flat if t.numel()}, p


def test_no_gradient_is_said_once(monkeypatch):
    """One warning an op."""
    import warnings

    from xkernels_amd.moe import hip_tuning as h

    monkeypatch.setattr(h, "_told", set())
    for op in ("one", "other"):
        with pytest.warns(RuntimeWarning, match=f"{op} records no autograd graph"):
            h._no_graph(op)
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            h._no_graph(op)
