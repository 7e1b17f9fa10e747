"""lora_projection and its backward on the GPU against 64-bit forms.

Bounds come from the arithmetic (_tuning_ref). Shapes: one token to several
sorted tiles, either side of the size up to which workgroups find their rows
themselves (256), odd and unaligned widths, ranks that fill no operand, one
adapter to many, adapters and whole batches without rows, rows without an adapter.
"""
from __future__ import annotations

import pytest
import torch

import xkernels_amd as xk
from xkernels_amd import _lib
from tests._tuning_ref import check, checkpoint_ref, lora_grad_ref, lora_ref

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _case(M, K, N, L, r, dt, seed=0, bare=0.2, runs=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).to(dt)
    a = (torch.randn(L, r, K, generator=g) / K ** 0.5).to(dt)
    b = (torch.randn(L, N, r, generator=g) / r ** 0.5).to(dt)
    ids = torch.randint(0, L, (M,), generator=g, dtype=torch.int32)
    if runs:
        ids = ids.sort().values
    ids[torch.rand(M, generator=g) < bare] = -1
    base = torch.randn(M, N, generator=g).to(dt)
    dy = torch.randn(M, N, generator=g).to(dt)
    sc = torch.rand(L, generator=g) + 0.5
    return [t.cuda() for t in (x, a, b, ids, base, dy, sc)]


SHAPES = [  # M, K, N, L, r
    (1, 64, 32, 1, 16), (1, 7168, 512, 8, 16), (2, 40, 24, 3, 8), (17, 256, 96, 2, 4), (64, 1000, 328, 32, 16),
    (100, 33, 47, 5, 3), (255, 512, 256, 4, 32), (256, 96, 160, 300, 8), (257, 512, 264, 4, 12),
    (300, 2880, 384, 2, 8), (513, 127, 65, 7, 5), (700, 640, 1032, 3, 64), (1025, 320, 136, 1, 128),
    (2000, 130, 258, 40, 100), (4100, 64, 64, 2, 16),
]


@pytest.mark.parametrize("M,K,N,L,r", SHAPES)
@pytest.mark.parametrize("dt", [BF, F32])
def test_forward(M, K, N, L, r, dt, dev):
    x, a, b, ids, base, _, sc = _case(M, K, N, L, r, dt, seed=M + K)
    out, hidden = xk.lora_projection(x, a, b, ids, base=base, scaling=sc, return_hidden=True)
    want, h, bound, hb = lora_ref(x, a, b, ids, base, sc)
    assert out.dtype == dt and hidden.dtype == F32
    check(out, want, bound, "out")
    check(hidden, h, hb, "hidden")
    bare = (ids < 0).nonzero().flatten()
    assert torch.equal(out[bare], base[bare]) and not hidden[bare].any()
    # the same bits without the hidden output and on a second call
    assert torch.equal(xk.lora_projection(x, a, b, ids, base=base, scaling=sc), out)


@pytest.mark.parametrize("M,K,N,L,r", SHAPES)
@pytest.mark.parametrize("dt", [BF, F32])
def test_backward(M, K, N, L, r, dt, dev):
    x, a, b, ids, _, dy, sc = _case(M, K, N, L, r, dt, seed=M + N, runs=M % 2 == 0)
    _, hidden = xk.lora_projection(x, a, b, ids, scaling=sc, return_hidden=True)
    got = xk.lora_projection_backward(dy, x, a, b, ids, hidden, scaling=sc)
    want, bounds = lora_grad_ref(dy, x, a, b, ids, hidden, sc)
    for name, g, w, bd in zip(("grad_x", "grad_a", "grad_b"), got, want, bounds):
        assert g.dtype == dt
        check(g, w, bd, name)
    again = xk.lora_projection_backward(dy, x, a, b, ids, hidden, scaling=sc)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("M,L,runs", [(70001, 1000, False), (70001, 1, False), (65536, 7, True), (66000, 1024, True),
                                     (1500, 1024, False)])
def test_many_rows(M, L, runs, dev):
    """The sort's sizes: batches that are counted apart, and the most adapters."""
    x, a, b, ids, base, dy, sc = _case(M, 32, 16, L, 4, BF, seed=L, runs=runs)
    out, hidden = xk.lora_projection(x, a, b, ids, base=base, scaling=sc, return_hidden=True)
    want, h, bound, hb = lora_ref(x, a, b, ids, base, sc)
    check(out, want, bound, "out")
    check(hidden, h, hb, "hidden")
    got = xk.lora_projection_backward(dy, x, a, b, ids, hidden, scaling=sc)
    want, bounds = lora_grad_ref(dy, x, a, b, ids, hidden, sc)
    for name, g, w, bd in zip(("grad_x", "grad_a", "grad_b"), got, want, bounds):
        check(g, w, bd, name)


@pytest.mark.parametrize("M,K,N,L,r", [(1, 64, 32, 1, 16), (70, 100, 40, 3, 8), (600, 2880, 200, 2, 16), (333, 47, 9, 4, 6),
                                       (1500, 256, 128, 1, 32)])
@pytest.mark.parametrize("dt", [BF, F32])
def test_backward_from_8_bits(M, K, N, L, r, dt, dev):
    x, a, b, ids, _, dy, sc = _case(M, K, N, L, r, dt, seed=M * 3)
    _, hidden = xk.lora_projection(x, a, b, ids, scaling=sc, return_hidden=True)
    held = xk.act_checkpoint(x)
    got = xk.lora_projection_backward(dy, held, a, b, ids, hidden, scaling=sc)
    want, bounds = lora_grad_ref(dy, checkpoint_ref(x)[0], a, b, ids, hidden, sc)
    for name, g, w, bd in zip(("grad_x", "grad_a", "grad_b"), got, want, bounds):
        check(g, w, bd, name)
    # the restored activations give the same bits
    again = xk.lora_projection_backward(dy, xk.act_restore(held, dt), a, b, ids, hidden, scaling=sc)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("M", [1, 40, 400])
def test_plain_call_without_base_and_scaling(M, dev):
    x, a, b, ids, *_ = _case(M, 96, 80, 3, 16, BF, seed=M)
    out = xk.lora_projection(x, a, b, ids)
    want, _, bound, _ = lora_ref(x, a, b, ids)
    check(out, want, bound)
    assert not out[ids < 0].any()


@pytest.mark.parametrize("M", [5, 200, 300, 1000])
@pytest.mark.parametrize("which", ["none", "one", "out of range", "int64"])
def test_ids(M, which, dev):
    """Every row bare; all rows on the last of many adapters; ids past the last, or whose
    lower 32 bits are a valid one, have no adapter."""
    L = 9
    x, a, b, _, base, dy, sc = _case(M, 72, 56, L, 8, BF, seed=M)
    if which == "none":
        ids = torch.full((M,), -1, dtype=torch.int32)
    elif which == "one":
        ids = torch.full((M,), L - 1, dtype=torch.int32)
    elif which == "out of range":
        ids = torch.tensor([L, -7, 2 ** 31 - 1, -2 ** 31, 3], dtype=torch.int32).repeat(M)[:M]
    else:
        ids = torch.tensor([2 ** 32 + 1, 4, -2 ** 33, L], dtype=torch.int64).repeat(M)[:M]
    plain = torch.where((ids >= 0) & (ids < L), ids, -1).int()
    ids = ids.cuda()
    out, hidden = xk.lora_projection(x, a, b, ids, base=base, scaling=sc, return_hidden=True)
    want, h, bound, hb = lora_ref(x, a, b, plain, base, sc)
    check(out, want, bound, "out")
    check(hidden, h, hb, "hidden")
    got = xk.lora_projection_backward(dy, x, a, b, ids, hidden, scaling=sc)
    want, bounds = lora_grad_ref(dy, x, a, b, plain, hidden, sc)
    for g, w, bd in zip(got, want, bounds):
        check(g, w, bd)
    used = plain[plain >= 0].unique()
    rest = [i for i in range(L) if i not in used.tolist()]
    assert not got[1][rest].any() and not got[2][rest].any()


@pytest.mark.parametrize("M", [30, 400])
@pytest.mark.parametrize("dt", [BF, F32])
def test_rows_apart(M, dt, dev):
    """Column slices of wider tensors, at aligned and at odd offsets, and a transposed x."""
    x, a, b, ids, base, dy, sc = _case(M, 128, 96, 3, 16, dt, seed=M)
    want, h, bound, _ = lora_ref(x, a, b, ids, base, sc)
    gw, gb = None, None
    for off in (8, 3):
        wide = torch.full((M, 300), float("nan"), dtype=dt, device="cuda")
        wide[:, off:off + 128] = x
        wb = torch.full((M, 200), float("nan"), dtype=dt, device="cuda")
        wb[:, off:off + 96] = base
        out, hidden = xk.lora_projection(wide[:, off:off + 128], a, b, ids, base=wb[:, off:off + 96], scaling=sc,
                                         return_hidden=True)
        check(out, want, bound, f"offset {off}")
        wb[:, off:off + 96] = dy
        got = xk.lora_projection_backward(wb[:, off:off + 96], wide[:, off:off + 128], a, b, ids, hidden, scaling=sc)
        if gw is None:
            gw, gb = lora_grad_ref(dy, x, a, b, ids, hidden, sc)
        for g, w, bd in zip(got, gw, gb):
            check(g, w, bd + 1e-6 * w.abs())  # (hidden of this call, not of the first)
    out = xk.lora_projection(x.t().contiguous().t(), a, b, ids, base=base, scaling=sc)
    check(out, want, bound, "transposed")
    one = xk.lora_projection(x[:1].expand(M, 128), a, b, ids, base=base, scaling=sc)
    w1, _, b1, _ = lora_ref(x[:1].expand(M, 128), a, b, ids, base, sc)
    check(one, w1, b1, "one row for all")


def test_rows_do_not_mix(dev):
    """A row of NaN or infinities stays its own, among rows of its adapter and others."""
    for M in (60, 500):
        x, a, b, ids, base, dy, sc = _case(M, 128, 64, 2, 20, BF, seed=M, bare=0.0)
        out = xk.lora_projection(x, a, b, ids, base=base, scaling=sc)
        x2, base2 = x.clone(), base.clone()
        x2[7], base2[9], x2[11, 5] = float("nan"), float("nan"), float("inf")
        out2 = xk.lora_projection(x2, a, b, ids, base=base2, scaling=sc)
        assert out2[7].isnan().all() and out2[9].isnan().all()
        assert not torch.isfinite(out2[11]).any()
        rest = [i for i in range(M) if i not in (7, 9, 11)]
        assert torch.equal(out2[rest], out[rest])
        ids[7] = -1  # a bare row's x is not read
        out3 = xk.lora_projection(x2, a, b, ids, base=base, scaling=sc)
        assert torch.equal(out3[7], base[7])


def test_infinite_hidden_stays_infinite(dev):
    """An h past bf16's or fp32's range keeps its sign through the pair."""
    a = torch.zeros(1, 4, 8, dtype=BF, device="cuda")
    a[0, 0, 0] = 1
    b = torch.zeros(1, 8, 4, dtype=BF, device="cuda")
    b[0, :, 0] = 1
    b[0, 3, 0] = -1
    x = torch.zeros(2, 8, dtype=BF, device="cuda")
    x[0, 0] = float("inf")
    x[1, 0] = 3.3e38
    out = xk.lora_projection(x, a, b, torch.zeros(2, dtype=torch.int32, device="cuda"),
                             scaling=torch.tensor([1.0], device="cuda"))
    # inf * 0 in the other ranks of a hidden row is NaN by the formula too: h has one rank in use
    assert torch.isnan(out[0]).all() or torch.isinf(out[0]).all()
    assert torch.isfinite(out[1]).all() and out[1, 3] == -out[1, 0]


@pytest.mark.parametrize("dt", [BF, F32])
def test_empty(dt, dev):
    x, a, b, ids, base, dy, sc = _case(4, 64, 32, 3, 8, dt)
    out, hidden = xk.lora_projection(x[:0], a, b, ids[:0], base=base[:0], scaling=sc, return_hidden=True)
    assert out.shape == (0, 32) and hidden.shape == (0, 8)
    gx, ga, gb = xk.lora_projection_backward(dy[:0], x[:0], a, b, ids[:0], hidden, scaling=sc)
    assert gx.shape == (0, 64) and not ga.any() and not gb.any() and ga.shape == a.shape and gb.shape == b.shape


def test_gradient_against_differences(dev):
    """Directional differences of the fp32 forward: f is bilinear in (A, B) and linear in x,
    so a central difference along one of them is exact but for rounding."""
    x, a, b, ids, _, dy, sc = _case(40, 48, 40, 3, 8, F32, seed=5)
    f = lambda x, a, b: float((xk.lora_projection(x, a, b, ids, scaling=sc).double() * dy.double()).sum())  # noqa: E731
    _, hidden = xk.lora_projection(x, a, b, ids, scaling=sc, return_hidden=True)
    grads = xk.lora_projection_backward(dy, x, a, b, ids, hidden, scaling=sc)
    g = torch.Generator(device="cuda").manual_seed(1)
    for i, t in enumerate((x, a, b)):
        d = torch.randn(t.shape, generator=g, device="cuda")
        args_p, args_m = [x, a, b], [x, a, b]
        args_p[i], args_m[i] = t + d, t - d
        diff = (f(*args_p) - f(*args_m)) / 2
        want = float((grads[i].double() * d.double()).sum())
        # each f is a sum of 40 * 40 terms off by 2^-20 of its size or less
        size = float(xk.lora_projection(*[v.abs() for v in args_p], ids, scaling=sc).double().abs().sum()) * float(dy.abs().max())
        assert abs(diff - want) <= 2.0 ** -19 * size, (i, diff, want, size)


@pytest.mark.parametrize("M", [8, 600])
def test_captured(M, dev):
    """A serving step (projection + adapters) and a tuning step replay with new inputs; eager
    work and synchronisations between the replays."""
    x, a, b, ids, base, dy, sc = _case(M, 256, 128, 4, 16, BF, seed=M)
    out, hidden = xk.lora_projection(x, a, b, ids, base=base, scaling=sc, return_hidden=True)
    xk.lora_projection_backward(dy, x, a, b, ids, hidden, scaling=sc)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, hidden = xk.lora_projection(x, a, b, ids, base=base, scaling=sc, return_hidden=True)
        held = xk.act_checkpoint(x)
        grads = xk.lora_projection_backward(dy, held, a, b, ids, hidden, scaling=sc)
    for seed in range(4):
        fresh = _case(M, 256, 128, 4, 16, BF, seed=100 + seed)
        for t, f in zip((x, a, b, ids, base, dy, sc), fresh):
            t.copy_(f)
        graph.replay()
        got = [t.clone() for t in (out, hidden, *grads)]
        torch.cuda.synchronize()
        o, h = xk.lora_projection(x, a, b, ids, base=base, scaling=sc, return_hidden=True)
        g = xk.lora_projection_backward(dy, xk.act_checkpoint(x), a, b, ids, h, scaling=sc)
        assert all(torch.equal(p, q) for p, q in zip(got, (o, h, *g))), seed


def test_streams(dev):
    """Two streams at once, each with its own scratch."""
    cases = [_case(300, 512, 256, 4, 16, BF, seed=s) for s in (1, 2)]
    want = [xk.lora_projection(c[0], c[1], c[2], c[3], base=c[4], scaling=c[6]) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                got.append(xk.lora_projection(c[0], c[1], c[2], c[3], base=c[4], scaling=c[6]))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("M", [3, 250, 700])
@pytest.mark.parametrize("N", [64, 47])
@pytest.mark.parametrize("dt", [BF, F32])
def test_out_over_base(M, N, dt, dev):
    """The C entry point may write the result over the base."""
    x, a, b, ids, base, _, sc = _case(M, 96, N, 3, 12, dt, seed=M)
    want = xk.lora_projection(x, a, b, ids, base=base, scaling=sc)
    need = _lib.query("xk_lora_projection_workspace_bytes", M, 96, 3, 12)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    _lib.call("xk_lora_projection", x.data_ptr(), _lib.XK_DT_BF16 if dt == BF else _lib.XK_DT_FP32, 96, M, 96,
              a.data_ptr(), b.data_ptr(), 3, N, 12, ids.data_ptr(), sc.data_ptr(), base.data_ptr(), N, base.data_ptr(),
              None, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(base, want)


@pytest.mark.parametrize("M", [20, 500])
@pytest.mark.parametrize("dt", [BF, F32])
def test_weights_at_odd_offsets(M, dt, dev):
    """Adapters that begin between two 16-byte pieces, as slices of a bank do: the same values."""
    x, a, b, ids, base, dy, sc = _case(M, 128, 64, 4, 16, dt, seed=M)
    want = xk.lora_projection(x, a, b, ids, base=base, scaling=sc, return_hidden=True)
    grads = xk.lora_projection_backward(dy, x, a, b, ids, want[1], scaling=sc)
    bank = torch.full((a.numel() + b.numel() + 8,), float("nan"), dtype=dt, device="cuda")
    a2 = bank[1:1 + a.numel()].view(a.shape)
    b2 = bank[3 + a.numel():3 + a.numel() + b.numel()].view(b.shape)
    a2.copy_(a)
    b2.copy_(b)
    got = xk.lora_projection(x, a2, b2, ids, base=base, scaling=sc, return_hidden=True)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    got = xk.lora_projection_backward(dy, x, a2, b2, ids, want[1], scaling=sc)
    assert all(torch.equal(p, q) for p, q in zip(got, grads))


@pytest.mark.parametrize("M", [200, 600])
def test_bare_rows_hold_anything(M, dev):
    """NaN in the x, grad_out and hidden of rows without an adapter reaches nothing."""
    x, a, b, ids, base, dy, sc = _case(M, 64, 48, 3, 8, BF, seed=M, bare=0.4)
    bare = ids < 0
    _, hidden = xk.lora_projection(x, a, b, ids, base=base, scaling=sc, return_hidden=True)
    want = xk.lora_projection_backward(dy, x, a, b, ids, hidden, scaling=sc)
    for t in (x, dy, hidden):
        t[bare] = float("nan")
    got = xk.lora_projection_backward(dy, x, a, b, ids, hidden, scaling=sc)
    assert all(torch.equal(p, q) for p, q in zip(got, want)) and not got[0][bare].any()


@pytest.mark.parametrize("dt", [torch.int16, torch.int8, torch.uint8])
def test_narrow_ids(dt, dev):
    x, a, b, ids, base, _, sc = _case(90, 64, 48, 3, 8, BF, bare=0.0)
    ids[5] = 100
    want = xk.lora_projection(x, a, b, ids, base=base, scaling=sc)
    assert torch.equal(xk.lora_projection(x, a, b, ids.to(dt), base=base, scaling=sc), want)
    assert torch.equal(want[5], base[5])


def test_more_than_32_bits_of_values(dev):
    """x, base, out, grad_out and grad_x past 2^31 values: the last rows, whose adapter's
    gradients come from them alone."""
    M, W, r = 66000, 33000, 4
    x = torch.zeros(M, W, dtype=BF, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    x[-3:] = torch.randn(3, W, generator=g, device="cuda").to(BF)
    a = (torch.randn(2, r, W, generator=g, device="cuda") / W ** 0.5).to(BF)
    b = torch.randn(2, W, r, generator=g, device="cuda").to(BF)
    ids = torch.zeros(M, dtype=torch.int32, device="cuda")
    ids[-3:] = 1
    out, hidden = xk.lora_projection(x, a, b, ids, base=x, return_hidden=True)
    last = slice(M - 3, M)
    want, h, bound, hb = lora_ref(x[last], a, b, ids[last], x[last], None)
    check(out[last], want, bound, "out")
    check(hidden[last], h, hb, "hidden")
    assert not out[:-3].any() and not hidden[:-3].any()
    got = xk.lora_projection_backward(out, x, a, b, ids, hidden)
    want, bounds = lora_grad_ref(out[last], x[last], a, b, ids[last], hidden[last], None)
    check(got[0][last], want[0], bounds[0], "grad_x")
    assert not got[0][:-3].any()
    for i in (1, 2):
        check(got[i][1], want[i][1], bounds[i][1], "weights")
        assert not got[i][0].any()


def test_refusals(dev):
    """Shapes and types that do not fit, before any launch."""
    x, a, b, ids, base, dy, sc = _case(6, 64, 32, 3, 8, BF)
    _, h = xk.lora_projection(x, a, b, ids, return_hidden=True)
    bad = [lambda: xk.lora_projection(x[:, :60], a, b, ids), lambda: xk.lora_projection(x, a, b[:2], ids),
           lambda: xk.lora_projection(x, a, b, ids[:5]), lambda: xk.lora_projection(x.float(), a, b, ids),
           lambda: xk.lora_projection(x, a, b, ids, base=base.float()), lambda: xk.lora_projection(x, a, b, ids.float()),
           lambda: xk.lora_projection(x, a, b, ids, base=base[:, :30]), lambda: xk.lora_projection(x[0], a, b, ids),
           lambda: xk.lora_projection(x, a, b, ids, scaling=sc[:2]), lambda: xk.lora_projection(x, a[0], b, ids),
           lambda: xk.lora_projection(x.half(), a.half(), b.half(), ids), lambda: xk.lora_projection(x, a, b.float(), ids),
           lambda: xk.lora_projection(x, a.cpu(), b, ids),
           lambda: xk.lora_projection_backward(dy[:, :30], x, a, b, ids, h),
           lambda: xk.lora_projection_backward(dy, x[:5], a, b, ids, h),
           lambda: xk.lora_projection_backward(dy, x, a, b, ids, h[:, :7]),
           lambda: xk.lora_projection_backward(dy, x.float(), a, b, ids, h),
           lambda: xk.lora_projection_backward(dy, xk.act_checkpoint(x)._replace(scales=ids[:, None]), a, b, ids, h),
           lambda: xk.lora_projection_backward(dy, (x, xk.act_checkpoint(x).scales), a, b, ids, h)]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} went through")


@pytest.mark.parametrize("r,dt", [(8, F32), (16, BF), (64, BF), (128, BF), (128, F32)])
@pytest.mark.parametrize("K,N", [(520, 264), (2050, 77)])
def test_short_adapters(r, dt, K, N, dev):
    """Adapters of one row to a few tiles, in windows of their own and shared ones."""
    sizes = [1, 64, 65, 0, 3, 200, 31, 0, 129]
    ids = torch.tensor([i for i, n in enumerate(sizes) for _ in range(n)], dtype=torch.int32)
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(r))].cuda()
    x, a, b, _, _, dy, sc = _case(len(ids), K, N, len(sizes), r, dt, seed=r)
    _, hidden = xk.lora_projection(x, a, b, ids, scaling=sc, return_hidden=True)
    got = xk.lora_projection_backward(dy, x, a, b, ids, hidden, scaling=sc)
    want, bounds = lora_grad_ref(dy, x, a, b, ids, hidden, sc)
    for name, g, w, bd in zip(("grad_x", "grad_a", "grad_b"), got, want, bounds):
        check(g, w, bd, name)
    for i in (3, 7):
        assert not got[1][i].any() and not got[2][i].any()


def test_gradients_on_streams(dev):
    """Two backward passes at once."""
    cases = [_case(500, 512, 264, 4, 16, BF, seed=s) for s in (1, 2)]
    hs = [xk.lora_projection(c[0], c[1], c[2], c[3], return_hidden=True)[1] for c in cases]
    run = lambda c, h: xk.lora_projection_backward(c[5], c[0], c[1], c[2], c[3], h, scaling=c[6])  # noqa: E731
    want = [run(c, h) for c, h in zip(cases, hs)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, h, st in zip(cases, hs, streams):
            with torch.cuda.stream(st):
                got.append(run(c, h))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for g, w in zip(got, want) for p, q in zip(g, w))


@pytest.mark.parametrize("K", [96, 70])
@pytest.mark.parametrize("dt", [BF, F32])
def test_backward_from_8_bits_at_the_top(K, dt, dev):
    """Activations whose 8-bit neighbour passes the type's range enter the gradients as they are
    restored, the largest finite value: the same bits, and finite ones."""
    x, a, b, _, _, dy, _ = _case(3, K, 16, 1, 4, dt, seed=K)
    x[0, 3], x[1, 40], x[2, K - 1] = torch.finfo(dt).max, torch.finfo(dt).min, torch.finfo(dt).max
    dy *= 2.0 ** -9
    ids = torch.zeros(3, dtype=torch.int32, device="cuda")
    hidden = torch.randn(3, 4, device="cuda")
    held = xk.act_checkpoint(x)
    back = xk.act_restore(held, dt)
    assert torch.isfinite(back).all() and back[0, 3] == torch.finfo(dt).max
    got = xk.lora_projection_backward(dy, held, a, b, ids, hidden)
    want = xk.lora_projection_backward(dy, back, a, b, ids, hidden)
    assert all(torch.isfinite(t).all() for t in got)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    ref, bounds = lora_grad_ref(dy, back, a, b, ids, hidden)
    for name, g, w, bd in zip(("grad_x", "grad_a", "grad_b"), got, ref, bounds):
        check(g, w, bd, name)


@pytest.mark.parametrize("K", [8192, 8191])
@pytest.mark.parametrize("dt", [BF, F32])
def test_backward_from_every_byte(K, dt, dev):
    """Every e4m3 code at every scale byte, reserved ones among them, in a gradient of one row
    and one rank (x itself times a power of two): as act_restore gives them."""
    a, b = torch.ones(1, 1, K, dtype=dt, device="cuda"), torch.ones(1, 8, 1, dtype=dt, device="cuda")
    ids, hidden = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.ones(1, 1, device="cuda")
    scales = torch.arange(256, dtype=torch.uint8).view(1, 256).cuda()
    dy = torch.zeros(1, 8, dtype=dt, device="cuda")
    for power in (0, 40, -40):
        dy[0, 3] = 2.0 ** power
        for first in range(0, 256, 32):
            codes = (torch.arange(32) + first).to(torch.uint8).repeat(256)[:K].view(1, K)
            held = xk.ActCheckpoint(codes.cuda().view(torch.float8_e4m3fn), scales)
            got = xk.lora_projection_backward(dy, held, a, b, ids, hidden)[1]
            want = xk.lora_projection_backward(dy, xk.act_restore(held, dt), a, b, ids, hidden)[1]
            assert torch.equal(got.isnan(), want.isnan()), (power, first)
            bad = ((got != want) & ~want.isnan()).flatten().nonzero().flatten()
            assert bad.numel() == 0, (power, first, bad.numel(), bad[:4].tolist(), got.flatten()[bad[:4]], want.flatten()[bad[:4]])


@pytest.mark.parametrize("M", [2, 300])
@pytest.mark.parametrize("r", [1, 20, 40, 100])
@pytest.mark.parametrize("dt", [BF, F32])
def test_infinite_hidden_keeps_its_sign(M, r, dt, dev):
    """Infinities of either sign in one column of x, weights that are nowhere 0 or infinite
    where they meet them: infinities of the formula's signs, no NaN."""
    K, N = 72, 40
    a = torch.zeros(1, r, K, dtype=dt, device="cuda")
    a[:, :, 0] = 1
    b = torch.ones(1, N, r, dtype=dt, device="cuda")
    b[:, 1::2] = -1
    x = torch.ones(M, K, dtype=dt, device="cuda")
    x[0, 0], x[1, 0] = float("inf"), float("-inf")
    ids = torch.zeros(M, dtype=torch.int32, device="cuda")
    out, hidden = xk.lora_projection(x, a, b, ids, return_hidden=True)
    sign = b[0, :, 0]
    assert torch.equal(hidden[0], torch.full_like(hidden[0], float("inf"))) and torch.equal(hidden[1], -hidden[0])
    assert torch.equal(out[0], sign * float("inf")) and torch.equal(out[1], -sign * float("inf"))
    assert torch.equal(out[2:], (r * sign).expand(M - 2, N))


@pytest.mark.parametrize("M", [3, 300])
@pytest.mark.parametrize("r", [1, 20, 40, 100])
def test_hidden_past_bf16s_range(M, r, dev):
    """An h and a g between bf16's largest value and fp32's, times 2^-2: finite, as in 32 bits."""
    K, N, top = 64, 48, 2.0 ** 127
    big = torch.tensor([1.5 * top, 0.498046875 * top]).to(BF)  # both exact; their sum rounds to 2^128 in bf16
    assert torch.isfinite(big.float().sum()) and torch.isinf(big.float().sum().to(BF))
    a, b = torch.zeros(1, r, K, dtype=BF), torch.zeros(1, N, r, dtype=BF)
    a[0, 0, :2], b[0, :, 0] = 1, 0.25
    a[0, 0, 2:] = 0.25
    x = torch.zeros(M, K, dtype=BF)
    x[0, :2], x[1, :2] = big, -big
    ids = torch.zeros(M, dtype=torch.int32)
    x, a, b, ids = (t.cuda() for t in (x, a, b, ids))
    out, hidden = xk.lora_projection(x, a, b, ids, return_hidden=True)
    want, h, bound, hb = lora_ref(x, a, b, ids)
    check(hidden, h, hb, "hidden")
    check(out, want, bound, "out")
    b[0, :2, 0] = 1  # g = big[0] + big[1]
    dy = torch.zeros(M, N, dtype=BF, device="cuda")
    dy[0, :2], dy[2 % M, 2:] = big.cuda(), 0.5
    hidden[0] = 0  # (as x: a product with grad_out that stays finite)
    x[:2] = 0.25
    hidden[1, 0] = float(big.float().sum())  # times grad_out of 0.25
    dy[1, 4] = 0.25
    a[0, 0] = 0.25
    got = xk.lora_projection_backward(dy, x, a, b, ids, hidden)
    want, bounds = lora_grad_ref(dy, x, a, b, ids, hidden)
    for name, g, w, bd in zip(("grad_x", "grad_a", "grad_b"), got, want, bounds):
        check(g, w, bd, name)


@pytest.mark.parametrize("M", [200, 300, 5000])
@pytest.mark.parametrize("N", [64, 47])
@pytest.mark.parametrize("r", [16, 128])
def test_small_products_beside_a_large_base(M, N, r, dev):
    """fp32 products each below half a step of the base: their sum, which is not, counts."""
    ids = torch.zeros(M, dtype=torch.int32, device="cuda")
    x = torch.ones(M, 8, device="cuda")
    a = torch.full((1, r, 8), 2.0 ** -3, device="cuda")
    b = torch.full((1, N, r), 0.9 * 2.0 ** -25, device="cuda")
    base = torch.ones(M, N, device="cuda")
    out = xk.lora_projection(x, a, b, ids, base=base)
    want, _, bound, _ = lora_ref(x, a, b, ids, base)
    check(out, want, bound)
