"""moe_balance_loss and moe_router_backward on the GPU against 64-bit forms, with
bounds from the arithmetic (_tuning_ref): one row to many planes, expert counts
of every kernel (128, 256, 512 a row of lanes, and past it), masks that leave
some or no rows, ids out of range, repeated ids, infinite and NaN logits."""
from __future__ import annotations

import pytest
import torch

import xkernels_amd as xk
from tests._tuning_ref import F32, balance_ref, check, router_grad_ref, softmax_delta

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SHAPES = [(1, 8, 2), (3, 4, 4), (200, 48, 8), (256, 100, 6), (257, 256, 8), (1000, 384, 8), (5000, 64, 1),
          (300, 511, 16), (70, 512, 16), (40, 513, 8), (300, 1000, 20), (5, 3000, 2), (64, 1, 1), (33, 40, 24)]


def _case(M, E, k, dt, seed=0, pad=0.0):
    g = torch.Generator().manual_seed(seed)
    z = (1.5 * torch.randn(M, E, generator=g) + torch.randn(E, generator=g)).to(dt)
    ids = torch.topk(z.float(), k, dim=1).indices.int()
    u = torch.randn(M, k, generator=g)
    mask = torch.rand(M, generator=g) >= pad if pad else None
    return z.cuda(), ids.cuda(), u.cuda(), None if mask is None else mask.cuda()


def _check_loss(z, ids, mask):
    got = xk.moe_balance_loss(z, ids, mask=mask)
    loss, counts, tokens = balance_ref(z, ids, mask)
    assert got.loss.dtype == torch.float32 and got.counts.dtype == got.tokens.dtype == torch.int32
    assert torch.equal(got.counts.cpu().long(), counts) and int(got.tokens) == tokens
    rel = softmax_delta(z.double().cpu()) + (z.shape[0] + 64) * F32 / 2
    check(got.loss, loss, rel * loss, "loss")
    return got


@pytest.mark.parametrize("M,E,k", SHAPES)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("pad", [0.0, 0.4])
def test_loss_and_counts(M, E, k, dt, pad, dev):
    z, ids, _, mask = _case(M, E, k, dt, seed=M + E, pad=pad)
    got = _check_loss(z, ids, mask)
    again = xk.moe_balance_loss(z, ids, mask=mask)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("M,E,k", SHAPES)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("renorm,parts", [(True, "both"), (False, "both"), (True, "weights"), (False, "weights"),
                                          (True, "loss")])
def test_gradient(M, E, k, dt, renorm, parts, dev):
    z, ids, u, mask = _case(M, E, k, dt, seed=M + k, pad=0.3 if M > 4 else 0.0)
    st = xk.moe_balance_loss(z, ids, mask=mask)
    gl = torch.tensor(0.7, device="cuda") if parts != "weights" else None
    gw = u if parts != "loss" else None
    got = xk.moe_router_backward(z, ids, grad_weights=gw, renormalize=renorm, grad_loss=gl,
                                 counts=st.counts if gl is not None else None,
                                 tokens=st.tokens if gl is not None else None, mask=mask)
    want, bound = router_grad_ref(z, ids, gw, renorm, gl, st.counts, mask)
    assert got.dtype == dt
    check(got, want, bound)
    if mask is not None:
        assert not got[~mask].any()


@pytest.mark.parametrize("E,k", [(64, 4), (600, 4), (64, 20)])
def test_ids_out_of_range_and_repeated(E, k, dev):
    z, ids, u, _ = _case(50, E, k, torch.float32, seed=E)
    ids[3] = -1
    ids[4, 0], ids[5, 1], ids[6, 2] = E, 2 ** 31 - 1, -2 ** 31
    ids[7, :3] = 5
    ids[8] = 1
    st = _check_loss(z, ids, None)
    for renorm in (True, False):
        got = xk.moe_router_backward(z, ids, grad_weights=u, renormalize=renorm, grad_loss=torch.ones((), device="cuda"),
                                     counts=st.counts)
        want, bound = router_grad_ref(z, ids, u, renorm, 1.0, st.counts)
        check(got, want, bound)
    wide = ids.long()
    wide[9, 0] = 2 ** 32 + 2
    narrow = ids.clone()
    narrow[9, 0] = -1
    a, b = xk.moe_balance_loss(z, wide), xk.moe_balance_loss(z, narrow)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("M,E", [(10, 64), (400, 64), (20, 700)])
def test_masked_rows_are_not_read(M, E, dev):
    """NaN and infinities in padded rows, and a mask that leaves nothing."""
    z, ids, u, _ = _case(M, E, 4, torch.bfloat16, seed=M)
    mask = torch.ones(M, dtype=torch.bool, device="cuda")
    mask[[1, 5, M - 1]] = False
    want = xk.moe_balance_loss(z, ids, mask=mask)
    grad = xk.moe_router_backward(z, ids, grad_weights=u, grad_loss=want.loss, counts=want.counts, tokens=want.tokens,
                                  mask=mask)
    z2, ids2, u2 = z.clone(), ids.clone(), u.clone()
    z2[1], z2[5, 0], z2[M - 1] = float("nan"), float("inf"), float("-inf")
    ids2[1], u2[5] = 3, float("nan")
    got = xk.moe_balance_loss(z2, ids2, mask=mask)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    grad2 = xk.moe_router_backward(z2, ids2, grad_weights=u2, grad_loss=want.loss, counts=want.counts,
                                   tokens=want.tokens, mask=mask)
    assert torch.equal(grad, grad2) and not grad2[~mask].any()
    none = torch.zeros(M, dtype=torch.bool, device="cuda")
    st = xk.moe_balance_loss(z2, ids2, mask=none)
    assert float(st.loss) == 0.0 and int(st.tokens) == 0 and not st.counts.any()
    g = xk.moe_router_backward(z2, ids2, grad_weights=u2, grad_loss=st.loss + 1, counts=st.counts, tokens=st.tokens,
                               mask=none)
    assert not g.any()


@pytest.mark.parametrize("M,E", [(12, 96), (300, 300), (12, 700)])
def test_special_logits(M, E, dev):
    """Experts masked with -inf or the type's lowest value have no probability and no
    gradient; a row with NaN or +inf is NaN in its own gradient and the loss only."""
    z, ids, u, _ = _case(M, E, 4, torch.float32, seed=E)
    z[2, 10:] = float("-inf")
    z[3, 4:] = torch.finfo(torch.float32).min
    ids[2], ids[3] = torch.arange(4, device="cuda"), torch.arange(4, device="cuda")
    st = _check_loss(z.clamp(min=-1e4), ids, None)  # the same probabilities: 0
    st2 = xk.moe_balance_loss(z, ids)
    torch.testing.assert_close(st2.loss, st.loss, rtol=1e-6, atol=0)
    for renorm in (True, False):
        kw = dict(grad_weights=u, renormalize=renorm, grad_loss=torch.ones((), device="cuda"), counts=st2.counts)
        got = xk.moe_router_backward(z, ids, **kw)
        assert torch.isfinite(got).all() and not got[2, 10:].any() and not got[3, 4:].any()
        bad = z.clone()
        bad[5, 1], bad[6, 0], bad[7] = float("nan"), float("inf"), float("-inf")
        g2 = xk.moe_router_backward(bad, ids, **kw)
        rows = [5, 6, 7]
        assert g2[rows].isnan().any(1).all()
        rest = [i for i in range(M) if i not in rows]
        assert torch.equal(g2[rest], got[rest])
    assert xk.moe_balance_loss(bad, ids).loss.isnan()


def test_empty_batch(dev):
    for E in (16, 700):
        z = torch.empty(0, E, device="cuda")
        ids = torch.empty(0, 2, dtype=torch.int32, device="cuda")
        st = xk.moe_balance_loss(z, ids)
        assert float(st.loss) == 0 and int(st.tokens) == 0 and not st.counts.any() and st.counts.numel() == E
        assert xk.moe_router_backward(z, ids, grad_weights=torch.empty(0, 2, device="cuda")).shape == (0, E)


def test_gradient_against_differences(dev):
    """Central differences of the weights' and the loss's 64-bit forms along a direction."""
    z, ids, u, _ = _case(30, 24, 4, torch.float32, seed=3)
    st = xk.moe_balance_loss(z, ids)
    got = xk.moe_router_backward(z, ids, grad_weights=u, renormalize=True, grad_loss=torch.ones((), device="cuda"),
                                 counts=st.counts).double().cpu()
    z64, i64, u64, c = z.double().cpu(), ids.long().cpu(), u.double().cpu(), st.counts.double().cpu()

    def f(z):
        p = torch.softmax(z, 1)
        w = p.gather(1, i64)
        return float((w / w.sum(1, keepdim=True) * u64).sum() + 24 / (30 * 30 * 4) * (c @ p.sum(0)))

    d = torch.randn(z.shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    h = 1e-5
    diff = (f(z64 + h * d) - f(z64 - h * d)) / (2 * h)
    # the difference's own error is about h^2 of third derivatives; the kernel's 2^-18 of the terms
    assert abs(diff - float((got * d).sum())) <= 1e-6 + 2.0 ** -18 * float((got * d).abs().sum())


def test_step_together_and_captured(dev):
    """Router, loss and both gradients as a training step runs them, eager and in a graph."""
    M, E, k = 300, 48, 4
    z = _case(M, E, k, torch.bfloat16, seed=1)[0]
    u = torch.randn(M, k, device="cuda")
    coef = torch.tensor(0.01, device="cuda")

    def step():
        w, ids = xk.topk_softmax(z, k)
        st = xk.moe_balance_loss(z, ids)
        return w, *st, xk.moe_router_backward(z, ids, grad_weights=u, grad_loss=coef, counts=st.counts)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        z.copy_(_case(M, E, k, torch.bfloat16, seed=10 + seed)[0])
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, step()))


def test_strided_and_unaligned(dev):
    z, ids, u, _ = _case(90, 64, 4, torch.bfloat16, seed=2)
    want = xk.moe_router_backward(z, ids, grad_weights=u)
    wide = torch.zeros(90, 131, dtype=z.dtype, device="cuda")
    wide[:, 3:67] = z
    assert torch.equal(xk.moe_router_backward(wide[:, 3:67], ids, grad_weights=u), want)
    flat = torch.zeros(90 * 64 + 1, dtype=z.dtype, device="cuda")
    off = flat[1:].view(90, 64)
    off.copy_(z)
    assert torch.equal(xk.moe_router_backward(off, ids, grad_weights=u), want)
    assert all(torch.equal(p, q) for p, q in zip(xk.moe_balance_loss(off, ids), xk.moe_balance_loss(z, ids)))


@pytest.mark.parametrize("M", [40, 700])
def test_mask_types(M, dev):
    """Masks of whole numbers, of floats and of strided booleans: nonzero counts."""
    z, ids, u, mask = _case(M, 96, 4, torch.bfloat16, seed=M, pad=0.4)
    want = xk.moe_balance_loss(z, ids, mask=mask)
    kw = dict(grad_weights=u, grad_loss=want.loss, counts=want.counts, tokens=want.tokens)
    grad = xk.moe_router_backward(z, ids, mask=mask, **kw)
    for other in (mask.to(torch.uint8) * 2, mask.long() << 40, mask.float() * 0.25, mask.repeat_interleave(2)[::2]):
        got = xk.moe_balance_loss(z, ids, mask=other)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        assert torch.equal(xk.moe_router_backward(z, ids, mask=other, **kw), grad)


@pytest.mark.parametrize("M,E", [(80, 64), (900, 256), (60, 700)])
def test_padded_batch_captured(M, E, dev):
    """One graph for batches of any fill: the mask and what it leaves change between replays."""
    z, ids, u, mask = _case(M, E, 4, torch.bfloat16, seed=1, pad=0.5)
    coef = torch.tensor(0.01, device="cuda")

    def step():
        st = xk.moe_balance_loss(z, ids, mask=mask)
        return *st, xk.moe_router_backward(z, ids, grad_weights=u, renormalize=False, grad_loss=coef, counts=st.counts,
                                           tokens=st.tokens, mask=mask)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed, fill in enumerate((1.0, 0.3, 0.0, 0.8)):
        fresh = _case(M, E, 4, torch.bfloat16, seed=20 + seed)
        z.copy_(fresh[0])
        ids.copy_(fresh[1])
        mask.copy_(torch.rand(M, generator=torch.Generator().manual_seed(seed)) < fill)
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, step())), seed
        assert int(got[2]) == int(mask.sum())


def test_more_than_32_bits_of_logits(dev):
    """Rows past 2^31 logits; all but the last three padded."""
    M, E, k = 4200000, 512, 2
    z = torch.zeros(M, E, dtype=torch.float16, device="cuda")
    few = _case(3, E, k, torch.float16, seed=9)
    z[-3:] = few[0]
    ids = torch.zeros(M, k, dtype=torch.int32, device="cuda")
    ids[-3:] = few[1]
    u = torch.ones(M, k, device="cuda")
    u[-3:] = few[2]
    mask = torch.zeros(M, dtype=torch.bool, device="cuda")
    mask[-3:] = True
    st = xk.moe_balance_loss(z, ids, mask=mask)
    loss, counts, tokens = balance_ref(few[0], few[1], None)
    assert torch.equal(st.counts.cpu().long(), counts) and int(st.tokens) == tokens == 3
    check(st.loss, loss, (softmax_delta(few[0].double().cpu()) + 67 * F32 / 2) * loss, "loss")
    gl = torch.tensor(0.7, device="cuda")
    got = xk.moe_router_backward(z, ids, grad_weights=u, grad_loss=gl, counts=st.counts, tokens=st.tokens, mask=mask)
    want, bound = router_grad_ref(few[0], few[1], few[2], True, gl, st.counts)
    check(got[-3:], want, bound)
    assert not got[:-3].any()


def test_refusals(dev):
    z, ids, u, mask = _case(6, 16, 2, torch.float32, pad=0.5)
    st = xk.moe_balance_loss(z, ids)
    bad = [lambda: xk.moe_balance_loss(z, ids[:5]), lambda: xk.moe_balance_loss(z, ids[:, :0]),
           lambda: xk.moe_balance_loss(z, ids.float()), lambda: xk.moe_balance_loss(z.double(), ids),
           lambda: xk.moe_balance_loss(z[0], ids), lambda: xk.moe_balance_loss(z, ids, mask=mask[:5]),
           lambda: xk.moe_balance_loss(z[:, :1], ids), lambda: xk.moe_balance_loss(z, ids.cpu()),
           lambda: xk.moe_router_backward(z, ids), lambda: xk.moe_router_backward(z, ids, grad_loss=st.loss),
           lambda: xk.moe_router_backward(z, ids, grad_loss=st.loss, counts=st.counts, mask=mask),
           lambda: xk.moe_router_backward(z, ids, grad_loss=st.loss, counts=st.counts[:5]),
           lambda: xk.moe_router_backward(z, ids, grad_loss=u, counts=st.counts),
           lambda: xk.moe_router_backward(z, ids, grad_weights=u[:, :1])]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} went through")


@pytest.mark.parametrize("E", [48, 600])
def test_counts_of_several_ranks(E, dev):
    """Parts of a batch, each with the summed counts and rows: together the whole batch's gradient."""
    z, ids, u, mask = _case(700, E, 4, torch.float32, seed=E, pad=0.2)
    whole = xk.moe_balance_loss(z, ids, mask=mask)
    gl = torch.tensor(0.3, device="cuda")
    want, bound = router_grad_ref(z, ids, u, True, gl, whole.counts, mask)
    parts = [slice(0, 100), slice(100, 420), slice(420, 700)]
    sts = [xk.moe_balance_loss(z[p], ids[p], mask=mask[p]) for p in parts]
    counts, tokens = sum(s.counts for s in sts), sum(s.tokens for s in sts)
    assert torch.equal(counts, whole.counts) and int(tokens) == int(whole.tokens)
    got = torch.cat([xk.moe_router_backward(z[p], ids[p], grad_weights=u[p], grad_loss=gl, counts=counts, tokens=tokens,
                                            mask=mask[p]) for p in parts])
    check(got, want, bound)


@pytest.mark.parametrize("M,E,k", [(300000, 600, 1), (1100000, 520, 2), (1 << 22, 48, 2), (1 << 26, 6, 1)])
def test_sums_over_many_rows(M, E, k, dev):
    """Equal logits: a probability of 1 / E is added M times, each time with the same rounding.
    The loss is 1 whatever the ids. A lane's 64 additions, 4 lanes', 8 waves', 8 planes' and 8
    parts' sums in 32 bits are off by half a step (2^-24) each at most, as are 1 / E, a plane, a
    part and the loss; what lies beyond is added in 64 bits. None of it grows with M."""
    off = (64 + 2 + 8 + 8 + 8 + 4) * 2.0 ** -24
    z = torch.zeros(M, E, dtype=torch.bfloat16, device="cuda")
    ids = (torch.arange(M * k, device="cuda", dtype=torch.int64) * 7 % E).view(M, k).int()
    st = xk.moe_balance_loss(z, ids)
    assert int(st.tokens) == M and int(st.counts.sum()) == M * k
    assert abs(float(st.loss) - 1) <= off, float(st.loss) - 1
    mask = torch.ones(M, dtype=torch.bool, device="cuda")
    mask[::3] = False
    half = xk.moe_balance_loss(z, ids, mask=mask)
    assert int(half.tokens) == int(mask.sum())
    assert abs(float(half.loss) - 1) <= off, float(half.loss) - 1


@pytest.mark.parametrize("E,k", [(48, 4), (384, 8), (511, 4), (600, 4), (40, 20)])
def test_counts_past_24_bits(E, k, dev):
    """Counts summed over many batches: near 2^28, a few apart. What the gradient takes is their
    distance from the mean, which is as exact as that of small counts."""
    z, ids, _, _ = _case(70, E, k, torch.float32, seed=E)
    g = torch.Generator().manual_seed(k)
    counts = (2 ** 28 + torch.randint(-40, 41, (E,), generator=g)).int()
    T = 2 ** 30
    gl = torch.tensor(1e9, device="cuda")
    got = xk.moe_router_backward(z, ids, grad_loss=gl, counts=counts.cuda(),
                                 tokens=torch.tensor(T, dtype=torch.int32, device="cuda"))
    z64 = z.double().cpu()
    p, delta = torch.softmax(z64, 1), softmax_delta(z64)
    c = counts.double() - counts.double().mean()
    pc = (p @ c).unsqueeze(1)
    f = 1e9 * E / (float(T) * T * k)
    size = (c - pc).abs() + c.abs() + (p @ c.abs()).unsqueeze(1)
    check(got, f * p * (c - pc), f * p * (3 * delta + 16 * F32) * size)


@pytest.mark.parametrize("M,E", [(40, 100), (300, 384), (40, 700)])
@pytest.mark.parametrize("renorm", [True, False])
def test_probabilities_below_the_least_normal_number(M, E, renorm, dev):
    """Logits 85 to 110 below their row's largest: probabilities down to fp32's least step (2^-149)
    and past it, and gradients that are theirs alone."""
    g = torch.Generator().manual_seed(E)
    z = -85 - 25 * torch.rand(M, E, generator=g)
    z[:, 0] = 0
    ids = torch.stack([torch.randperm(E - 1, generator=g)[:4] + 1 for _ in range(M)]).int()
    ids[::2, 1] = 0
    u = torch.randn(M, 4, generator=g)
    z, ids, u = z.cuda(), ids.cuda(), u.cuda()
    st = _check_loss(z, ids, None)
    gl = torch.tensor(0.7, device="cuda")
    got = xk.moe_router_backward(z, ids, grad_weights=u, renormalize=renorm, grad_loss=gl, counts=st.counts)
    want, bound = router_grad_ref(z, ids, u, renorm, gl, st.counts)
    check(got, want, bound + 8 * 2.0 ** -149)  # (each of a value's few factors and sums has that step)
    # alone: the plain weights' gradient is the probability times u and its distance from the rest
    got = xk.moe_router_backward(z, ids, grad_weights=u, renormalize=renorm)
    want, bound = router_grad_ref(z, ids, u, renorm)
    check(got, want, bound + 8 * 2.0 ** -149)
