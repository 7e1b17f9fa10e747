"""The tuning ops together with the framework's own, as a program uses them: a serving
step of router, frozen INT4 experts and a shared INT4 projection with adapters; a
tuning step of router and adapters through torch's autograd, checked against
autograd in 64 bits."""
from __future__ import annotations

import pytest
import torch

import xkernels_amd as xk
from oracle.torch_ref import dequant_w4a16
from tests._tuning_ref import check, half_step, lora_ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


class Adapters(torch.autograd.Function):
    """Adapters beside a frozen projection, the input kept in 8 bits."""

    @staticmethod
    def forward(ctx, x, a, b, base, ids, scaling):
        out, hidden = xk.lora_projection(x, a, b, ids, base=base, scaling=scaling, return_hidden=True)
        ctx.held = xk.act_checkpoint(x)
        ctx.save_for_backward(a, b, ids, scaling, hidden)
        return out

    @staticmethod
    def backward(ctx, grad):
        a, b, ids, scaling, hidden = ctx.saved_tensors
        gx, ga, gb = xk.lora_projection_backward(grad, ctx.held, a, b, ids, hidden, scaling=scaling)
        return gx, ga, gb, grad, None, None


class Router(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, mask):
        w, ids = xk.topk_softmax(logits, k)
        stats = xk.moe_balance_loss(logits, ids, mask=mask)
        ctx.save_for_backward(logits, ids, stats.counts, stats.tokens, mask)
        ctx.mark_non_differentiable(ids)
        return w, ids, stats.loss

    @staticmethod
    def backward(ctx, gw, _, gl):
        logits, ids, counts, tokens, mask = ctx.saved_tensors
        return xk.moe_router_backward(logits, ids, grad_weights=gw, grad_loss=gl, counts=counts, tokens=tokens,
                                      mask=mask), None, None


def _weights(E, N, K, seed):
    packed, scale, _ = xk.make_w4a16_weights(E, N, K, 32, device="cpu", seed=seed)
    return packed.cuda(), scale.cuda()


@pytest.mark.parametrize("M", [1, 33, 500])
def test_serving_step(M, dev):
    E, N, K, k, L, r = 8, 256, 512, 2, 5, 16
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g).to(BF).cuda()
    logits = torch.randn(M, E, generator=g).to(BF).cuda()
    experts, shared = _weights(E, N, K, 1), _weights(1, N, K, 2)
    a = (torch.randn(L, r, K, generator=g) / K ** 0.5).to(BF).cuda()
    b = torch.randn(L, N, r, generator=g).to(BF).cuda()
    ids = torch.randint(-1, L, (M,), generator=g, dtype=torch.int32).cuda()
    sc = torch.rand(L, generator=g).cuda()
    zero, one = torch.zeros(M, 1, dtype=torch.int32, device="cuda"), torch.ones(M, 1, device="cuda")
    w, e = xk.topk_softmax(logits, k)
    routed = xk.fused_moe_int4_w4a16(x, *experts, e, w)
    base = xk.fused_moe_int4_w4a16(x, *shared, zero, one)
    out = xk.lora_projection(x, a, b, ids, base=base, scaling=sc)
    want, _, bound, _ = lora_ref(x, a, b, ids, base, sc)
    check(out, want, bound, "adapters")
    # and the whole sum against dense 64-bit products, to the INT4 op's own tolerance
    dense = x.double() @ dequant_w4a16(*shared).double()[0].t()
    delta, _, _, _ = lora_ref(x, a, b, ids, None, sc)
    total = (out.double() + routed.double()).cpu()
    ref = dense.cpu() + delta
    W = dequant_w4a16(*experts).double()
    ref = ref + sum(w[:, j:j + 1].double().cpu() * torch.einsum("mk,mnk->mn", x.double().cpu(), W[e[:, j].long()].cpu())
                    for j in range(k))
    torch.testing.assert_close(total, ref, rtol=2e-2, atol=2e-2 * float(ref.abs().mean()))


def test_tuning_step(dev):
    M, E, N, K, k, L, r = 300, 16, 192, 256, 4, 3, 8
    g = torch.Generator().manual_seed(0)
    x0 = torch.randn(M, K, generator=g).to(BF).cuda()
    gate = (torch.randn(E, K, generator=g) / K ** 0.5).cuda().requires_grad_()
    a = (torch.randn(L, r, K, generator=g) / K ** 0.5).to(BF).cuda().requires_grad_()
    b = (torch.randn(L, N, r, generator=g) / r ** 0.5).to(BF).cuda().requires_grad_()
    shared = _weights(1, N, K, 3)
    ids = torch.randint(0, L, (M,), generator=g, dtype=torch.int32).cuda()
    sc = torch.full((L,), 2.0, device="cuda")
    mask = (torch.rand(M, generator=g) < 0.9).cuda()
    zero, one = torch.zeros(M, 1, dtype=torch.int32, device="cuda"), torch.ones(M, 1, device="cuda")
    target = torch.randn(M, N, generator=g).cuda()
    for step in range(3):
        logits = (x0.float() @ gate.t())
        w, e, balance = Router.apply(logits, k, mask)
        base = xk.fused_moe_int4_w4a16(x0, *shared, zero, one)
        y = Adapters.apply(x0, a, b, base, ids, sc)
        loss = (w[:, :1] * (y.float() - target)).square().mean() + 0.01 * balance
        ga, gb, gg = torch.autograd.grad(loss, (a, b, gate))

        # the same in 64 bits, at this step's base and selection
        x8 = xk.act_restore(xk.act_checkpoint(x0)).double()
        a64, b64, g64 = (t.detach().double().requires_grad_() for t in (a, b, gate))
        z = x0.double() @ g64.t()
        p = torch.softmax(z, 1)
        sel = p.gather(1, e.long())
        w64 = sel / sel.sum(1, keepdim=True)
        counts = torch.bincount(e[mask].long().flatten(), minlength=E).double()
        bal = E / (int(mask.sum()) ** 2 * k) * (counts @ p[mask].sum(0))
        pick = torch.nn.functional.one_hot(ids.long(), L).double()
        # (values from x, the gradient of a from the 8-bit x)
        h = torch.einsum("mk,lrk,ml->mr", x0.double(), a64.detach(), pick)
        h = h + torch.einsum("mk,lrk,ml->mr", x8, a64 - a64.detach(), pick)
        y64 = base.double() + 2.0 * torch.einsum("mr,lnr,ml->mn", h, b64, pick)
        # rows that the mask leaves out get no gradient through the router's weights
        wm = torch.where(mask.unsqueeze(1), w64, w64.detach())
        l64 = (wm[:, :1] * (y64 - target.double())).square().mean() + 0.01 * bal
        wa, wb, wg = torch.autograd.grad(l64, (a64, b64, g64))
        # bf16 y and bf16 grad_out: half a step each, on every term of a sum whose terms'
        # magnitudes a random sum's norm stands for: 4 half steps of the norm
        for name, got, want in (("a", ga, wa), ("b", gb, wb), ("gate", gg, wg)):
            off = float((got.double() - want).norm() / want.norm())
            assert off <= 4 * half_step(BF), (step, name, off)
        with torch.no_grad():
            a -= 0.1 * ga
            b -= 0.1 * gb
            gate -= 0.1 * gg


def test_calls_outside_autograd_say_so(dev, monkeypatch):
    """The forwards warn in grad mode, once each, and give the same values; wrapped or under
    no_grad they are silent."""
    import warnings

    from xkernels_amd.moe import hip_tuning

    monkeypatch.setattr(hip_tuning, "_told", set())
    g = torch.Generator().manual_seed(2)
    x = torch.randn(9, 64, generator=g).to(BF).cuda()
    a, b = torch.randn(2, 4, 64, generator=g).to(BF).cuda(), torch.randn(2, 32, 4, generator=g).to(BF).cuda()
    ids = torch.randint(0, 2, (9,), generator=g, dtype=torch.int32).cuda()
    z = torch.randn(9, 16, generator=g).cuda()
    top = torch.topk(z, 2, 1).indices.int()
    sc = torch.ones(2, device="cuda")
    base = torch.zeros(9, 32, dtype=BF, device="cuda")
    calls = {"lora_projection": lambda: (xk.lora_projection(x, a, b, ids, base=base, scaling=sc),),
             "moe_balance_loss": lambda: tuple(xk.moe_balance_loss(z, top)),
             "act_checkpoint": lambda: tuple(t.view(torch.uint8) for t in xk.act_checkpoint(x))}
    want = {k: f() for k, f in calls.items()}
    for t in (x, a, z):
        t.requires_grad_()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with torch.no_grad():
            for f in calls.values():
                f()
        Adapters.apply(x, a, b, base, ids, sc).sum().backward()
        Router.apply(z, 2, torch.ones(9, dtype=torch.bool, device="cuda"))[2].backward()
    assert a.grad is not None and z.grad is not None
    for name, f in calls.items():
        with pytest.warns(RuntimeWarning, match=name):
            got = f()
        assert all(torch.equal(p, q) for p, q in zip(got, want[name]))
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            f()


@pytest.mark.parametrize("renorm", [True, False])
def test_router_gradient_through_the_experts(renorm, dev):
    """The router's weights get their gradient from the experts themselves: a slot's is the output's
    gradient times that slot's expert output, which the fused op gives for the slot alone."""
    from tests._tuning_ref import gamma, router_grad_ref

    M, E, N, K, k = 70, 16, 192, 256, 4
    g = torch.Generator().manual_seed(4)
    x = torch.randn(M, K, generator=g).to(BF).cuda()
    z = torch.randn(M, E, generator=g).cuda()
    experts = _weights(E, N, K, 5)
    gy = torch.randn(M, N, generator=g).cuda()
    w, ids = xk.topk_softmax(z, k, renormalize=renorm)
    st = xk.moe_balance_loss(z, ids)
    one = torch.ones(M, 1, device="cuda")
    slots = [xk.fused_moe_int4_w4a16(x, *experts, ids[:, j:j + 1].contiguous(), one) for j in range(k)]
    gw = torch.stack([(gy * o.float()).sum(1) for o in slots], 1)
    gl = torch.tensor(0.01, device="cuda")
    got = xk.moe_router_backward(z, ids, grad_weights=gw, renormalize=renorm, grad_loss=gl, counts=st.counts)
    # in 64 bits, from the dequantised weights
    W = dequant_w4a16(*experts).double().cpu()
    o64 = torch.stack([torch.einsum("mk,mnk->mn", x.double().cpu(), W[ids[:, j].long().cpu()]) for j in range(k)], 1)
    mag = torch.stack([torch.einsum("mk,mnk->mn", x.double().cpu().abs(), W[ids[:, j].long().cpu()].abs())
                       for j in range(k)], 1)
    gy64 = gy.double().cpu().unsqueeze(1)
    u64 = (gy64 * o64).sum(2)
    # a slot's output: fp32 sums over K, half a step of bf16 (and of the slot's own sum over one slot);
    # their products' fp32 sum over N
    off_o = 2 * half_step(BF) * o64.abs() + gamma(K) * mag
    off_u = (gy64.abs() * (off_o + gamma(N) * o64.abs())).sum(2)
    check(gw, u64, off_u, "grad_weights")
    want, bound = router_grad_ref(z, ids, u64, renorm, gl, st.counts)
    p = torch.softmax(z.double().cpu(), 1)
    pj = p.gather(1, ids.long().cpu())
    wj = pj / pj.sum(1, keepdim=True) if renorm else pj
    mean = (wj * off_u).sum(1, keepdim=True)
    bound = bound.scatter_add(1, ids.long().cpu(), wj * (off_u + mean if renorm else off_u))
    if not renorm:
        bound = bound + p * mean
    check(got, want, bound, "logits")
