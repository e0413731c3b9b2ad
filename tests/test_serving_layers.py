"""The layers over the 4-bit products and the choice of experts without a GPU: what k_dense.Linear4, routing.route_experts and
RoutingHook refuse, and what they hand to the library's calls, with plain torch operations in their place."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import _native
import k_dense
import routing
import serving_ref as S


def _plain_calls(monkeypatch):
    made = []

    def linear_i4(x, q, scale, zero=None, group=128, out=None, dtype=None):
        made.append(("linear", zero is not None, group, out is not None, dtype))
        with torch.no_grad():
            return (x.double() @ q.double().t()).to(dtype or x.dtype)

    def linear_i4_dx(dy, q, scale, K, zero=None, group=128):
        assert dy.is_contiguous() and K == q.shape[1]
        made.append(("dx", zero is not None, group))
        return (dy.double() @ q.double()).to(dy.dtype)

    def route_experts(logits, topk=8, bias=None, score="sigmoid", groups=1, top_groups=1, group_best=2, renorm=True, scale=1.0, dtype=None):
        made.append(("route", topk, bias is not None, score, groups, top_groups, group_best, renorm, scale, dtype))
        sel, w = S.route(logits.detach(), topk, bias, score, groups, top_groups, group_best, renorm, scale)
        return sel, w.to(dtype or torch.float16)

    def route_experts_backward(dw, logits, sel, score="sigmoid", renorm=True, scale=1.0):
        assert dw.is_contiguous()
        with torch.enable_grad():
            return S.route_gradient(logits.detach(), sel, dw, score, renorm, scale)[0].to(logits.dtype)

    monkeypatch.setattr(_native, "linear_i4", linear_i4)
    monkeypatch.setattr(_native, "linear_i4_dx", linear_i4_dx)
    monkeypatch.setattr(_native, "route_experts", route_experts)
    monkeypatch.setattr(_native, "route_experts_backward", route_experts_backward)
    monkeypatch.setattr(_native, "quant_i4", lambda w, group=128, zeros=False: (w.float(), torch.ones(1), torch.ones(1) if zeros else None))
    return made


def test_linear4_on_plain_calls(monkeypatch):
    made = _plain_calls(monkeypatch)
    w = torch.randn(6, 40).half()
    lin = k_dense.Linear4(w.clone().requires_grad_(), group=32, zeros=True)
    x = torch.randn(2, 3, 40).half()
    assert not lin(x).requires_grad and made[-1] == ("linear", True, 32, False, None)
    assert lin(x, dtype=torch.float32).dtype == torch.float32
    a = x.clone().requires_grad_()
    y = lin(a * 2)
    assert y.shape == (2, 3, 6)
    y.sum().backward()          # an expanded gradient reaches the call as a tensor of its own
    want = w.double().sum(0) * 2
    assert (a.grad.double() - want).abs().max() <= 2.0 ** -9 * want.abs().max()
    with torch.no_grad():
        assert not lin(a).requires_grad
    y = lin(a)
    d, = torch.autograd.grad(y, a, torch.ones_like(y).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|once differentiable"):
        d.sum().backward()


def test_linear4_refusals(monkeypatch):
    v, s = torch.zeros((4, 100), dtype=torch.uint8), torch.ones((1, 4)).half()
    for bad, word in (((v[0], s), "values"), ((v, s.t()), "scale"), ((v, s, s.repeat(2, 1)), "zero")):
        with pytest.raises(ValueError, match=word):
            k_dense.Linear4.from_values(*bad)
    with pytest.raises(ValueError, match="group"):
        k_dense.Linear4.from_values(v, s, group=100)
    with pytest.raises(ValueError, match="device"):
        k_dense.Linear4.from_values(v, s)
    for bad in (torch.zeros(8).half(), torch.zeros(8, 0).half(), torch.zeros(2, 3, 4).half()):
        with pytest.raises(ValueError, match="Linear4"):
            k_dense.Linear4(bad)
    with pytest.raises(ValueError, match="device"):
        k_dense.Linear4(torch.zeros(4, 8).half())
    _plain_calls(monkeypatch)
    lin = k_dense.Linear4(torch.randn(4, 8).half())
    x = torch.randn(2, 8).half()
    a = x.clone().requires_grad_()
    for kw in (dict(dtype=torch.float32), dict(out=torch.zeros(2, 4).half())):
        lin(x, **kw)
        with pytest.raises(RuntimeError, match="Linear4.*gradient"):
            lin(a, **kw)
        with torch.no_grad():
            lin(a, **kw)
    with pytest.raises(RuntimeError, match="Linear4.*gradient"):
        lin(x, out=torch.zeros(2, 4).half().requires_grad_())
    with fwd.dual_level(), pytest.raises(RuntimeError, match="Linear4.*forward-mode"):
        lin(fwd.make_dual(x, torch.ones_like(x)))


def test_differentiable_router_on_plain_calls(monkeypatch):
    made = _plain_calls(monkeypatch)
    g = torch.Generator().manual_seed(5)
    x, bias = torch.randn((5, 24), generator=g), torch.randn(24, generator=g) * 0.1
    kw = dict(bias=bias, groups=4, top_groups=2, group_best=1, renorm=False, scale=2.5, dtype=torch.float32)
    sel, w = routing.route_experts(x, 3, **kw)
    assert not w.requires_grad and made[-1] == ("route", 3, True, "sigmoid", 4, 2, 1, False, 2.5, torch.float32)
    a = x.clone().requires_grad_()
    sel2, w2 = routing.route_experts(a, 3, **kw)
    assert torch.equal(sel, sel2) and not sel2.requires_grad and w2.requires_grad
    w2.sum().backward()
    want = S.route_gradient(x, sel, torch.ones(5, 3), "sigmoid", False, 2.5)[0]
    assert torch.equal(a.grad, want.float())
    with pytest.raises(RuntimeError, match="bias"):
        routing.route_experts(x, 3, **dict(kw, bias=bias.clone().requires_grad_()))
    with torch.no_grad():
        assert not routing.route_experts(a, 3, **dict(kw, bias=bias.clone().requires_grad_()))[1].requires_grad
    for i in range(2):
        with fwd.dual_level(), pytest.raises(RuntimeError, match="route_experts.*forward-mode"):
            t = [x, bias]
            t[i] = fwd.make_dual(t[i], torch.ones_like(t[i]))
            routing.route_experts(t[0], 3, **dict(kw, bias=t[1]))


def test_hook_with_a_general_router(monkeypatch):
    made = _plain_calls(monkeypatch)
    ing = routing.Ingress(8, max_bsz=2, topk=4, device="cpu")
    kw = dict(E=16, topk=4, slotof=torch.zeros(16, dtype=torch.int32), pol=torch.zeros(20), ingress=ing)
    W = torch.randn(16, 8)
    for bad in (dict(W_router=W, router=dict(topk=3)), dict(W_router=W, router=dict(dtype=torch.float32)), dict(orig=print, router={})):
        with pytest.raises(ValueError, match="routing hook"):
            routing.RoutingHook(**kw, **bad)
    split = []

    def plain_split(sel, w, zz, E, first, slotof, score, pol, ctrl, hx, picks, seq, li, many, so, wo, dflag, stats, rres):
        split.append(seq)
        so.copy_(sel.view(-1))
        wo.copy_(w.view(-1))

    monkeypatch.setattr(_native, "split", plain_split)
    hook = routing.RoutingHook(W_router=W, router=dict(bias=torch.zeros(16), score="softmax", groups=4, top_groups=2, scale=2.0), **kw)
    z = torch.randn(2, 8).half()
    sel, w = hook.routing_fn(2, None, z, {})
    assert made[-1] == ("route", 4, True, "softmax", 4, 2, 2, True, 2.0, None) and split == [1] and hook.pending
    ref = S.route(z.float() @ W.t(), 4, torch.zeros(16), "softmax", 4, 2, 2, True, 2.0)
    assert torch.equal(sel, ref[0]) and torch.equal(w, ref[1].half()) and sel.shape == (2, 4)
    for bsz, params in ((3, {}), (2, {"tp_warmup": True})):
        sel, w = hook.routing_fn(bsz, None, torch.randn(bsz, 8).half(), params)
        assert sel.shape == (bsz, 4) and split == [1] and not hook.pending
    assert hook.bypassed == 2
