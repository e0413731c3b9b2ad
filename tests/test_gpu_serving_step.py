"""The choice of experts, the 4-bit output head and the adjusted logits as a served step uses them, each part against its
definition on the tensors the part before made, then captured and replayed beside eager steps; the layers over the calls with
their gradients; the routing hook with a general router."""
import math

import numpy as np
import pytest

import dense_ref as R
import serving_ref as S

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
H, I, E = 512, 256, 24
ROUTER = dict(score="sigmoid", groups=4, top_groups=2, group_best=2, renorm=True, scale=1.5)


@pytest.fixture(scope="module")
def layer(gpu):
    import synth
    L = synth.SynthLayer(72, E, H, I, (3, 3, 3))
    L.register(gpu, 72)
    return L


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def test_decode_step(gpu, layer):
    """Router -> routed experts -> 4-bit head -> adjusted logits -> drawn token."""
    import _native
    import k_dense
    M, V, L = 4, 4001, 300
    g = _gen(3)
    W = (torch.randn((E, H), generator=g) * 0.1).cuda()
    bias = (torch.randn(E, generator=g) * 0.2).cuda()
    weight = (torch.randn((V, H), generator=g) / math.sqrt(H)).half().cuda()
    head = k_dense.Linear4(weight, group=64, zeros=True)
    x = torch.randn((M, H), generator=g).half().cuda()
    history = torch.randint(0, V, (M, L), generator=g, dtype=torch.int32).cuda()
    lengths = torch.tensor([0, 1, 200, L], dtype=torch.int32).cuda()
    lists = dict(history=history, lengths=lengths, prompt=torch.tensor([0, 1, 120, 0], dtype=torch.int32).cuda(),
                 repetition=torch.tensor([1.3, 1.1, 0.8, 1.0]).cuda(), frequency=torch.tensor([0.2, 0.0, 0.1, -0.3]).cuda(),
                 presence=torch.tensor([0.5, 0.1, 0.0, 0.2]).cuda(),
                 bias_ids=torch.randint(0, V, (M, 5), generator=g, dtype=torch.int32).cuda(), bias=torch.randn((M, 5), generator=g).cuda(),
                 allowed=torch.randint(-2 ** 31, 2 ** 31 - 1, (M, (V + 31) // 32), generator=g, dtype=torch.int64).int().cuda())
    u = torch.rand(M, generator=g).cuda()
    draw = dict(temperature=torch.full((M,), 0.8, device="cuda"), top_k=torch.full((M,), 50, dtype=torch.int32, device="cuda"),
                top_p=torch.full((M,), 0.9, device="cuda"))

    def step(y):
        logits = x.float() @ W.t()
        sel, w = _native.route_experts(logits, 6, bias=bias, **ROUTER)
        gpu.moe_forward(72, x, sel, w, y)
        h = (x + y).half()
        raw = head(h, dtype=F32)
        adjusted = _native.adjust_logits(raw, **lists)
        return (logits, sel, w, h, raw, adjusted) + tuple(_native.sample(adjusted, u, **draw))

    y = torch.empty((M, H), dtype=F32, device="cuda")
    logits, sel, w, h, raw, adjusted, tok, prob = step(y)
    want_sel, want_w = S.route(logits, 6, bias.cpu(), **ROUTER)
    assert torch.equal(sel.cpu(), want_sel)
    # fp64 weights, rounded to fp32 and then to fp16
    S.same(w, want_w, want_w * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -24, "weights")
    S.same(raw, *S.linear(h, head.q, head.scale, head.zero, H, 64, F32, True), "head")
    S.same(adjusted, *S.adjust(raw, **lists), "adjusted")
    for b, (t, p, m) in enumerate(R.sample(adjusted, u, **draw)):
        assert m > 2.0 ** -36 and int(tok[b]) == t
        assert abs(float(prob[b]) - p) <= p * 2.0 ** -23 + V * 2.0 ** -42

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(y)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    yg = torch.empty_like(y)
    with torch.cuda.graph(graph):
        outs = step(yg)
    for _ in range(4):
        x.copy_(torch.randn((M, H), generator=g))
        u.copy_(torch.rand(M, generator=g))
        lengths.copy_(torch.randint(0, L + 1, (M,), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = step(y)
        torch.cuda.synchronize()
        assert torch.equal(yg, y)
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("split", [False, True])
def test_routing_hook_with_a_general_router(gpu, layer, split):
    """Not split: route_experts' own picks. Split, with every expert resident and nothing forced to the host: the same picks
    through the split."""
    import _native
    import routing
    g = _gen(6)
    W = (torch.randn((E, H), generator=g) * 0.1).cuda()
    router = dict(ROUTER, bias=(torch.randn(E, generator=g) * 0.2).cuda())
    pol = torch.tensor([0.4, 0.023, 0.11, 0.104, 0.2, 32, 0.0, 0.0] + [0.0] * 12, device="cuda")
    hook = routing.RoutingHook(W_router=W, E=E, topk=6, li=72, slotof=torch.arange(E, dtype=torch.int32, device="cuda"), pol=pol,
                               ingress=routing.Ingress(H, max_bsz=4, topk=6), router=router)
    for bsz in (1, 3) if split else (5, 40):
        z = torch.randn((bsz, H), generator=g).half().cuda()
        want = _native.route_experts((z.float() @ W.t()).contiguous(), 6, **router)
        sel, w = hook.routing_fn(bsz, None, z, {})
        torch.cuda.synchronize()
        assert torch.equal(sel, want[0]) and torch.equal(w, want[1])
    assert hook.bypassed == (0 if split else 2)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("shape", [(5,), (2, 3), (70,)])
def test_linear4(gpu, dt, shape):
    import _native
    import k_dense
    g = _gen(9)
    N, K = 136, 200
    weight = torch.randn((N, K), generator=g).to(dt).cuda()
    lin = k_dense.Linear4(torch.nn.Parameter(weight), group=32)
    v, s, _ = S.quant(weight.cpu(), 32, False)
    assert torch.equal(S.unpack(lin.q, K), v) and torch.equal(lin.scale.cpu(), s) and lin.zero is None
    same = k_dense.Linear4.from_values(v.to(torch.uint8).cuda(), lin.scale, group=32)
    assert torch.equal(same.q, lin.q)
    x = torch.randn(shape + (K,), generator=g).to(dt).cuda().requires_grad_()
    rows = x.detach().reshape(-1, K)
    y = lin(x)
    assert y.shape == shape + (N,) and y.dtype == dt and torch.equal(y.detach(), same(x.detach()))
    S.same(y.detach().reshape(-1, N), *S.linear(rows, lin.q, lin.scale, None, K, 32, dt, True), "y")
    # a gradient that is broadcast, through a product before the layer
    d, = torch.autograd.grad(lin(x * 2).sum(), x)
    one = _native.linear_i4_dx(torch.ones_like(y).reshape(-1, N), lin.q, lin.scale, K, group=32)
    assert torch.equal(d.reshape(-1, K), one * 2)
    out = torch.empty(shape + (N,), dtype=F32, device="cuda")
    with torch.no_grad():
        lin(x, out=out)
    S.same(out.reshape(-1, N), *S.linear(rows, lin.q, lin.scale, None, K, 32, F32, True), "fp32 y")


def test_capture_with_gradients_is_refused(gpu, monkeypatch):
    import k_dense
    import routing
    lin = k_dense.Linear4(torch.randn((16, 128), generator=_gen(1)).half().cuda())
    x = torch.randn((3, 128), generator=_gen(2)).half().cuda().requires_grad_()
    z = torch.randn((3, 16), generator=_gen(3)).cuda().requires_grad_()
    y, (_, w) = lin(x), routing.route_experts(z, 4)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for f in (lambda: lin(x), lambda: y.sum().backward(), lambda: routing.route_experts(z, 4), lambda: w.sum().backward()):
        with pytest.raises(RuntimeError, match="stream capture"):
            f()


@pytest.mark.parametrize("score,renorm", [("sigmoid", True), ("sigmoid", False), ("softmax", True), ("softmax", False)])
def test_router_in_training(gpu, score, renorm):
    """Router weights trained through the experts' weights: the logits' gradient against the formula, the router's as torch makes
    it of that, and both against a plain router with the same choice."""
    import routing
    M, topk = 33, 4
    g = _gen(12)
    x, W = torch.randn((M, H), generator=g).cuda(), (torch.randn((E, H), generator=g) * 0.05).cuda().requires_grad_()
    bias, c = (torch.randn(E, generator=g) * 0.1).cuda(), torch.randn((M, topk), generator=g).cuda()
    logits = x @ W.t()
    logits.retain_grad()
    sel, w = routing.route_experts(logits, topk, bias=bias, score=score, groups=4, top_groups=3, renorm=renorm, scale=2.0, dtype=F32)
    want_sel, want_w = S.route(logits.detach(), topk, bias.cpu(), score, 4, 3, 2, renorm, 2.0)
    assert torch.equal(sel.cpu(), want_sel)
    S.same(w.detach(), want_w, want_w * 2.0 ** -23 + 2.0 ** -140, "w")
    (w * c).sum().backward()
    S.same(logits.grad, *S.route_gradient(logits.detach(), sel, c, score, renorm, 2.0), "dlogits")
    a, b = logits.grad.double().cpu().t(), x.double().cpu()
    S.same(W.grad, a @ b, (M + 2) * R.U32 * (a.abs() @ b.abs()) + 2.0 ** -140, "dW")
