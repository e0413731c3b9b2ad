"""The general router on the GPU (gfl_route_experts and its backward) against its 64-bit definition: the picks equal, the weights and
gradients within the roundings."""
import pytest

import serving_ref as S
from dense_ref import half_step, tiny

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _logits(M, E, dt, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.full((M, E + pad), NAN)
    x[:, :E] = torch.randn((M, E), generator=g) * 2
    return x.to(dt).cuda()[:, :E], torch.randn(E, generator=g).mul_(0.1).cuda()


def _check(x, topk, dtype=F16, **kw):
    import _native
    print("route_experts", list(x.shape), x.dtype, topk, {k: v for k, v in kw.items() if k != "bias"}, flush=True)
    sel, w = _native.route_experts(x, topk, dtype=dtype, **kw)
    bias = kw.get("bias")
    want_s, want_w = S.route(x, topk, **dict(kw, bias=None if bias is None else bias.cpu()))
    assert torch.equal(sel.cpu(), want_s)
    assert w.dtype == dtype
    S.same(w, want_w, (half_step(dtype) + 2.0 ** -48) * want_w.abs() + tiny(dtype), "w")
    return sel, w


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("M,E,topk", [(1, 288, 8), (1, 8, 2), (7, 60, 4), (65, 128, 8), (130, 256, 6), (5, 1024, 16), (3, 64, 64),
                                      (2, 1, 1), (9, 77, 5), (33, 513, 1), (1025, 40, 3)])
def test_scores(gpu, M, E, topk, score, dt):
    x, b = _logits(M, E, dt, M + E)
    for bias in (None, b):
        for renorm in (True, False):
            _check(x, topk, bias=bias, score=score, renorm=renorm, scale=2.5, dtype=F32 if renorm else BF16)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("M,E,groups,top,topk", [(1, 256, 8, 4, 8), (70, 256, 8, 4, 8), (9, 160, 8, 3, 6), (5, 60, 3, 2, 7),
                                                 (4, 64, 64, 9, 9), (3, 1023, 33, 5, 16), (6, 96, 2, 1, 6), (2000, 128, 4, 2, 8),
                                                 (3, 1024, 64, 63, 64), (12, 21, 7, 7, 3), (1, 1024, 2, 1, 64)])
def test_groups(gpu, M, E, groups, top, topk, score):
    x, b = _logits(M, E, F32, E + groups)
    for best in (1, 2):
        for bias in (None, b):
            _check(x, topk, bias=bias, score=score, groups=groups, top_groups=top, group_best=best, dtype=F32)


@pytest.mark.parametrize("dt,score,bias", [(F32, "sigmoid", True), (F32, "softmax", True), (F32, "softmax", False), (BF16, "sigmoid", False),
                                           (F16, "sigmoid", True)])
@pytest.mark.parametrize("M,E,groups,top,topk", [(6200, 72, 1, 1, 8), (6200, 256, 8, 4, 8), (6200, 1024, 32, 9, 30), (12300, 16, 1, 1, 2),
                                                 (12300, 128, 4, 2, 6), (12300, 250, 1, 1, 15), (12300, 40, 5, 3, 8)])
def test_many_tokens(gpu, M, E, groups, top, topk, dt, score, bias):
    """Batches whose tokens share a wave, two or four to one; a part of them by the definition, all of them as in a smaller batch."""
    import _native
    x, b = _logits(M, E, dt, M + E)
    x[::7] = x[::7].round() if dt == F32 else x[::7]          # rows with ties
    kw = dict(bias=b if bias else None, score=score, groups=groups, top_groups=top, dtype=F32)
    sel, w = _native.route_experts(x, topk, **kw)
    for i in range(0, M, 1000):
        s2, w2 = _native.route_experts(x[i:i + 1000], topk, **kw)
        assert torch.equal(sel[i:i + 1000], s2) and torch.equal(w[i:i + 1000], w2)
    rows = torch.arange(0, M, 61, device="cuda")
    want_s, want_w = S.route(x[rows], topk, bias=b.cpu() if bias else None, score=score, groups=groups, top_groups=top)
    assert torch.equal(sel[rows].cpu(), want_s)
    S.same(w[rows], want_w, (half_step(F32) + 2.0 ** -48) * want_w.abs(), "w")


def test_many_tokens_gradient(gpu):
    import _native
    for E, topk in ((64, 4), (16, 2), (288, 8)):
        x, b = _logits(8200, E, BF16, E)
        dw = torch.randn((8200, topk), generator=torch.Generator().manual_seed(1)).cuda()
        for score, renorm in (("softmax", False), ("sigmoid", True)):
            sel, _ = _native.route_experts(x, topk, bias=b, score=score, renorm=renorm)
            got = _native.route_experts_backward(dw, x, sel, score=score, renorm=renorm)
            rows = torch.arange(0, 8200, 37, device="cuda")
            S.same(got[rows], *S.route_gradient(x[rows], sel[rows], dw[rows], score, renorm), "dlogits")


def test_crowded_borders(gpu):
    """Rows of few distinct keys: more candidates at the border than fp32 can order, in every lane layout."""
    import _native
    for M in (5, 6200, 12300):
        g = torch.Generator().manual_seed(M)
        x = torch.randint(0, 3, (M, 96), generator=g).float()
        b = torch.randint(0, 2, (96,), generator=g).float() * 3e-8 + 0.125
        x[1::2] += torch.randint(0, 4, (len(x[1::2]), 96), generator=g) * 2.0 ** -20
        x = x.cuda()
        for kw in (dict(), dict(bias=b.cuda()), dict(groups=6, top_groups=2), dict(bias=b.cuda(), score="softmax")):
            sel, w = _native.route_experts(x, 7, dtype=F32, **kw)
            rows = torch.arange(0, M, max(1, M // 97), device="cuda")
            want_s, want_w = S.route(x[rows], 7, **{k: v.cpu() if k == "bias" else v for k, v in kw.items()})
            assert torch.equal(sel[rows].cpu(), want_s), kw


def test_ties_go_to_the_lower_index(gpu):
    x = torch.zeros((4, 96))
    x[1, 40:50] = 3.0
    x[2] = torch.arange(96) % 3
    x[3, ::2] = -0.0
    b = torch.zeros(96)
    b[90] = 1e-9     # below fp32's step at 0.5 + b, above fp64's
    for dt in (F32, BF16):
        for score in ("sigmoid", "softmax"):
            for bias in (None, b.cuda()):
                for kw in ({}, dict(groups=4, top_groups=2)):
                    _check(x.to(dt).cuda(), 8, bias=bias, score=score, **kw)


def test_scores_that_fp32_cannot_tell_apart(gpu):
    """Keys 1e-9 apart, in an order that is not the index's."""
    x = torch.full((3, 64), 0.25)
    b = torch.arange(64).flip(0).float() * 1e-9
    sel, _ = _check(x.cuda(), 8, bias=b.cuda())
    assert sel[0].tolist() == list(range(8))
    sel, _ = _check(x.cuda(), 8, bias=b.flip(0).contiguous().cuda())
    assert sel[0].tolist() == list(range(63, 55, -1))


def test_experts_that_are_not_there(gpu):
    """-inf and NaN are never picked; rows with too few, or none, end in -1 with weight 0; +inf and huge values."""
    x, b = _logits(9, 40, F32, 3)
    x[0, 3:] = -INF
    x[1] = -INF
    x[2] = NAN
    x[3, ::2] = NAN
    x[4, 7] = INF
    x[5, 5] = x[5, 25] = INF
    x[6] = -3e38
    x[7, 1:] = -1000.0
    b2 = b.clone()
    b2[9], b2[11], b2[13] = NAN, -INF, INF
    for score in ("sigmoid", "softmax"):
        for bias in (None, b, b2):
            for kw in ({}, dict(groups=8, top_groups=3), dict(groups=8, top_groups=2, group_best=1)):
                for renorm in (True, False):
                    sel, w = _check(x, 6, bias=bias, score=score, renorm=renorm, **kw)
                    assert bool((sel[1:3] == -1).all()) and bool((w[1:3] == 0).all())
    sel, w = _check(x, 6)
    assert sel[0].tolist()[3:] == [-1] * 3


def test_strided_rows_empty_and_streams(gpu):
    import _native
    x, b = _logits(21, 77, F32, 5, pad=3)
    sel, w = _check(x, 5, bias=b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sel2, w2 = _native.route_experts(x, 5, bias=b)
    s.synchronize()
    assert torch.equal(sel, sel2) and torch.equal(w, w2)
    sel, w = _native.route_experts(x[:0], 5)
    assert sel.shape == w.shape == (0, 5)
    assert _native.route_experts_backward(w, x[:0], sel).shape == (0, 77)


@pytest.mark.parametrize("dt,wt", [(F32, F32), (BF16, F32), (F16, F16), (F32, BF16)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("M,E,topk", [(1, 288, 8), (65, 60, 4), (3, 1024, 64), (2, 1, 1), (130, 129, 2), (1500, 64, 8)])
def test_gradient(gpu, M, E, topk, score, dt, wt):
    import _native
    x, _ = _logits(M, E, dt, M * 3 + E, pad=2)
    g = torch.Generator().manual_seed(E)
    dw = torch.randn((M, topk), generator=g).to(wt).cuda()
    for renorm in (True, False):
        sel, _ = _native.route_experts(x, topk, score=score, renorm=renorm, scale=1.5)
        print("route_experts_backward", M, E, topk, score, dt, renorm, flush=True)
        got = _native.route_experts_backward(dw, x, sel, score=score, renorm=renorm, scale=1.5)
        assert got.dtype == dt
        S.same(got, *S.route_gradient(x, sel, dw, score, renorm, 1.5), "dlogits")


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [True, False])
def test_gradient_against_differences(gpu, score, renorm):
    import _native
    x, b = _logits(5, 33, F32, 8)
    sel, _ = _native.route_experts(x, 4, bias=b, score=score, renorm=renorm)
    g = torch.Generator().manual_seed(1)
    dw, v = torch.randn((5, 4), generator=g).cuda(), torch.randn((5, 33), generator=g).double()
    got = _native.route_experts_backward(dw, x, sel, score=score, renorm=renorm).double().cpu()
    xd, h = x.double().cpu(), 1e-6
    f = lambda t: float((S.route_weights(t, sel.cpu(), score, renorm) * dw.double().cpu()).sum())
    num = (f(xd + h * v) - f(xd - h * v)) / (2 * h)
    _, bound = S.route_gradient(x, sel, dw, score, renorm)
    # the difference is off by h^2 / 6 of the third derivative and 2^-52 / h of the value
    assert abs(float((got * v).sum()) - num) <= float((bound * v.abs()).sum()) + 1e-8


def test_gradient_skips_missing_picks_and_takes_rows_that_are_not_there(gpu):
    import _native
    x, _ = _logits(4, 20, F32, 2)
    x[0, 2:] = -INF
    x[1] = -INF
    x[2, 3] = NAN
    dw = torch.randn((4, 5), generator=torch.Generator().manual_seed(3)).cuda()
    for score in ("sigmoid", "softmax"):
        for renorm in (True, False):
            sel, _ = _native.route_experts(x, 5, score=score, renorm=renorm)
            got = _native.route_experts_backward(dw, x, sel, score=score, renorm=renorm).cpu()
            assert bool((got[0, 2:] == 0).all()) and bool((got[1] == 0).all()) and float(got[2, 3]) == 0
            assert bool(torch.isfinite(got).all())
            keep = x[:1, :2]
            S.same(got[:1, :2], *S.route_gradient(keep, sel[:1, :2], dw[:1, :2], score, renorm), "two experts left")
            odd = sel.clone()
            odd[3, 1], odd[3, 2] = 20, -7      # ids that no expert has
            ok = sel.clone()
            ok[3, 1:3] = -1
            a, b = (_native.route_experts_backward(dw, x, t, score=score, renorm=renorm) for t in (odd, ok))
            assert torch.equal(a, b)


def test_the_closed_form_router_agrees(gpu):
    """_native.route (fp32 scores, no bias) picks the same experts with weights within its roundings."""
    import _native
    x, _ = _logits(200, 288, F32, 9)
    sel, w = _native.route(x, 8)
    sel2, w2 = _native.route_experts(x, 8)
    assert torch.equal(sel, sel2)
    assert float((w.double() - w2.double()).abs().max()) <= 2.0 ** -11


def test_captured(gpu):
    import _native
    x, b = _logits(33, 96, F32, 6)
    dw = torch.randn((33, 4), generator=torch.Generator().manual_seed(1)).cuda()
    _native.route_experts_backward(dw, x, _native.route_experts(x, 4, bias=b, groups=4, top_groups=2)[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sel, w = _native.route_experts(x, 4, bias=b, groups=4, top_groups=2)
        dx = _native.route_experts_backward(dw, x, sel)
    for seed in (1, 2, 3):
        x.copy_(_logits(33, 96, F32, seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        want = _native.route_experts(x, 4, bias=b, groups=4, top_groups=2)
        assert torch.equal(sel, want[0]) and torch.equal(w, want[1])
        assert torch.equal(dx, _native.route_experts_backward(dw, x, want[0]))
