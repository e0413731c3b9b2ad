"""The general router where its choice is close or its logits are extreme, against the 64-bit definition by whole tensors."""
import pytest

import serving_ref as S

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _first(v, n):
    """Indices of the n largest along the last dimension, equal ones by index."""
    return torch.sort(v, dim=-1, descending=True, stable=True)[1][..., :n]


def _kept(key, groups, top_groups, group_best):
    """Which experts belong to the kept groups, by fp64 keys without -inf."""
    k = key.view(key.shape[0], groups, -1)
    worth = torch.sort(k, dim=2, descending=True)[0][:, :, :group_best].sum(2)
    kept = torch.zeros_like(worth, dtype=torch.bool).scatter_(1, _first(worth, top_groups), True)
    return kept[:, :, None].expand_as(k).reshape(key.shape)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("group_best", [1, 2])
@pytest.mark.parametrize("M", [300, 6200, 12300])
@pytest.mark.parametrize("forced", [0.1, 16.0, 64.0, 1000.0, 10000.0, 3e38])
def test_close_groups_with_large_biases(gpu, M, forced, group_best, score):
    """Groups of nearly the same keys in which one expert is forced by its bias and the rest are held off, so that a group's worth is a
    small difference of large keys: fp32 orders some of them otherwise than fp64."""
    import _native
    E, groups, top, topk = 32, 4, 2, 4
    g = _gen(M + int(min(forced, 1e6)))
    step = max(min(forced, 1e4) * 2.0 ** -20, 2.0 ** -18)
    x = torch.randn((M, 8), generator=g).repeat(1, groups) + step * torch.randn((M, E), generator=g)
    b = torch.full((E,), -forced)
    b[::8] = forced
    if forced > 1e30:
        b[::8] *= -1.0           # both of a group's best: their fp32 sum is not finite
    p = torch.sigmoid(x.double()) if score == "sigmoid" else torch.softmax(x.double(), 1)
    key = p + b.double()
    kept = _kept(key, groups, top, group_best)
    want = _first(torch.where(kept, key, -INF), topk)
    sel, _ = _native.route_experts(x.cuda(), topk, bias=b.cuda(), score=score, groups=groups, top_groups=top, group_best=group_best)
    wrong = (sel.cpu() != want).any(1)
    assert not wrong.any(), f"{int(wrong.sum())} of {M}"


@pytest.mark.parametrize("dt,wt", [(F32, F32), (BF16, F32), (F16, BF16)])
@pytest.mark.parametrize("lead", [0.0, 12.0, 16.0, 20.0, 25.0, 40.0])
@pytest.mark.parametrize("M,E,topk", [(70, 128, 8), (8200, 128, 8), (5, 1000, 64)])
def test_gradient_of_rows_that_few_experts_lead(gpu, M, E, topk, lead, dt, wt):
    """Softmax without renormalisation: dx = p (ds - sum p ds) = p_i sum_j p_j (ds_i - ds_j), the second form without cancellation. Of
    every three rows, one is led by one expert, one by all the picks, whose dw are then equal."""
    import _native
    g = _gen(M + E)
    x = torch.randn((M, E), generator=g)
    x[::3, 17] += lead
    x[1::3, 3:3 + topk] += lead
    x = x.to(dt)
    dw = torch.randn((M, topk), generator=g)
    dw[1::3] = dw[1::3, :1]
    dw = dw.to(wt)
    sel, _ = _native.route_experts(x.cuda(), topk, score="softmax", renorm=False, scale=16.0)
    got = _native.route_experts_backward(dw.cuda(), x.cuda(), sel, score="softmax", renorm=False, scale=16.0)
    rows = torch.arange(0, M, max(1, M // 100))
    sel, got, dw = sel.cpu()[rows], got.cpu()[rows], dw.double()[rows] * 16
    p = torch.softmax(x[rows].double(), 1)
    ds = torch.zeros_like(p).scatter_(1, sel, dw)
    diff = ds[:, :, None] - ds[:, None, :]
    value, spread = p * (diff * p[:, None, :]).sum(2), p * (diff.abs() * p[:, None, :]).sum(2)
    # a softmax of exponentials within 2^-35 of theirs, its sum and the weighted one in fp64; then fp32, then the type
    err = 2.0 ** -32 * spread + (E + topk + 10) * 2.0 ** -53 * p * ((p * ds.abs()).sum(1, keepdim=True) + ds.abs())
    S.same(got, value, err + (S.half_step(dt) + 2.0 ** -24) * (value.abs() + err) + S.tiny(dt) + 2.0 ** -150, "dlogits")


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("M", [5, 8200])
def test_gradient_does_not_read_the_weights_of_missing_picks(gpu, M, score, renorm):
    """NaN and infinities in dw where sel is -1 or an id that no expert has: as if they were 0."""
    import _native
    g = _gen(M)
    x = torch.randn((M, 32), generator=g)
    x[::2, 3:] = -INF
    x, dw = x.cuda(), torch.randn((M, 6), generator=g).cuda()
    sel, _ = _native.route_experts(x, 6, score=score, renorm=renorm)
    assert bool((sel[::2, 3:] == -1).all())
    odd = sel.clone()
    odd[1, 2], odd[1, 4] = 32, -9
    zero = torch.where((odd < 0) | (odd > 31), 0.0, dw)
    bad = zero.clone()
    bad[::2, 3], bad[::2, 4], bad[::2, 5], bad[1, 2], bad[1, 4] = NAN, INF, -INF, NAN, INF
    a, b = (_native.route_experts_backward(t, x, odd, score=score, renorm=renorm) for t in (zero, bad))
    assert bool(torch.isfinite(a).all()) and torch.equal(a, b)


@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("M", [9, 6200, 12300])
def test_saturated_scores_go_by_the_logit_with_and_without_groups(gpu, M, score, dt):
    """Logits whose fp64 scores are equal (sigmoid 1 from 37 on, softmax 0 some 745 below the largest) are still in order. The first
    group has the largest and is kept, so that its choice is that of a router of its experts alone."""
    import _native
    g = _gen(M)
    x = torch.randn((M, 32), generator=g)
    if score == "sigmoid":
        x[:, :16] = x[:, :16] * 3 + 60
    else:
        x[:, 1:16] = x[:, 1:16] * 30 - 2000
        x[:, 16:] -= 4000
        x[:, 0] = 0
    x[::3, 2], x[::3, 9], x[1::3, 4], x[2::3, 5] = x[::3, 11], x[::3, 11], -INF, NAN
    x = x.to(dt)
    v = torch.where(x > -INF, x.double(), -INF)[:, :16]
    for topk in (1, 4, 12):
        sel, _ = _native.route_experts(x.cuda(), topk, score=score, groups=2, top_groups=1)
        assert torch.equal(sel.cpu(), _first(v, topk))
        whole, _ = _native.route_experts(x.cuda(), topk, score=score)
        assert torch.equal(whole, sel)
    one = torch.full((1, 8), -9.0)
    one[0, 0], one[0, 1] = 40.0, 60.0
    assert _native.route_experts(one.cuda(), 1, groups=2, top_groups=1)[0].tolist() == [[1]]


@pytest.mark.parametrize("M", [4, 6200, 12300])
def test_renormalised_softmax_of_picks_far_below_the_largest(gpu, M):
    """A bias that holds off the experts that lead by 2000: weights and gradients are those of a softmax of the picks alone."""
    import _native
    g = _gen(M)
    x = torch.randn((M, 40), generator=g)
    x[:, 30:] += 2000
    b = torch.zeros(40)
    b[30:], b[:30] = -5.0, torch.arange(30) * 1e-3
    dw = torch.randn((M, 6), generator=g)
    sel, w = _native.route_experts(x.cuda(), 6, bias=b.cuda(), score="softmax", dtype=F32)
    dx = _native.route_experts_backward(dw.cuda(), x.cuda(), sel, score="softmax")
    assert torch.equal(sel.cpu(), torch.arange(29, 23, -1).expand(M, -1))
    p = torch.softmax(x[:, 24:30].double().flip(1), 1)
    S.same(w, p, (2.0 ** -24 + 2.0 ** -48) * p, "w")
    d = dw.double()
    want = torch.zeros((M, 40), dtype=torch.float64)
    want[:, 24:30] = (p * (d - (p * d).sum(1, keepdim=True))).flip(1)
    err = torch.zeros_like(want)
    err[:, 24:30] = (2.0 ** -48 * p * (d.abs() + (p * d.abs()).sum(1, keepdim=True))).flip(1)
    S.same(dx, want, err + 2.0 ** -24 * (want.abs() + err) + 2.0 ** -150, "dlogits")


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("M,E,topk", [(1, 288, 8), (65, 128, 8), (3, 1024, 64), (6200, 64, 6), (12300, 128, 8)])
def test_softmax_weights_of_the_whole_row_in_fp32(gpu, M, E, topk, dt):
    """Not renormalised: a row's sum is of exponentials within 2^-35, the weight's own rounded once."""
    import _native
    x = (torch.randn((M, E), generator=_gen(E)) * 3).to(dt)
    sel, w = _native.route_experts(x.cuda(), topk, score="softmax", renorm=False, scale=2.5, dtype=F32)
    v = x.double()
    want = _first(v, topk)
    assert torch.equal(sel.cpu(), want)
    p = 2.5 * torch.softmax(v, 1).gather(1, want)
    S.same(w, p, (2.0 ** -24 + 2.0 ** -34) * p + 2.0 ** -150, "w")


@pytest.mark.parametrize("E", [64, 100, 128, 1024])
@pytest.mark.parametrize("M", [3, 8200])
def test_rows_without_experts_have_no_gradient(gpu, M, E):
    """All logits NaN, or -inf, or some of each: nothing is picked, and dx is 0."""
    import _native
    x = torch.randn((M, E), generator=_gen(E))
    x[::3], x[1::3] = NAN, -INF
    x[1::6, ::2] = NAN
    dw = torch.randn((M, 4), generator=_gen(1)).cuda()
    for score in ("sigmoid", "softmax"):
        for renorm in (True, False):
            sel, w = _native.route_experts(x.cuda(), 4, score=score, renorm=renorm)
            dx = _native.route_experts_backward(dw, x.cuda(), sel, score=score, renorm=renorm)
            for i in (0, 1):
                assert bool((sel[i::3] == -1).all()) and bool((w[i::3] == 0).all()) and bool((dx[i::3] == 0).all())
            assert bool((sel[2::3] >= 0).all()) and bool(torch.isfinite(dx).all())
