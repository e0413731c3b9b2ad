"""Infinities and NaN through the gated feed-forward block, with and without its clamp: what is not a number in a token or a
weight is not a number in what depends on it, as in the formulas, and nowhere else."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16 = torch.float16, torch.bfloat16
H, I = 128, 96


def _inputs(M, dt):
    g = torch.Generator()
    g.manual_seed(M)
    r = lambda *s: torch.randn(s, generator=g).to(dt).cuda()
    return r(M, H), r(I, H) / 8, r(I, H) / 8, r(H, I) / 8, r(M, H)


def _pass(x, wg, wu, wd, dy, L):
    import _native
    y, g, u = _native.ffn_forward(x, wg, wu, wd, act_limit=L, save=True)
    return (y,) + tuple(_native.ffn_backward(dy, x, g, u, wg, wu, wd, act_limit=L))


def _same(a, b):
    return torch.equal(a, b) and bool(torch.isfinite(a).all())


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("L", [0.0, 0.5, 10.0])
@pytest.mark.parametrize("M", [1, 2, 8, 20, 200])
def test_a_token_that_is_not_finite(gpu, M, L, dt):
    """NaN, and an infinity (g is then -inf in some channels, whose silu is not a number), in one token: its output and dx
    are NaN, the other tokens' as without it, and the weights' gradients, sums over the tokens, are NaN."""
    x, wg, wu, wd, dy = _inputs(M, dt)
    clean = _pass(x, wg, wu, wd, dy, L)
    rest = torch.arange(M, device="cuda") != M // 2
    for bad in (math.nan, math.inf, -math.inf):
        t = x.clone()
        t[M // 2, 5] = bad
        print("not finite", M, L, dt, bad, flush=True)
        y, dx, dwg, dwu, dwd = _pass(t, wg, wu, wd, dy, L)
        assert bool(y[M // 2].isnan().all()) and _same(y[rest], clean[0][rest])
        assert bool(dx[M // 2].isnan().all()) and _same(dx[rest], clean[1][rest])
        if bad != bad:
            assert all(bool(t.isnan().all()) for t in (dwg, dwu, dwd))
        else:
            # channels whose g is -inf: dWu and dWd through silu(g) = NaN (dWg's column 5, an infinite x, too)
            low = (t[M // 2].float() @ wg.float().t()) == -math.inf
            assert bool(low.any()) and bool(dwu[low].isnan().all()) and bool(dwd[:, low].isnan().all())


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("L", [0.0, 0.5, 10.0])
@pytest.mark.parametrize("M", [1, 8, 200])
@pytest.mark.parametrize("which", ["gate", "up"])
def test_a_weight_that_is_not_a_number(gpu, which, M, L, dt):
    """A NaN in one channel of gate or up: every output, and the gradients that the channel's h or dg carries."""
    x, wg, wu, wd, dy = _inputs(M, dt)
    (wg if which == "gate" else wu)[7, 3] = math.nan
    print("weight", which, M, L, dt, flush=True)
    y, dx, dwg, dwu, dwd = _pass(x, wg, wu, wd, dy, L)
    assert bool(y.isnan().all()) and bool(dx.isnan().all())
    assert bool(dwg[7].isnan().all()) and bool(dwd[:, 7].isnan().all())
    if which == "gate":
        assert bool(dwu[7].isnan().all())
    other = torch.arange(I, device="cuda") != 7
    assert all(bool(torch.isfinite(t).all()) for t in (dwg[other], dwu[other], dwd[:, other]))


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M", [1, 8, 200])
def test_infinite_gates_are_clamped(gpu, M, dt):
    """silu(+inf) and u = +-inf under a clamp are L and +-L: finite outputs; no gradient passes."""
    import _native
    L = 2.0
    x, wg, wu, wd, dy = _inputs(M, dt)
    x[:, 0] = 1.0
    wg[4, 0], wu[5, 0], wu[6, 0] = math.inf, math.inf, -math.inf
    print("clamped", M, dt, flush=True)
    y, g, u = _native.ffn_forward(x, wg, wu, wd, act_limit=L, save=True)
    assert bool((g[:, 4] == math.inf).all()) and bool((u[:, 5] == math.inf).all()) and bool((u[:, 6] == -math.inf).all())
    big = [w.clone() for w in (wg, wu)]
    big[0][4, 0], big[1][5, 0], big[1][6, 0] = 1e4, 1e4, -1e4
    z = _native.ffn_forward(x, *big, wd, act_limit=L)
    assert _same(y, z)
    _, dwg, dwu, dwd = _native.ffn_backward(dy, x, g, u, wg, wu, wd, act_limit=L, need=(False, True, True, True))
    assert bool((dwg[4] == 0).all()) and bool((dwu[5:7] == 0).all()) and bool(torch.isfinite(dwd).all())
