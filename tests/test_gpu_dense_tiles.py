"""The dense operators' largest tiles (256 x 256) in every product: sizes that gm_plan gives them (test_gemm_plan.py checks
that), K steps and columns that do not fill the last tile. Some tokens' outputs, and the gradients of some of the I
channels, against the 64-bit definition over those tokens and those channels."""
import math

import pytest

import dense_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

# (M, H, I): every product of a training pass in large tiles; the columns of gate|up and of down's gradient in two launches
ALL = (1934, 4104, 5128)


def _pass(M, H, I, dt, L, seed):
    import _native
    g = torch.Generator()
    g.manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    x, dy = r(M, H).to(dt).cuda(), r(M, H).to(dt).cuda()
    wg, wu = ((r(I, H) * 1.5 / math.sqrt(H)).to(dt).cuda() for _ in range(2))
    wd = (r(H, I) / math.sqrt(I)).to(dt).cuda()
    print("ffn_tiles", M, H, I, dt, L, flush=True)
    y, gate, up = _native.ffn_forward(x, wg, wu, wd, act_limit=L, save=True)
    assert torch.equal(y, _native.ffn_forward(x, wg, wu, wd, act_limit=L))
    dx, dwg, dwu, dwd = _native.ffn_backward(dy, x, gate, up, wg, wu, wd, act_limit=L)
    for again, first in zip(_native.ffn_backward(dy, x, gate, up, wg, wu, wd, act_limit=L), (dx, dwg, dwu, dwd)):
        assert torch.equal(again, first)
    rows = torch.tensor(list(range(0, M, 97)) + [M - 1], device="cuda")
    ref = R.FFN(x[rows], wg, wu, wd, L)
    R.within(y[rows], ref.y, ref.ey, "y")
    R.within(dx[rows], *ref.backward(dy[rows])[0], "dx")
    ch = torch.tensor(list(range(0, I, 61)) + [I - 1], device="cuda")
    ref = R.FFN(x, wg[ch], wu[ch], wd[:, ch], L)
    for n, a, (v, e) in zip(("dwg", "dwu", "dwd"), (dwg[ch], dwu[ch], dwd[:, ch]), ref.backward(dy)[1:]):
        R.within(a, v, e, n)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("L", [0.0, 0.75])
def test_every_product_in_large_tiles(gpu, dt, L):
    _pass(*ALL, dt, L, 11)
