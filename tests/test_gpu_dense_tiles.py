"""The dense operators' largest tiles (256 x 256) in every product: sizes that gm_plan gives them (test_gemm_plan.py checks
that), K steps and columns that do not fill the last tile. Some tokens' outputs, and the gradients of some of the I
channels, against the 64-bit definition over those tokens and those channels."""
import math

import pytest

import dense_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

# (M, H, I): every product of a training pass in large tiles; the columns of gate|up and of down's gradient in two launches.
# Rows in whole chunks of 16 bytes; of 8; of 4 bytes.
ALL = (1934, 4104, 5128)
RAGGED = [(1934, 4100, 5124), (1935, 4098, 5130)]
# a product of those whose last columns take a launch of their own, its K steps not whole either
REST = {"dh": (4014, 2056, 5128), "dwg_dwu": (4014, 2056, 5128), "dx": (4014, 4104, 4104)}
# (M, N, K) of an 8-bit product; of these the last two in two launches
I8 = [(2050, 6168, 1304), (2050, 6170, 1301), (4014, 6018, 2440), (4014, 6024, 2440)]


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


@pytest.mark.parametrize("L", [0.0, 0.75])
@pytest.mark.parametrize("M,H,I,dt", [RAGGED[0] + (BF16,), RAGGED[1] + (F16,)])
def test_every_product_in_large_tiles_of_ragged_rows(gpu, M, H, I, dt, L):
    _pass(M, H, I, dt, L, 12)


@pytest.mark.parametrize("M,H,I,dt", [REST["dh"] + (BF16,), REST["dx"] + (F16,)])
def test_last_columns_in_a_launch_of_their_own(gpu, M, H, I, dt):
    _pass(M, H, I, dt, 0.75, 13)


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("M,N,K", I8)
def test_gemm_i8_in_large_tiles(gpu, M, N, K, dt):
    """Rows of a wider buffer with a stride of a multiple of 4 bytes, so that K may end inside a word."""
    import _native
    g = torch.Generator()
    g.manual_seed(M + N + K)
    ld = (K + 3) // 4 * 4

    def rows(n):
        wide = torch.full((n, ld), 99, dtype=torch.int8)
        wide[:, :K] = torch.randint(-127, 128, (n, K), generator=g, dtype=torch.int8)
        return wide.cuda()[:, :K]
    a, b = rows(M), rows(N)
    sa, sb = (((torch.rand(n, generator=g) + 0.5) / 127).cuda() for n in (M, N))
    sa = sa / K
    print("gemm_i8_tiles", M, N, K, dt, flush=True)
    out = _native.gemm_i8(a, sa, b, sb, dtype=dt)
    assert torch.equal(out, _native.gemm_i8(a, sa, b, sb, dtype=dt))
    at = torch.tensor(list(range(0, M, 97)) + [M - 1], device="cuda")
    want = a[at].double().cpu() @ b.double().cpu().t() * sa[at].double().cpu()[:, None] * sb.double().cpu()
    R.within(out[at], want, want.abs() * (R.half_step(dt) + 4 * 2.0 ** -24) + R.tiny(dt), "out")
