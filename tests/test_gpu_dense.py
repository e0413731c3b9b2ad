"""The dense operators on the GPU (gfl_ffn_*, gfl_quant_i8 / gfl_gemm_i8 / gfl_linear_i8, gfl_sample) against their 64-bit
definitions, every output within the bound that dense_ref derives from the roundings."""
import math

import numpy as np
import pytest

import dense_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _rng(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _ffn_inputs(M, H, I, dt, seed, wide=1.0, pad=0):
    g = _rng(seed)
    r = lambda *s: torch.randn(s, generator=g)
    x = r(M, H)
    if pad:
        buf = torch.full((M, H + 2 * pad), float("nan"))
        buf[:, pad:pad + H] = x
        x = buf.to(dt).cuda()[:, pad:pad + H]
    else:
        x = x.to(dt).cuda()
    return (x, (r(I, H) * wide / math.sqrt(H)).to(dt).cuda(), (r(I, H) * wide / math.sqrt(H)).to(dt).cuda(),
            (r(H, I) / math.sqrt(I)).to(dt).cuda(), r(M, H).to(dt).cuda())


# (M, H, I): one token to many, whole tiles, ragged ones, sizes that no vector load fits
SHAPES = [(1, 256, 256), (1, 1024, 384), (3, 512, 136), (16, 640, 264), (17, 256, 512), (64, 384, 200), (65, 264, 328),
          (129, 512, 392), (300, 520, 1032), (1, 5120, 1536), (2, 131, 77), (19, 101, 257), (140, 259, 333), (1, 1, 1),
          (5, 7, 9), (513, 64, 72), (8, 1536, 520)]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M,H,I", SHAPES)
def test_ffn_forward(gpu, M, H, I, dt):
    import _native
    x, wg, wu, wd, _ = _ffn_inputs(M, H, I, dt, M * 31 + H + I)
    ref = R.FFN(x, wg, wu, wd)
    print("ffn_forward", M, H, I, dt, flush=True)
    R.within(_native.ffn_forward(x, wg, wu, wd), ref.y, ref.ey, "y")


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("L", [0.0, 0.75])
@pytest.mark.parametrize("M,H,I", [(1, 512, 256), (7, 256, 264), (33, 136, 512), (66, 384, 520), (200, 264, 136),
                                   (3, 77, 131), (70, 129, 255)])
def test_ffn_training_pass(gpu, M, H, I, L, dt):
    import _native
    x, wg, wu, wd, dy = _ffn_inputs(M, H, I, dt, M + H + I, wide=1.5)
    ref = R.FFN(x, wg, wu, wd, L)
    print("ffn_training", M, H, I, L, dt, flush=True)
    y, g, u = _native.ffn_forward(x, wg, wu, wd, act_limit=L, save=True)
    R.within(y, ref.y, ref.ey, "y")
    assert torch.equal(y, _native.ffn_forward(x, wg, wu, wd, act_limit=L))
    got = _native.ffn_backward(dy, x, g, u, wg, wu, wd, act_limit=L)
    for n, a, (v, e) in zip(("dx", "dwg", "dwu", "dwd"), got, ref.backward(dy)):
        R.within(a, v, e, n)


def test_ffn_large_tiles(gpu):
    """The largest tiles (256 x 256), forward and gradients."""
    import _native
    M, H, I = 2050, 2304, 2056
    for dt in (F16, BF16):
        x, wg, wu, wd, dy = _ffn_inputs(M, H, I, dt, 5)
        ref = R.FFN(x, wg, wu, wd)
        print("ffn_large", dt, flush=True)
        y, g, u = _native.ffn_forward(x, wg, wu, wd, save=True)
        R.within(y, ref.y, ref.ey, "y")
        for n, a, (v, e) in zip(("dx", "dwg", "dwu", "dwd"), _native.ffn_backward(dy, x, g, u, wg, wu, wd),
                                ref.backward(dy)):
            R.within(a, v, e, n)


def _part_of_a_pass(M, H, I, dt):
    import _native
    x, wg, wu, wd, dy = _ffn_inputs(M, H, I, dt, M + I)
    print("ffn_part", M, H, I, dt, flush=True)
    y, g, u = _native.ffn_forward(x, wg, wu, wd, save=True)
    dx, dwg, dwu, dwd = _native.ffn_backward(dy, x, g, u, wg, wu, wd)
    rows = torch.tensor(list(range(0, M, 97)) + [M - 1], device="cuda")
    ref = R.FFN(x[rows], wg, wu, wd)
    R.within(y[rows], ref.y, ref.ey, "y")
    R.within(dx[rows], *ref.backward(dy[rows])[0], "dx")
    ch = torch.tensor(list(range(0, I, 61)) + [I - 1], device="cuda")
    ref = R.FFN(x, wg[ch], wu[ch], wd[:, ch])
    for n, a, (v, e) in zip(("dwg", "dwu", "dwd"), (dwg[ch], dwu[ch], dwd[:, ch]), ref.backward(dy)[1:]):
        R.within(a, v, e, n)


@pytest.mark.parametrize("M,H,I,dt", [(1934, 1280, 6144, F16), (4014, 6144, 1280, BF16), (4014, 1280, 6144, F16),
                                      (1154, 6144, 2048, BF16), (1154, 4096, 6144, F16)])
def test_ffn_products_in_two_launches(gpu, M, H, I, dt):
    """Sizes at which one of the products (gate|up; down and dx; dh; the gradients of gate and up; of down) takes a launch of
    large tiles and another for its last columns. Some tokens' outputs, and the gradients of some of the I channels, against
    the definition over those tokens and those channels."""
    _part_of_a_pass(M, H, I, dt)


def test_ffn_large_tiles_with_rows_that_end_inside_a_chunk(gpu):
    """Whole K steps (2048 tokens) of rows of 2050 and 2308: the last row's last chunk reaches past the matrix."""
    _part_of_a_pass(2048, 2050, 2308, BF16)


@pytest.mark.parametrize("pad", [8, 32, 3])
def test_ffn_strided_rows_and_outputs(gpu, pad):
    """Rows of a wider buffer (NaN around them), an out of wider rows whose surroundings stay as they were, fp32 out, and
    out += block."""
    import _native
    M, H, I = 37, 264, 392
    x, wg, wu, wd, dy = _ffn_inputs(M, H, I, F16, pad, pad=pad)
    ref = R.FFN(x, wg, wu, wd)
    buf = torch.full((M + 2, H + pad), 7.0, dtype=F16, device="cuda")
    out = buf[1:1 + M, :H]
    print("ffn_strided", pad, flush=True)
    _native.ffn_forward(x, wg, wu, wd, out=out)
    R.within(out, ref.y, ref.ey, "y")
    assert bool((buf[0] == 7).all() and (buf[-1] == 7).all() and (buf[:, H:] == 7).all())
    ref32 = R.FFN(x, wg, wu, wd, out_dt=F32)
    o32 = _native.ffn_forward(x, wg, wu, wd, out=torch.empty((M, H), dtype=F32, device="cuda"))
    R.within(o32, ref32.y, ref32.ey, "fp32 out")
    base = torch.randn((M, H), device="cuda")
    acc = base.clone()
    _native.ffn_forward(x, wg, wu, wd, out=acc, accumulate=True)
    assert torch.equal(acc, base + o32)
    y, g, u = _native.ffn_forward(x, wg, wu, wd, save=True)
    wide_dy = torch.full((M, H + pad), float("nan"), dtype=F16, device="cuda")
    wide_dy[:, :H] = dy
    a = _native.ffn_backward(wide_dy[:, :H], x, g, u, wg, wu, wd)
    for n, t, (v, e) in zip(("dx", "dwg", "dwu", "dwd"), a, ref.backward(dy)):
        R.within(t, v, e, n)


@pytest.mark.parametrize("ld", [(1 << 22) - 8, (1 << 22) - 1])
def test_ffn_widest_strides(gpu, ld):
    """Rows as far apart as allowed: offsets within a tile near 2^31 bytes, within the tensors past it."""
    import _native
    M, H, I = 300, 136, 72
    x, wg, wu, wd, dy = _ffn_inputs(M, H, I, F16, 12)

    def spread(t):
        out = torch.zeros((M, ld), dtype=F16, device="cuda")[:, :H]
        return out if t is None else out.copy_(t)

    print("ffn_widest", ld, flush=True)
    y, g, u = _native.ffn_forward(x, wg, wu, wd, save=True)
    xs, dys = spread(x), spread(dy)
    ys, gs, us = _native.ffn_forward(xs, wg, wu, wd, out=spread(None), save=True)
    ref = R.FFN(x, wg, wu, wd)
    R.within(ys, ref.y, ref.ey, "y")
    for n, a, (v, e) in zip(("dx", "dwg", "dwu", "dwd"), _native.ffn_backward(dys, xs, gs, us, wg, wu, wd), ref.backward(dy)):
        R.within(a, v, e, n)
    R.within(_native.ffn_forward(xs[:5], wg, wu, wd), ref.y[:5], ref.ey[:5], "y of 5")
    R.within(_native.ffn_forward(xs[298:], wg, wu, wd), ref.y[298:], ref.ey[298:], "y of 2")


@pytest.mark.parametrize("ld", [(1 << 22) - 16, (1 << 22) - 1])
def test_gemm_i8_widest_strides(gpu, ld):
    import _native
    a, sa, b, sb = _i8(600, 520, 144, 4)
    want, bound, _ = _i8_ref(a, sa, b, sb, F32)
    far = [torch.zeros((len(t), ld), dtype=torch.int8, device="cuda")[:, :144].copy_(t) for t in (a, b)]
    print("gemm_i8_widest", ld, flush=True)
    R.within(_native.gemm_i8(far[0], sa, far[1], sb, dtype=F32), want, bound)
    for m in (1, 9):
        R.within(_native.gemm_i8(far[0][-m:], sa[-m:], far[1], sb, dtype=F32), want[-m:], bound[-m:])


def test_ffn_partial_gradients_and_empty(gpu):
    import _native
    M, H, I = 21, 128, 96
    x, wg, wu, wd, dy = _ffn_inputs(M, H, I, BF16, 3)
    _, g, u = _native.ffn_forward(x, wg, wu, wd, save=True)
    full = _native.ffn_backward(dy, x, g, u, wg, wu, wd)
    for mask in range(16):
        need = [bool(mask >> i & 1) for i in range(4)]
        part = _native.ffn_backward(dy, x, g, u, wg, wu, wd, need=need)
        for f, p, n in zip(full, part, need):
            assert (p is None) == (not n) and (p is None or torch.equal(p, f))
    y, g, u = _native.ffn_forward(x[:0], wg, wu, wd, save=True)
    assert y.shape == (0, H) and g.shape == (0, I)
    dx, *dw = _native.ffn_backward(dy[:0], x[:0], g, u, wg, wu, wd)
    assert dx.shape == (0, H) and all(bool((t == 0).all()) for t in dw)
    assert _native.ffn_forward(x.view(3, 7, H), wg, wu, wd).shape == (3, 7, H)


def test_ffn_gradients_against_differences(gpu):
    """sum(y * dy) differentiated along a random direction of each input, by the definition in 64 bits at the inputs the
    device saw: the gradients' inner product with the direction."""
    import _native
    M, H, I = 9, 96, 64
    x, wg, wu, wd, dy = _ffn_inputs(M, H, I, F16, 11)
    _, g, u = _native.ffn_forward(x, wg, wu, wd, save=True)
    grads = [t.double().cpu() for t in _native.ffn_backward(dy, x, g, u, wg, wu, wd)]
    ins = [t.double().cpu() for t in (x, wg, wu, wd)]
    d = dy.double().cpu()
    ref = R.FFN(x, wg, wu, wd)
    bounds = [e for _, e in ref.backward(dy)]

    def value(ts):
        a, b, c, e = ts
        gg, uu = a @ b.t(), a @ c.t()
        return float(((gg * torch.sigmoid(gg) * uu) @ e.t() * d).sum())

    for i in range(4):
        v = torch.randn(ins[i].shape, generator=_rng(50 + i), dtype=torch.float64)
        h = 1e-5
        up, dn = list(ins), list(ins)
        up[i], dn[i] = ins[i] + h * v, ins[i] - h * v
        num = (value(up) - value(dn)) / (2 * h)
        # the central difference is off by h^2/6 of the third derivative, far below the roundings' share
        assert abs(float((grads[i] * v).sum()) - num) <= float((bounds[i] * v.abs()).sum()) + 1e-4


def test_ffn_not_finite(gpu):
    """An infinite or NaN token spoils its own row only."""
    import _native
    M, H, I = 20, 128, 96
    x, wg, wu, wd, _ = _ffn_inputs(M, H, I, BF16, 4)
    clean = _native.ffn_forward(x, wg, wu, wd)
    x[3, 5], x[11, 0] = float("nan"), float("inf")
    y = _native.ffn_forward(x, wg, wu, wd)
    rows = [i for i in range(M) if i not in (3, 11)]
    assert torch.equal(y[rows], clean[rows]) and bool(torch.isnan(y[3]).all()) and not bool(torch.isfinite(y[11]).any())


# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M,K,pad", [(1, 128, 0), (5, 5120, 0), (33, 4104, 8), (7, 131, 0), (2, 9001, 3), (1, 1, 0)])
def test_quant_i8(gpu, M, K, pad, dt):
    import _native
    g = _rng(M + K)
    x = torch.full((M, K + pad), float("nan"), dtype=dt, device="cuda")[:, :K]
    # whole numbers over small powers of two: many quotients fall on a half
    x.copy_((torch.randint(-256, 257, (M, K), generator=g) / 16.0 * torch.exp2(torch.randint(-3, 4, (M, 1), generator=g))))
    if M > 4:
        x[1] = 0
    q, s = _native.quant_i8(x)
    wq, ws = R.quant(x)
    assert torch.equal(q.double().cpu(), wq)
    R.within(s, ws, ws * 2.0 ** -24 + 2.0 ** -150)


def test_quant_i8_range_and_not_finite(gpu):
    import _native
    for dt in (F16, BF16):
        big = torch.finfo(dt).max
        x = torch.randn((6, 300), generator=_rng(1)).to(dt).cuda()
        x[0, 7] = big
        x[1] = torch.where(torch.arange(300) % 2 == 0, big, -big).to(dt).cuda()
        x[2, 3], x[3, 4], x[4, 5] = float("inf"), float("nan"), float("-inf")
        q, s = _native.quant_i8(x)
        wq, ws = R.quant(x[[0, 1, 5]])
        assert torch.equal(q[[0, 1, 5]].double().cpu(), wq)
        R.within(s[[0, 1, 5]], ws, ws * 2.0 ** -24)
        assert bool((q[2:5] == 0).all()) and not bool(torch.isfinite(s[2:5]).any())
        w = torch.randint(-127, 128, (32, 300), generator=_rng(2), dtype=torch.int8).cuda()
        y = _native.linear_i8(x, w, torch.ones(32, device="cuda"), dtype=F32)
        assert bool(torch.isnan(y[2:5]).all())
        # row 0 of bf16: the largest bf16 times a weight of up to 127 lies past fp32's range, as the definition's value does
        want = wq[[0, 2]] @ w.double().cpu().t() * ws[[0, 2]][:, None]
        fits = want.abs() < torch.finfo(F32).max * (1 - 2.0 ** -20)
        past = want.abs() > torch.finfo(F32).max * (1 + 2.0 ** -20)
        got = y[[0, 5]].double().cpu()
        assert bool(fits[1].all()) and bool(((got - want).abs() <= want.abs() * 5 * 2.0 ** -24)[fits].all())
        assert torch.equal(got[past], torch.sign(want[past]) * math.inf)


def _i8(M, N, K, seed, extreme=False):
    g = _rng(seed)
    r = lambda *s: torch.randint(-128, 128, s, generator=g, dtype=torch.int8).cuda()
    a, b = r(M, K), r(N, K)
    if extreme:
        a.fill_(-128)
        b.fill_(-128)
    sa, sb = (torch.rand(n, generator=g).cuda() + 0.1 for n in (M, N))
    return a, sa, b, sb


def _i8_ref(a, sa, b, sb, dt):
    acc = a.double().cpu() @ b.double().cpu().t()
    want = acc * sa.double().cpu()[:, None] * sb.double().cpu()[None, :]
    lim = torch.finfo(dt).max
    return want, want.abs() * (R.half_step(dt) + 4 * 2.0 ** -24) + R.tiny(dt), lim


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("M,N,K", [(1, 256, 512), (1, 5120, 1024), (4, 1000, 136), (16, 264, 2048), (17, 129, 4096), (64, 96, 1040),
                                   (65, 640, 272), (300, 392, 528), (2, 77, 131), (20, 33, 65), (150, 261, 1001), (1, 1, 1),
                                   (9, 65, 8192), (700, 1300, 64)])
def test_gemm_i8(gpu, M, N, K, dt):
    import _native
    a, sa, b, sb = _i8(M, N, K, M + N + K)
    sa = sa / K      # products within fp16's range
    want, bound, lim = _i8_ref(a, sa, b, sb, dt)
    assert float(want.abs().max()) < lim
    print("gemm_i8", M, N, K, dt, flush=True)
    R.within(_native.gemm_i8(a, sa, b, sb, dtype=dt), want, bound)


def test_gemm_i8_sums_past_2_31(gpu):
    """-128 * -128 over the longest K: the sum fills the int32."""
    import _native
    a, sa, b, sb = _i8(3, 40, 131071, 1, extreme=True)
    want, bound, _ = _i8_ref(a, sa, b, sb, F32)
    assert float((a.double().cpu() @ b.double().cpu().t()).max()) == 131071 * 16384
    R.within(_native.gemm_i8(a, sa, b, sb, dtype=F32), want, bound)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_gemm_i8_in_two_launches(gpu, dt):
    import _native
    a, sa, b, sb = _i8(4014, 6144, 2432, 10)
    rows = torch.tensor(list(range(0, 4014, 97)) + [4013], device="cuda")
    want, bound, _ = _i8_ref(a[rows], sa[rows], b, sb, dt)
    R.within(_native.gemm_i8(a, sa, b, sb, dtype=dt)[rows], want, bound)


def test_gemm_i8_large_tiles_and_strides(gpu):
    import _native
    M, N, K = 2100, 2304, 1040
    a, sa, b, sb = _i8(M, N, K, 9)
    want, bound, _ = _i8_ref(a, sa, b, sb, BF16)
    R.within(_native.gemm_i8(a, sa, b, sb, dtype=BF16), want, bound)
    wide = torch.full((M, K + 48), 99, dtype=torch.int8, device="cuda")
    wide[:, 16:16 + K] = a
    out = torch.full((M, N + 3), 5.0, dtype=BF16, device="cuda")
    _native.gemm_i8(wide[:, 16:16 + K], sa, b, sb, out=out[:, :N])
    R.within(out[:, :N], want, bound)
    assert bool((out[:, N:] == 5).all())


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M,N,K", [(1, 512, 640), (3, 200, 333), (40, 256, 1024)])
def test_linear_i8(gpu, M, N, K, dt):
    import _native
    _, _, b, sb = _i8(1, N, K, 3)
    x = torch.randn((M, K), generator=_rng(M)).to(dt).cuda()
    q, s = _native.quant_i8(x)
    sb = sb / K
    got = _native.linear_i8(x, b, sb)
    assert got.dtype == dt and torch.equal(got, _native.gemm_i8(q, s, b, sb, dtype=dt))
    wq, ws = R.quant(x)
    want = wq @ b.double().cpu().t() * ws[:, None] * sb.double().cpu()
    # one more rounding than the product alone: the scale's
    R.within(got, want, want.abs() * (R.half_step(dt) + 5 * 2.0 ** -24) + R.tiny(dt))


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M,N,K,pad", [(1, 1, 8, 0), (2, 7, 1000, 8), (1, 513, 5120, 0), (2, 20011, 264, 0), (1, 40, 8192, 0),
                                       (2, 33, 8192, 24), (1, 24, 8200, 0), (2, 24, 520, 4), (1, 17, 4096, 0), (2, 9, 1032, 1)])
def test_linear_i8_few_tokens(gpu, M, N, K, pad, dt):
    """One and two tokens, whichever launches they take: the same bits as the rows quantised by a call of their own; rows
    of zeros and rows that are not finite too."""
    import _native
    _, _, b, sb = _i8(1, N, K, 5)
    x = torch.randn((M, K + pad), generator=_rng(K + N)).to(dt).cuda()[:, :K]
    for k in range(4):
        if k == 1:
            x[M - 1] = 0
        elif k == 2:
            x[0, K // 2] = math.inf
        elif k == 3:
            x[0, K // 2] = math.nan
        q, s = _native.quant_i8(x)
        for out in (dt, F32):
            got, want = _native.linear_i8(x, b, sb, dtype=out), _native.gemm_i8(q, s, b, sb, dtype=out)
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
            assert bool(got[0].isnan().all()) == (k >= 2)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M,N,K,pad", [(1, 33, 1032, 0), (2, 33, 5000, 8), (1, 16385, 1024, 0), (2, 20011, 1272, 0), (2, 16384, 2056, 0),
                                       (1, 40000, 1024, 0)])
def test_linear_i8_few_tokens_in_one_launch(gpu, M, N, K, pad, dt):
    """Sizes that the launch of both takes (K from 1024 to 8192 in whole chunks): rows that end inside their last KB, and more
    columns than its workgroups take at once (16,384)."""
    test_linear_i8_few_tokens(gpu, M, N, K, pad, dt)


# ---------------------------------------------------------------------------------------------------------------

def _draw(logits, u, **kw):
    import _native
    dev = lambda t, dt: None if t is None else torch.as_tensor(t, dtype=dt).cuda()
    return _native.sample(logits.cuda(), dev(u, F32), temperature=dev(kw.get("temperature"), F32),
                          top_k=dev(kw.get("top_k"), torch.int32), top_p=dev(kw.get("top_p"), F32),
                          min_p=dev(kw.get("min_p"), F32))


def _check_draw(logits, u, skip=0, **kw):
    """Tokens as the definition has them. Rows whose border lies within 2^-36 of a compared value (V units of 2^-43 and
    fp64's own roundings) may fall on either side: at most `skip` of them."""
    V = logits.shape[1]
    f = lambda t: None if t is None else torch.as_tensor(t, dtype=F32)
    args = {k: (v if k == "top_k" else f(v)) for k, v in kw.items()}
    want = R.sample(logits, f(u), **args)
    tok, prob = _draw(logits, u, **kw)
    tok, prob = tok.cpu().tolist(), prob.double().cpu().tolist()
    near = [b for b, (_, _, m) in enumerate(want) if m < 2.0 ** -36]
    assert len(near) <= skip, near
    for b, (t, p, _) in enumerate(want):
        if b in near:
            continue
        assert tok[b] == t, (b, tok[b], t)
        assert abs(prob[b] - p) <= p * 2.0 ** -23 + V * 2.0 ** -42, (b, prob[b], p)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 63), (4, 1000), (7, 4097), (40, 32003), (2, 131072), (1, 200001)])
def test_sample_mixed(gpu, B, V, dt):
    g = _rng(B * V)
    r = lambda: torch.rand(B, generator=g)
    logits = (torch.randn((B, V), generator=g) * 3).to(dt)
    k = (torch.exp(r() * math.log(300.0))).int()
    k[r() < 0.3] = 0
    p, m, t = 0.5 + 0.5 * r(), 0.2 * r(), 0.3 + 1.5 * r()
    p[r() < 0.3], m[r() < 0.3], t[r() < 0.1] = 1.0, 0.0, 0.0
    _check_draw(logits, r(), temperature=t, top_k=k, top_p=p, min_p=m)
    _check_draw(logits, r())
    _check_draw(logits, r(), top_k=k)
    _check_draw(logits, r(), top_p=p, temperature=t)
    _check_draw(logits, r(), min_p=m)


@pytest.mark.parametrize("V", [500, 70000])
def test_sample_masks(gpu, V):
    """-inf and NaN places are never drawn, rows left empty give -1, +inf wins."""
    g = _rng(V)
    x = torch.randn((9, V), generator=g) * 2
    x[torch.rand((9, V), generator=g) < 0.7] = -math.inf
    x[1] = -math.inf
    x[2] = math.nan
    x[3, ::2] = math.nan
    x[4] = -math.inf
    x[4, V - 1] = -3.0
    x[5, 10], x[5, V // 2] = math.inf, math.inf
    x[6] = torch.finfo(F32).min
    x[7, 3] = torch.finfo(F32).max
    kw = dict(temperature=[0.8] * 9, top_k=[50] * 9, top_p=[0.9] * 9, min_p=[0.01] * 9)
    for u in (0.0, 0.37, 0.99999):
        for args in ({}, kw, dict(kw, top_k=[0] * 9), dict(temperature=[0.0] * 9)):
            _check_draw(x, [u] * 9, **args)
    tok, prob = _draw(x, [0.5] * 9)
    assert tok.tolist()[1:3] == [-1, -1] and prob.tolist()[1:3] == [0.0, 0.0]


@pytest.mark.parametrize("V", [700, 2930])
def test_sample_rows_with_few_or_no_logits_left(gpu, V):
    """A mask that leaves a row 0 to 5 logits or so, each row's own settings."""
    g = _rng(V + 1)
    B = 90
    r = lambda: torch.rand(B, generator=g)
    x = torch.randn((B, V), generator=g) * 3
    x[torch.rand((B, V), generator=g) < 1 - 2.0 / V] = -math.inf
    k = (torch.exp(r() * math.log(300.0))).int()
    k[r() < 0.3] = 0
    left = (x > -math.inf).sum(1)
    assert int(left.min()) == 0 and int(left.max()) > 2
    _check_draw(x, r(), temperature=0.5 + r(), top_k=k, top_p=0.6 + 0.4 * r(), min_p=0.1 * r())
    _check_draw(x, r(), temperature=0.5 + r(), top_p=0.6 + 0.4 * r())
    _check_draw(x, r())


@pytest.mark.parametrize("V", [300, 66000])
def test_sample_ties(gpu, V):
    """Equal logits: the lowest indices are kept, -0 equals +0, u walks the kept ones in order."""
    x = torch.zeros((6, V))
    x[0, ::2] = -0.0
    x[1, 5::7] = 1.0
    x[2, 100:] = -1.0
    x[3, :] = -math.inf
    x[3, 17::13] = 2.5
    x[4, 200] = 3.0
    for u in (0.0, 0.11, 0.501, 0.9999):
        _check_draw(x, [u] * 6, top_k=[7] * 6)
        _check_draw(x, [u] * 6, top_p=[0.3001] * 6, skip=6)
        _check_draw(x, [u] * 6, top_k=[40] * 6, top_p=[0.5013] * 6)
        _check_draw(x, [u] * 6, min_p=[0.9] * 6)
        _check_draw(x, [u] * 6, min_p=[1.0] * 6)
        _check_draw(x, [u] * 6, min_p=[2.0] * 6, top_p=[0.6] * 6, skip=6)
    tok, _ = _draw(x, [0.0] * 6, temperature=[0.0] * 6)
    assert tok.tolist() == [0, 5, 0, 17, 200, 0]


def test_sample_extremes(gpu):
    g = _rng(8)
    x = torch.randn((8, 3000), generator=g) * 5
    u = torch.rand(8, generator=g)
    _check_draw(x, u, temperature=[1e-6] * 8)
    _check_draw(x, u, temperature=[1e6] * 8)
    _check_draw(x, u, temperature=[math.nan, -1.0, 0.0, 1e-30, 1.0, 2.0, 3.0, 100.0])
    _check_draw(x, u, top_k=[1, 2, 2999, 3000, 3001, -5, 0, 2 ** 31 - 1])
    _check_draw(x, u, top_p=[0.0, -1.0, 1e-9, 0.5, 0.999999, 1.0, 2.0, math.nan])
    _check_draw(x, u, min_p=[0.0, -1.0, 1e-9, 0.5, 0.999999, 1.0, 2.0, math.nan])
    # u outside [0, 1) takes the first or last kept token
    tok, _ = _draw(x, [-1.0, 0.0, 1.0, 5.0, math.nan, 0.0, 1.0, 0.0], top_k=[3] * 8)
    keep = torch.topk(x, 3).indices.sort(1).values
    assert tok.cpu().tolist() == [int(keep[b, c]) for b, c in enumerate((0, 0, 2, 2, 0, 0, 2, 0))]


@pytest.mark.parametrize("dt", [F32, BF16])
def test_sample_large_k_and_low_temperature(gpu, dt):
    """A top-k larger than a row's list, one that ends below where weights round to zero, temperatures from near greedy to flat,
    finite masks of the type's lowest value, logits that span the type's range."""
    g = _rng(17)
    V = 70000
    x = (torch.randn((6, V), generator=g) * 2.5).to(dt)
    x[2, torch.rand(V, generator=g) < 0.9] = torch.finfo(dt).min
    x[3] = (torch.rand(V, generator=g) * 2 - 1).to(dt) * (torch.finfo(dt).max / 2)
    x[4, 1000:] = -math.inf
    u = torch.rand(6, generator=g)
    for t in (0.02, 0.7, 50.0, math.inf):
        for k in (3, 900, 1500, 5000, 69999):
            _check_draw(x, u, temperature=[t] * 6, top_k=[k] * 6, skip=1)
            _check_draw(x, u, temperature=[t] * 6, top_k=[k] * 6, top_p=[0.93] * 6, min_p=[1e-4] * 6, skip=1)
        _check_draw(x, u, temperature=[t] * 6, top_p=[0.8] * 6, skip=1)
        _check_draw(x, u, temperature=[t] * 6, top_p=[0.999] * 6, min_p=[0.02] * 6, skip=1)
        _check_draw(x, u, temperature=[t] * 6, min_p=[0.02] * 6, skip=1)


def test_sample_many_rows(gpu):
    """More rows than one round of launches takes: each row's token as the same rows give a round of their own."""
    import _native
    g = _rng(23)
    B, V = 2500, 700
    x = (torch.randn((B, V), generator=g) * 3).cuda()
    u, p = torch.rand(B, generator=g).cuda(), (0.5 + torch.rand(B, generator=g)).cuda()
    k = torch.randint(0, 60, (B,), generator=g, dtype=torch.int32).cuda()
    tok, prob = _native.sample(x, u, top_k=k, top_p=p)
    for lo, hi in ((0, 700), (700, 1500), (1500, 2500)):
        t, q = _native.sample(x[lo:hi], u[lo:hi], top_k=k[lo:hi], top_p=p[lo:hi])
        assert torch.equal(t, tok[lo:hi]) and torch.equal(q, prob[lo:hi])
    _check_draw(x[-40:].cpu(), u[-40:].cpu(), top_k=k[-40:].cpu(), top_p=p[-40:].cpu())


def test_sample_strided_rows(gpu):
    x = torch.randn((5, 1003), generator=_rng(2))
    buf = torch.full((5, 1100), 1e30, device="cuda")
    buf[:, 7:1010] = x.cuda()
    import _native
    u = torch.rand(5, generator=_rng(3)).cuda()
    a, b = _native.sample(buf[:, 7:1010], u), _native.sample(x.cuda(), u)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---------------------------------------------------------------------------------------------------------------

def test_dense_calls_in_a_graph(gpu):
    """A decode step's dense calls captured once and replayed on new inputs, with eager calls between the replays."""
    import _native
    M, H, I, V = 4, 512, 384, 5000
    x, wg, wu, wd, dy = _ffn_inputs(M, H, I, F16, 21)
    g = _rng(22)
    w = torch.randint(-127, 128, (V, H), generator=g, dtype=torch.int8).cuda()
    sw = (torch.rand(V, generator=g) / H).cuda()
    u, t, k = torch.rand(M, generator=g).cuda(), torch.full((M,), 0.7, device="cuda"), torch.full((M,), 40, dtype=torch.int32, device="cuda")
    p = torch.full((M,), 0.95, device="cuda")

    def step():
        y, gg, uu = _native.ffn_forward(x, wg, wu, wd, save=True)
        logits = _native.linear_i8(y, w, sw, dtype=F32)
        tok, prob = _native.sample(logits, u, temperature=t, top_k=k, top_p=p)
        return (y, logits, tok, prob) + tuple(_native.ffn_backward(dy, x, gg, uu, wg, wu, wd))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for r in range(4):
        x.copy_(torch.randn((M, H), generator=g).half())
        u.copy_(torch.rand(M, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_dense_calls_on_a_side_stream(gpu):
    """Calls on two streams at once do not share a workspace."""
    import _native
    a = _ffn_inputs(8, 1024, 768, BF16, 31)
    b = _ffn_inputs(8, 1024, 768, BF16, 32)
    wa, wb = _native.ffn_forward(*a[:4]), _native.ffn_forward(*b[:4])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        with torch.cuda.stream(side):
            gb = _native.ffn_forward(*b[:4])
        ga = _native.ffn_forward(*a[:4])
        torch.cuda.synchronize()
        assert torch.equal(ga, wa) and torch.equal(gb, wb)
