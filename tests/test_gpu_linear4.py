"""Products with 4-bit weights on the GPU (gfl_quant_i4, gfl_pack_i4, gfl_linear_i4, gfl_linear_i4_dx) against their 64-bit
definitions."""
import pytest

import serving_ref as S

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _weight(N, K, group, zeros, dt, seed):
    import _native
    g = _gen(seed)
    v = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    n = (K + group - 1) // group
    scale = ((torch.rand((n, N), generator=g) + 0.5) / 16).to(dt)
    zero = torch.randint(0, 16, (n, N), generator=g, dtype=torch.uint8) if zeros else None
    return v, _native.pack_i4(v.cuda()), scale.cuda(), zero.cuda() if zeros else None


def _tokens(M, K, dt, seed, whole=False, pad=0):
    g = _gen(seed)
    x = torch.randint(-8, 9, (M, K), generator=g).float() if whole else torch.randn((M, K), generator=g)
    buf = torch.full((M, K + pad), NAN)
    buf[:, pad // 2:pad // 2 + K] = x
    return buf.to(dt).cuda()[:, pad // 2:pad // 2 + K]


@pytest.mark.parametrize("N,K", [(1, 1), (3, 127), (5, 128), (16, 129), (7, 1000), (33, 640)])
def test_pack(gpu, N, K):
    v, q, _, _ = _weight(N, K, 32, False, F16, N + K)
    assert torch.equal(S.unpack(q, K), v.long())
    import _native
    wide = torch.full((N, K + 5), 255, dtype=torch.uint8, device="cuda")
    wide[:, :K] = v.cuda() | 0xA0          # the upper bits do not count
    assert torch.equal(_native.pack_i4(wide[:, :K]), q)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 1), (5, 300), (17, 128), (40, 1111)])
def test_quant(gpu, N, K, group, zeros, dt):
    import _native
    g = _gen(N + K + group)
    w = torch.randn((N, K), generator=g) * torch.exp2(torch.randint(-6, 3, (N, 1), generator=g).float())
    w[0, :40] = 0
    if N > 4:
        w[1, :128] = 0
        w[2] = w[2].abs() + 1            # 0 belongs to the range all the same
        w[3] = 2.0 ** -24                # fp16: scales that round to nothing
    w = w.to(dt)
    q, scale, zero = _native.quant_i4(w.cuda(), group=group, zeros=zeros)
    v, s, z = S.quant(w, group, zeros)
    assert torch.equal(S.unpack(q, K), v) and torch.equal(scale.cpu(), s)
    assert (zero is None) == (not zeros) and (zero is None or torch.equal(zero.cpu(), z))


def test_quant_not_finite(gpu):
    import _native
    for dt in (F16, BF16):
        w = torch.randn((4, 256), generator=_gen(2)).to(dt)
        w[0, 3], w[1, 200], w[2, 130] = INF, NAN, -INF
        w[3, 7] = torch.finfo(dt).max
        for zeros in (False, True):
            q, scale, zero = _native.quant_i4(w.cuda(), zeros=zeros)
            bad = torch.tensor([[True, False, False, False], [False, True, True, False]])
            assert torch.equal(torch.isnan(scale).cpu(), bad)
            v, s, _ = S.quant(torch.where(torch.isfinite(w), w, 0), 128, zeros)
            keep = ~bad.t().repeat_interleave(128, 1)
            assert torch.equal(S.unpack(q, 256)[keep], v[keep]) and bool((S.unpack(q, 256)[~keep] == 8).all())


SHAPES = [(1, 16, 128), (1, 5120, 1024), (2, 33, 640), (3, 1000, 4072), (5, 17, 129), (16, 264, 2048), (17, 129, 384), (31, 72, 1280),
          (48, 65, 2500), (64, 300, 520), (9, 1, 1), (1, 7, 9001), (33, 640, 100)]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("group,zeros", [(32, False), (32, True), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_few_tokens(gpu, M, N, K, group, zeros, dt):
    import _native
    _, q, scale, zero = _weight(N, K, group, zeros, dt, M + N + K)
    for whole, out_dt in ((True, F32), (False, dt)):
        x = _tokens(M, K, dt, N + K, whole)
        print("linear_i4", M, N, K, group, zeros, dt, out_dt, flush=True)
        got = _native.linear_i4(x, q, scale, zero=zero, group=group, dtype=out_dt)
        assert got.dtype == out_dt
        S.same(got, *S.linear(x, q, scale, zero, K, group, out_dt, True, whole), "y")


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("M,N,K", [(65, 129, 384), (200, 264, 1000), (300, 1000, 264), (513, 77, 131), (2050, 2304, 1040), (100, 40, 7)])
def test_many_tokens(gpu, M, N, K, group, zeros, dt):
    import _native
    _, q, scale, zero = _weight(N, K, group, zeros, dt, M + N + K)
    x = _tokens(M, K, dt, N)
    print("linear_i4", M, N, K, group, zeros, dt, flush=True)
    value, bound = S.linear(x, q, scale, zero, K, group, dt, False)     # either form, by sizes
    S.same(_native.linear_i4(x, q, scale, zero=zero, group=group), value,
           torch.maximum(bound, S.linear(x, q, scale, zero, K, group, dt, True)[1]), "y")
    x = _tokens(M, K, dt, N, True)
    got = _native.linear_i4(x, q, scale, zero=zero, group=group, dtype=F32)
    S.same(got, *S.linear(x, q, scale, zero, K, group, F32, True, True), "fp32 y")


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M,N,K,group,zeros", [(1, 128, 256, 128, False), (7, 264, 1000, 64, True), (20, 33, 131, 32, False),
                                               (70, 500, 264, 128, True), (300, 1032, 520, 32, True), (1030, 2048, 2056, 128, False),
                                               (3, 1, 1, 32, True), (1, 8, 300, 32, True), (16, 777, 384, 64, True), (24, 3001, 130, 128, True),
                                               (33, 9000, 264, 64, False), (130, 2048, 2056, 128, False), (260, 4104, 1030, 32, True),
                                               (400, 4096, 512, 128, False), (2, 9, 5, 128, False), (1, 7, 128, 64, True)])
def test_gradient(gpu, M, N, K, group, zeros, dt):
    import _native
    _, q, scale, zero = _weight(N, K, group, zeros, dt, M + N)
    dy = _tokens(M, N, dt, K, pad=6)
    print("linear_i4_dx", M, N, K, group, dt, flush=True)
    dx = _native.linear_i4_dx(dy, q, scale, K, zero=zero, group=group)
    w = S.weight(q, scale, zero, K, group)
    d = dy.double().cpu()
    value, mag = d @ w, d.abs() @ w.abs()
    u = S.half_step(dt)
    err = (u + (N + 2) * S.U32 * (1 + u)) * mag + S.tiny(dt) * d.abs().sum(1)[:, None]
    S.same(dx, value, err + u * (value.abs() + err) + S.tiny(dt), "dx")


def test_gradient_against_differences(gpu):
    import _native
    M, N, K = 6, 48, 96
    _, q, scale, zero = _weight(N, K, 32, True, F16, 4)
    x, dy = _tokens(M, K, F16, 1), _tokens(M, N, F16, 2)
    dx = _native.linear_i4_dx(dy, q, scale, K, zero=zero, group=32).double().cpu()
    w, v = S.weight(q, scale, zero, K, 32), torch.randn((M, K), generator=_gen(3), dtype=torch.float64)
    f = lambda t: float((t @ w.t() * dy.double().cpu()).sum())
    xd, h = x.double().cpu(), 1e-3
    num = (f(xd + h * v) - f(xd - h * v)) / (2 * h)      # linear: exact but for 2^-52 / h of the value
    mag = dy.double().cpu().abs() @ w.abs()
    bound = (2 * 2.0 ** -11 + (N + 2) * S.U32) * mag + 2.0 ** -24
    assert abs(float((dx * v).sum()) - num) <= float((bound * v.abs()).sum()) + 1e-7


@pytest.mark.parametrize("M", [1, 9, 70])
@pytest.mark.parametrize("pad", [2, 6, 64])
def test_strides_outputs_and_scale_types(gpu, M, pad):
    """Rows of a wider buffer with NaN around them, an out of wider rows whose surroundings stay, scales of the other type, more
    than two dimensions."""
    import _native
    N, K = 200, 392
    _, q, scale, zero = _weight(N, K, 64, True, BF16, pad)
    x = _tokens(M, K, F16, 5, pad=pad)
    buf = torch.full((M + 2, N + 3), 7.0, dtype=F16, device="cuda")
    got = _native.linear_i4(x, q, scale, zero=zero, group=64, out=buf[1:1 + M, :N])
    value, bound = S.linear(x, q, scale, zero, K, 64, F16, False)
    S.same(got, value, torch.maximum(bound, S.linear(x, q, scale, zero, K, 64, F16, True)[1]), "y")
    assert bool((buf[0] == 7).all() and (buf[-1] == 7).all() and (buf[:, N:] == 7).all())
    y = _native.linear_i4(x.contiguous().view(1, M, K), q, scale, zero=zero, group=64)
    assert y.shape == (1, M, N) and torch.equal(y[0], got)
    assert _native.linear_i4(x[:0], q, scale, zero=zero, group=64).shape == (0, N)
    assert _native.linear_i4_dx(got[:0], q, scale, K, zero=zero, group=64).shape == (0, K)


def test_what_lies_past_k_is_not_used(gpu):
    """Rows of x that end inside a block, NaN behind them; packed values past K of any kind."""
    import _native
    M, N, K = 5, 40, 150
    _, q, scale, zero = _weight(N, K, 64, True, BF16, 1)
    x = _tokens(M, K, BF16, 6, whole=True, pad=300)
    want = _native.linear_i4(x, q, scale, zero=zero, group=64, dtype=F32)
    S.same(want, *S.linear(x, q, scale, zero, K, 64, F32, True, True), "y")
    full = torch.full((N, 256), 15, dtype=torch.uint8)
    full[:, :K] = S.unpack(q, K)
    q2 = _native.pack_i4(full.cuda())
    assert torch.equal(_native.linear_i4(x, q2, scale, zero=zero, group=64, dtype=F32), want)
    big = x.repeat(20, 1)
    assert torch.equal(_native.linear_i4(big, q2, scale, zero=zero, group=64), _native.linear_i4(big, q, scale, zero=zero, group=64))
    dy = _tokens(3, N, BF16, 7)
    assert torch.equal(_native.linear_i4_dx(dy, q2, scale, K, zero=zero, group=64),
                       _native.linear_i4_dx(dy, q, scale, K, zero=zero, group=64))


@pytest.mark.parametrize("M", [4, 80])
def test_not_finite(gpu, M):
    """A NaN or an infinity spoils its own token, a NaN scale its channel."""
    import _native
    _, q, scale, _ = _weight(64, 256, 128, False, BF16, 3)
    x = _tokens(M, 256, BF16, 3)
    clean = _native.linear_i4(x, q, scale)
    x[1, 7], x[3, 200] = NAN, INF
    scale[1, 5] = NAN
    y = _native.linear_i4(x, q, scale)
    rows = [i for i in range(M) if i not in (1, 3)]
    cols = [i for i in range(64) if i != 5]
    assert torch.equal(y[rows][:, cols], clean[rows][:, cols])
    assert bool(torch.isnan(y[1]).all()) and not bool(torch.isfinite(y[3]).any()) and bool(torch.isnan(y[:, 5]).all())


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M,N,K,group,zeros", [(3, 20500, 200, 32, True), (16, 20500, 72, 128, False), (5, 10300, 300, 64, False),
                                               (2, 10300, 1200, 128, True), (16, 40, 5000, 128, True), (12, 300, 9001, 32, False),
                                               (33, 40, 5120, 64, True), (17, 700, 5130, 32, True), (512, 2048, 2050, 128, False),
                                               (700, 1030, 4104, 32, True), (1025, 2100, 2056, 64, True), (64, 5120, 2056, 128, False)])
def test_forms(gpu, M, N, K, group, zeros, dt):
    """Few tokens by many channels (a wave, two or four sharing a tile's inputs), few tokens of more inputs than fit in LDS, tiles
    of one to four times 16 tokens by 128 or 256 channels, with and without parts of the sums, many tiles of rows."""
    import _native
    _, q, scale, zero = _weight(N, K, group, zeros, dt, M + N + K)
    for whole, pad in ((True, 0), (False, 3)):
        x = _tokens(M, K, dt, N + K, whole, pad)
        print("linear_i4", M, N, K, group, zeros, dt, pad, flush=True)
        got = _native.linear_i4(x, q, scale, zero=zero, group=group, dtype=F32)
        S.same(got, *S.linear(x, q, scale, zero, K, group, F32, True, whole), "y")


def test_streams_and_captured(gpu):
    import _native
    _, q, scale, zero = _weight(300, 520, 32, True, F16, 8)
    for M in (1, 20, 100):
        x = _tokens(M, 520, F16, M)
        want = _native.linear_i4(x, q, scale, zero=zero, group=32)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = _native.linear_i4(x, q, scale, zero=zero, group=32)
        s.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = _native.linear_i4(x, q, scale, zero=zero, group=32)
            dx = _native.linear_i4_dx(y, q, scale, 520, zero=zero, group=32)
        for seed in (1, 2, 3):
            x.copy_(_tokens(M, 520, F16, seed))
            graph.replay()
            torch.cuda.synchronize()
            again = _native.linear_i4(x, q, scale, zero=zero, group=32)
            assert torch.equal(y, again)
            assert torch.equal(dx, _native.linear_i4_dx(again, q, scale, 520, zero=zero, group=32))


@pytest.mark.parametrize("M", [3, 40, 700])
def test_gradient_captured_and_on_a_stream(gpu, M):
    """Straight from the packed weights, in parts and not, and through weights of 16 bits; new gradients between the replays."""
    import _native
    N, K = (1040, 520) if M < 700 else (2056, 2048)
    _, q, scale, zero = _weight(N, K, 64, True, BF16, 9)
    dy = _tokens(M, N, BF16, M)
    f = lambda: _native.linear_i4_dx(dy, q, scale, K, zero=zero, group=64)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = f()
    s.synchronize()
    assert torch.equal(got, f())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    for i in range(3):
        dy.copy_(_tokens(M, N, BF16, M + i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, f())
