"""Tensors past 2^31 elements or bytes: what lies at their ends against the same call on that part alone, which the other tests
compare with the definitions."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _room(gpu):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("less than 40 GiB free")
    yield
    torch.cuda.empty_cache()


def _rand(*shape, dtype=BF16):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    return out.random_(0, 256) if dtype == torch.uint8 else out.normal_()


def test_route_experts(gpu):
    import _native
    M, E, topk = (1 << 21) + 77, 1024, 4
    x = _rand(M, E)
    kw = dict(groups=8, top_groups=4, dtype=F32)
    print("route_experts", M, E, flush=True)
    sel, w = _native.route_experts(x, topk, **kw)
    dw = _rand(M, topk, dtype=F32)
    d = _native.route_experts_backward(dw, x, sel)
    for a in (0, M // 2, M - 200):
        part = slice(a, a + 200)
        s, v = _native.route_experts(x[part].contiguous(), topk, **kw)
        assert torch.equal(s, sel[part]) and torch.equal(v, w[part])
        # few rows are spread over more lanes, and a row's sum has another order: a rounding in fp64, then bf16's
        e = _native.route_experts_backward(dw[part], x[part].contiguous(), s).float()
        assert bool(((d[part].float() - e).abs() <= 2.0 ** -7 * e.abs() + 2.0 ** -126).all())


@pytest.mark.parametrize("M", [1, 24])
def test_weights(gpu, M):
    """The largest packed weight, 2^31 bytes. Whole numbers: sums in any order are exact."""
    import _native
    N, K, group, few = 1 << 19, 8192, 128, 48
    q = _rand(N, K // 2, dtype=torch.uint8)
    scale = torch.ones((K // group, N), dtype=F16, device="cuda")
    x = torch.randint(-2, 3, (M, K), device="cuda").half()
    print("linear_i4", M, N, K, flush=True)
    y = _native.linear_i4(x, q, scale, group=group, dtype=F32)
    for a in (0, N // 2 - 16, N - few):
        part = slice(a, a + few)
        assert torch.equal(y[:, part], _native.linear_i4(x, q[part], scale[:, part].contiguous(), group=group, dtype=F32))
    dy = torch.zeros((M, N), dtype=F16, device="cuda")
    dy[:, -few:] = torch.randint(-2, 3, (M, few), device="cuda").half()
    print("linear_i4_dx", M, N, K, flush=True)
    dx = _native.linear_i4_dx(dy, q, scale, K, group=group)
    assert torch.equal(dx, _native.linear_i4_dx(dy[:, -few:].contiguous(), q[-few:], scale[:, -few:].contiguous(), K, group=group))


@pytest.mark.parametrize("pack", [False, True])
def test_quantising(gpu, pack):
    import _native
    N, K, few = (1 << 19) + 5, 4104, 40
    w = _rand(N, K, dtype=torch.uint8 if pack else BF16)
    print("pack_i4" if pack else "quant_i4", N, K, flush=True)
    f = (lambda t: (_native.pack_i4(t),)) if pack else (lambda t: _native.quant_i4(t, group=32, zeros=True))
    whole = f(w)
    for a in (0, N // 2, N - few):
        for i, (x, y) in enumerate(zip(whole, f(w[a:a + few]))):
            assert torch.equal(x[a:a + few] if i == 0 else x[:, a:a + few], y)


def test_tokens_of_long_rows(gpu):
    """Rows of x and of the output far apart: the last ones start past 2^31 elements."""
    import _native
    N, K, group, far = 200, 392, 64, (1 << 22) - 1
    q = _rand(N, 4 * 64, dtype=torch.uint8)
    scale = torch.full(((K + group - 1) // group, N), 0.125, dtype=F16, device="cuda")
    for M, dt in ((520, F16), (1040, BF16)):
        buf, out = (torch.empty((M, far), dtype=dt, device="cuda") for _ in range(2))
        buf[:, :K].normal_()
        print("linear_i4", M, N, K, "rows of", far, flush=True)
        _native.linear_i4(buf[:, :K], q, scale, group=group, out=out[:, 5:5 + N])
        x = buf[:, :K].contiguous()
        assert torch.equal(out[:, 5:5 + N], _native.linear_i4(x, q, scale, group=group))
        out[:, :N].normal_()
        dx = _native.linear_i4_dx(out[:, :N], q, scale, K, group=group)
        assert torch.equal(dx, _native.linear_i4_dx(out[:, :N].contiguous(), q, scale, K, group=group))


@pytest.mark.parametrize("M,N,K", [(100003, 3, 5), ((1 << 22) + 5000, 40, 130)])
def test_more_rows_than_a_launch_takes(gpu, M, N, K):
    import _native
    q = _native.pack_i4(_rand(N, K, dtype=torch.uint8))
    scale = torch.full(((K + 63) // 64, N), 0.125, dtype=F16, device="cuda")
    x = _rand(M, K, dtype=F16)
    print("linear_i4", M, N, K, flush=True)
    y = _native.linear_i4(x, q, scale, group=64, dtype=F32)
    for a in (0, M // 2, M - 64):      # one part each: the same sums
        assert torch.equal(y[a:a + 64], _native.linear_i4(x[a:a + 64], q, scale, group=64, dtype=F32))


def test_adjust_logits_of_the_most_rows(gpu):
    import _native
    B, V = 65535, 1 << 20
    if torch.cuda.mem_get_info()[0] < 170 << 30:
        pytest.skip("less than 170 GiB free")
    x = torch.empty((B, V), dtype=BF16, device="cuda")
    part = torch.empty((3, V), dtype=BF16, device="cuda").normal_()
    x[:3], x[-3:] = part, part
    ids = torch.randint(0, V, (B, 4), dtype=torch.int32, device="cuda")
    bias = torch.randn((B, 4), device="cuda")
    print("adjust_logits", B, V, flush=True)
    _native.adjust_logits(x, bias_ids=ids, bias=bias, out=x)
    for a in (0, B - 3):
        assert torch.equal(x[a:a + 3], _native.adjust_logits(part, bias_ids=ids[a:a + 3], bias=bias[a:a + 3]))


def test_adjust_logits(gpu):
    """Logits and histories past 2^31 elements, rows with and without tokens."""
    import _native
    B, V, L = 2100, 1 << 20, (1 << 20) - 1
    x = _rand(B, V)
    history = torch.empty((B, L), dtype=torch.int32, device="cuda").random_(0, V)
    lengths = torch.full((B,), 50, dtype=torch.int32, device="cuda")
    lengths[0], lengths[-1] = L, L - 3
    kw = dict(history=history, lengths=lengths, prompt=lengths // 2, repetition=torch.full((B,), 1.25, device="cuda"),
              frequency=torch.full((B,), 0.5, device="cuda"), allowed=torch.empty((B, V // 32), dtype=torch.int32, device="cuda").random_())
    print("adjust_logits", B, V, L, flush=True)
    out = _native.adjust_logits(x, **kw)
    for a in (0, B // 2, B - 3):
        part = slice(a, a + 3)
        assert torch.equal(out[part], _native.adjust_logits(x[part], **{k: v[part] for k, v in kw.items()}))
