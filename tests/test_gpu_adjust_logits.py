"""Penalties, biases and masks on logits on the GPU (gfl_adjust_logits) against their definition."""
import pytest

import serving_ref as S

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _inputs(B, V, L, n_bias, masked, seed, dt=F32, pad=0):
    g = _gen(seed)
    x = torch.full((B, V + pad), NAN)
    x[:, :V] = torch.randn((B, V), generator=g) * 3
    kw = {}
    if L is not None:
        h = (V * torch.rand((B, L), generator=g) ** 3).int().clamp(max=V - 1)
        lengths = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
        kw = dict(history=h, lengths=lengths, prompt=(lengths * torch.rand(B, generator=g)).int(),
                  repetition=torch.rand(B, generator=g) + 0.6, frequency=torch.randn(B, generator=g), presence=torch.randn(B, generator=g))
    if n_bias is not None:
        kw.update(bias_ids=torch.randint(-2, V + 2, (B, n_bias), generator=g, dtype=torch.int32),
                  bias=torch.randn((B, n_bias), generator=g) * 4)
    if masked is not None:
        words = (V + 31) // 32
        bits = torch.zeros((B, words * 32), dtype=torch.int64)
        bits[:, :V] = torch.rand((B, V), generator=g) >= masked
        m = (bits.view(B, words, 32) << torch.arange(32)).sum(2)
        kw["allowed"] = torch.where(m >= 2 ** 31, m - 2 ** 32, m).int()
    return x.to(dt).cuda()[:, :V], {k: v.cuda() for k, v in kw.items()}


def _check(x, kw, **more):
    import _native
    print("adjust_logits", list(x.shape), x.dtype, {k: list(v.shape) for k, v in kw.items()}, flush=True)
    got = _native.adjust_logits(x, **kw, **more)
    S.same(got, *S.adjust(x.cpu(), **{k: v.cpu() for k, v in kw.items()}), "logits")
    return got


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("B,V,L,n_bias,masked", [(1, 1000, 50, 3, 0.5), (3, 10007, 700, 40, 0.9), (2, 8192, 0, 0, None), (5, 33, 9, 2, 0.2),
                                                 (1, 1, 3, 1, 0.0), (2, 40000, None, 7, None), (2, 16385, None, None, 0.99),
                                                 (4, 31, 20, None, 1.0), (1, 20000, 3000, None, None), (7, 100, 1, 1, None)])
def test_adjust(gpu, B, V, L, n_bias, masked, dt):
    _check(*_inputs(B, V, L, n_bias, masked, B + V, dt))
    _check(*_inputs(B, V, L, n_bias, masked, B + V + 1, dt, pad=3))


@pytest.mark.parametrize("drop", ["lengths", "prompt", "repetition", "frequency", "presence", "allowed"])
def test_each_setting_left_off(gpu, drop):
    x, kw = _inputs(3, 500, 60, 5, 0.3, 7)
    del kw[drop]
    _check(x, kw)


def test_nothing_asked_is_a_copy(gpu):
    import _native
    x, _ = _inputs(3, 777, None, None, None, 1)
    x[0, 3], x[1, 4], x[2, 5] = NAN, INF, -INF
    got = _native.adjust_logits(x)
    assert got.data_ptr() != x.data_ptr() and torch.equal(got.nan_to_num(5.0), x.nan_to_num(5.0))
    assert _native.adjust_logits(x[:0]).shape == (0, 777)


def test_rows_with_everything_off(gpu):
    """repetition 1 or not above 0, frequency 0, presence 0: the row stays, whatever its history."""
    x, kw = _inputs(4, 300, 80, None, None, 2)
    kw["lengths"][:] = 80
    kw["repetition"][:] = torch.tensor([1.0, 0.0, -2.0, NAN])
    kw["frequency"][:] = 0
    kw["presence"][:] = 0
    assert torch.equal(_check(x, kw), x)


def test_ids_that_no_token_has_and_lengths_out_of_range(gpu):
    x, kw = _inputs(4, 200, 30, 6, None, 3)
    kw["history"][0, :5] = torch.tensor([-1, 200, 2 ** 31 - 1, -2 ** 31, 199], dtype=torch.int32)
    kw["bias_ids"][1, :4] = torch.tensor([-1, 200, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    kw["lengths"][:] = torch.tensor([30, 99, -4, 0])
    kw["prompt"][:] = torch.tensor([-3, 99, 7, 1])
    _check(x, kw)


def test_the_last_bias_of_an_id_counts(gpu):
    x, kw = _inputs(2, 50, None, 8, None, 4)
    kw["bias_ids"][:] = 11
    kw["bias"][0] = torch.arange(8.0)
    got = _check(x, kw)
    assert float(got[0, 11]) == float(x[0, 11] + 7)


def test_counts_beyond_16_bits_and_long_histories(gpu):
    B, V, L = 2, 300, 70000
    x = torch.randn((B, V), generator=_gen(1)).cuda()
    h = torch.full((B, L), 17, dtype=torch.int32)
    h[1] = torch.arange(L) % 299
    kw = dict(history=h.cuda(), frequency=torch.tensor([0.5, 0.25]).cuda(), presence=torch.tensor([0.0, 1.0]).cuda())
    _check(x, kw)


def test_longest_lists(gpu):
    """2^20 - 1 tokens of one kind fill the count; 2047 biases."""
    import _native
    V, L = 70, (1 << 20) - 1
    x = torch.zeros((1, V), device="cuda")
    h = torch.full((1, L), 69, dtype=torch.int32, device="cuda")
    ids = (torch.arange(2047, dtype=torch.int32) % 70).view(1, -1).cuda()
    got = _native.adjust_logits(x, history=h, frequency=torch.ones(1).cuda(), bias_ids=ids, bias=torch.ones((1, 2047)).cuda() * ids)
    want = torch.arange(70.0)
    want[69] -= L
    assert torch.equal(got[0].cpu(), want)


def test_infinities_nan_and_masks(gpu):
    """What is masked is -inf whatever it was; NaN and -inf elsewhere stay; a mask that leaves nothing."""
    x, kw = _inputs(4, 90, 40, 5, 0.5, 5)
    x[0, ::3], x[1, ::4], x[2, ::5] = NAN, INF, -INF
    kw["allowed"][3] = 0
    kw["lengths"][:] = 40
    got = _check(x, kw)
    assert bool(torch.isneginf(got[3]).all())
    low, kw2 = _inputs(2, 90, None, None, 0.5, 6, F16)
    low[:] = torch.finfo(F16).min
    _check(low, kw2)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_in_place_and_strided_out(gpu, dt):
    import _native
    x, kw = _inputs(5, 3001, 300, 9, 0.6, 8, dt, pad=7)
    want = _check(x, kw)
    buf = torch.full((7, 3010), 7.0, dtype=dt, device="cuda")
    _native.adjust_logits(x, out=buf[1:6, :3001], **kw)
    assert torch.equal(buf[1:6, :3001], want) and bool((buf[0] == 7).all() and (buf[6] == 7).all() and (buf[:, 3001:] == 7).all())
    y = x.clone()
    assert _native.adjust_logits(y, out=y, **kw).data_ptr() == y.data_ptr() and torch.equal(y, want)
    _native.adjust_logits(x, out=x, **kw)
    assert torch.equal(x, want)
    for drop in (("allowed",), ("bias", "bias_ids"), ("allowed", "bias", "bias_ids")):
        x, kw = _inputs(5, 3001, 300, 9, 0.6, 8, dt, pad=7)
        few = {k: v for k, v in kw.items() if k not in drop}
        want = _check(x, few)
        assert torch.equal(_native.adjust_logits(x, out=x, **few), want)


def test_strided_lists(gpu):
    x, kw = _inputs(3, 400, 64, 10, 0.5, 9)
    wide = {}
    for k, v in kw.items():
        if v.dim() == 2:
            w = torch.full((v.shape[0], v.shape[1] + 5), 1, dtype=v.dtype, device="cuda")
            w[:, 2:2 + v.shape[1]] = v
            wide[k] = w[:, 2:2 + v.shape[1]]
        else:
            wide[k] = v
    assert torch.equal(_check(x, kw), _check(x, wide))


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("B,V,L,n_bias,masked", [(67, 5000, 300, 4, 0.5), (64, 33000, 100, 0, None), (129, 2050, 2050, None, 0.1),
                                                 (3, 131072, 40000, 2047, 0.8), (2, 262147, 900, 2047, None), (70, 129, 33000, 300, None)])
def test_many_rows_and_large_vocabularies(gpu, B, V, L, n_bias, masked, dt):
    _check(*_inputs(B, V, L, n_bias, masked, B + V, dt, pad=5))


def test_streams_and_captured(gpu):
    import _native
    x, kw = _inputs(3, 5000, 200, 12, 0.5, 10)
    want = _native.adjust_logits(x, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _native.adjust_logits(x, **kw)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _native.adjust_logits(x, **kw)
    for seed in (1, 2, 3):
        x2, kw2 = _inputs(3, 5000, 200, 12, 0.5, seed)
        x.copy_(x2)
        for k in kw:
            kw[k].copy_(kw2[k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, _native.adjust_logits(x2, **kw2))
