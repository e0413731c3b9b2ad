"""Dense operators whose matrices hold more than 2^31 elements: the last rows, against the 64-bit definition."""
import math

import pytest

import dense_ref as R
from test_gpu_dense import _check_draw

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


@pytest.fixture(autouse=True)
def room():
    if not torch.cuda.is_available() or torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("64 GiB of device memory")
    yield
    torch.cuda.empty_cache()


def test_ffn_tokens(gpu):
    """x, out, dy and dx of 2.2e9 elements."""
    import _native
    M, H, I = 1_060_003, 2056, 72
    g = _gen(1)
    r = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=BF16)
    x, dy = r(M, H), r(M, H)
    wg, wu, wd = r(I, H) / math.sqrt(H), r(I, H) / math.sqrt(H), r(H, I) / math.sqrt(I)
    print("far ffn", flush=True)
    y, gate, up = _native.ffn_forward(x, wg, wu, wd, save=True)
    dx = _native.ffn_backward(dy, x, gate, up, wg, wu, wd, need=(True, False, False, False))[0]
    assert y.numel() > 2 ** 31
    for at in (slice(0, 40), slice(M // 2, M // 2 + 40), slice(M - 40, M)):
        ref = R.FFN(x[at], wg, wu, wd)
        R.within(y[at], ref.y, ref.ey, "y")
        R.within(dx[at], *ref.backward(dy[at])[0], "dx")


def test_gemm_i8_outputs(gpu):
    """Tokens, and outputs, of 2.2e9 elements; the tokens quantised in the same call."""
    import _native
    g = _gen(2)
    for M, N, K in ((1_060_003, 72, 2064), (1_060_003, 2056, 72)):
        x = torch.randn((M, K), generator=g, device="cuda", dtype=BF16)
        b = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
        sb = (torch.rand(N, generator=g, device="cuda") + 0.5) / (127 * math.sqrt(K))
        print("far i8", M, N, K, flush=True)
        y = _native.linear_i8(x, b, sb)
        assert max(x.numel(), y.numel()) > 2 ** 31
        for at in (slice(0, 40), slice(M - 40, M)):
            wq, ws = R.quant(x[at])
            want = wq @ b.double().cpu().t() * ws[:, None] * sb.double().cpu()
            R.within(y[at], want, want.abs() * (R.half_step(BF16) + 5 * 2.0 ** -24) + R.tiny(BF16), "y")
        del x, y


def test_sample_rows(gpu, monkeypatch):
    """Logits of 2.2e9 elements in several rounds of rows."""
    import _native
    import test_gpu_dense as T
    B, V = 16_400, 131_072
    g = _gen(3)
    x = torch.randn((B, V), generator=g, device="cuda", dtype=F16).mul_(2)
    u, t = torch.rand(B, generator=g, device="cuda"), 0.5 + torch.rand(B, generator=g, device="cuda")
    k = torch.full((B,), 50, dtype=torch.int32, device="cuda")
    p = torch.full((B,), 0.9, device="cuda")
    print("far sample", flush=True)
    for kw in (dict(top_k=k), dict(top_p=p)):
        tok, prob = _native.sample(x, u, temperature=t, **kw)
        at = torch.tensor([0, 1023, 1024, B - 17, B - 1], device="cuda")
        monkeypatch.setattr(T, "_draw", lambda *a, **b: (tok[at], prob[at]))
        _check_draw(x[at].float().cpu(), u[at].cpu(), temperature=t[at].cpu(), **{n: v[at].cpu() for n, v in kw.items()})
