"""Products with 4-bit weights in the form that their size gets: exact weights give the fp32 result rounded once, weights of 16 bits
something else, within bounds of its own."""
import pytest

import serving_ref as S
from test_gpu_linear4 import _tokens, _weight
from test_serving_plans import FORMS

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("size", FORMS)
def test_form(gpu, size, dt):
    import _native
    M, N, K, group = size
    print("linear_i4", size, dt, flush=True)
    _, q, scale, zero = _weight(N, K, group, group != 128, dt, M + N + K)
    x = _tokens(M, K, dt, N)
    y = _native.linear_i4(x, q, scale, zero=zero, group=group)
    y32 = _native.linear_i4(x, q, scale, zero=zero, group=group, dtype=F32)
    exact = FORMS[size] != "16 bits"
    assert torch.equal(y, y32.to(dt)) == exact
    # some rows and channels, each on its own
    rows, cols = (torch.arange(0, n, max(1, n // m), device="cuda") for n, m in ((M, 40), (N, 500)))
    part = (x[rows], q[cols], scale[:, cols], zero[:, cols] if zero is not None else None, K, group)
    S.same(y32[rows][:, cols], *S.linear(*part, F32, True), "fp32 y")
    S.same(y[rows][:, cols], *S.linear(*part, dt, exact), "y")


@pytest.mark.parametrize("M,N,K", [(1, 200, 73600), (2, 5200, 36736), (16, 100, 4480), (16, 30, 4488), (1, 10, 73856), (2, 21000, 4096)])
def test_tokens_that_just_fit_lds_and_just_do_not(gpu, M, N, K):
    import _native
    for group, dt in ((32, F16), (128, BF16)):
        print("linear_i4", M, N, K, group, flush=True)
        _, q, scale, zero = _weight(N, K, group, True, dt, M + N)
        x = _tokens(M, K, dt, N, whole=True)
        cols = torch.arange(0, N, max(1, N // 50), device="cuda")
        got = _native.linear_i4(x, q, scale, zero=zero, group=group, dtype=F32)[:, cols]
        S.same(got, *S.linear(x, q[cols], scale[:, cols], zero[:, cols], K, group, F32, True, True), "y")
