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
