"""Logits adjusted in place without a mask, by lists that name few of them (only those are read) and many (whole rows)."""
import pytest

import serving_ref as S

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("B,V,L,n_bias", [(3, 20011, 100, 7), (3, 20011, 600, 20), (3, 20011, 613, 20), (70, 9000, 0, 30), (70, 9000, 140, 0),
                                          (70, 9000, 2000, 300), (2, 40000, 33000, 9), (1, 300, 9, 0), (1, 300, 3, 1)])
def test_in_place(gpu, B, V, L, n_bias, dt):
    import _native
    g = torch.Generator().manual_seed(V + L)
    x = torch.full((B, V + 5), 7.0)
    x[:, :V] = torch.randn((B, V), generator=g) * 3
    x[0, ::7], x[0, 1::7], x[0, 2::7] = NAN, INF, -INF
    buf = x.to(dt).cuda()
    x, rest = buf[:, :V].clone(), buf[:, V:].clone()
    kw = {}
    if L:
        lengths = torch.randint(L // 2, L + 1, (B,), generator=g, dtype=torch.int32)
        kw = dict(history=(V * torch.rand((B, L), generator=g) ** 3).int(), lengths=lengths, prompt=lengths // 3,
                  repetition=torch.rand(B, generator=g) + 0.6, frequency=torch.randn(B, generator=g), presence=torch.randn(B, generator=g))
    if n_bias:
        kw.update(bias_ids=torch.randint(-2, V + 2, (B, n_bias), generator=g, dtype=torch.int32),
                  bias=torch.randn((B, n_bias), generator=g) * 4)
    dev = {k: v.cuda() for k, v in kw.items()}
    got = _native.adjust_logits(buf[:, :V], out=buf[:, :V], **dev)
    S.same(got, *S.adjust(x.cpu(), **kw), "logits")
    assert torch.equal(got.nan_to_num(5.0), _native.adjust_logits(x, **dev).nan_to_num(5.0))
    assert torch.equal(buf[:, V:].nan_to_num(5.0), rest.nan_to_num(5.0))
