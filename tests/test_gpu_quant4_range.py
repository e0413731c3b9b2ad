"""Rounding to 4 bits with zero points where a group's range is past the largest number, by the header's rule in 64 bits."""
import pytest

import serving_ref as S

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("top", [1e38, 1.7e38, 2.5e38, torch.finfo(torch.bfloat16).max])
def test_wide_ranges(gpu, top):
    import _native
    w = torch.randn((6, 64), generator=torch.Generator().manual_seed(1)).double() * 1e36
    w[1, 3], w[1, 9] = top, -top
    w[2, 5], w[2, 6] = -top, top / 3
    w[3, 33], w[4, 40] = top, -top
    w[5, :] = top
    w = w.to(torch.bfloat16)
    q, scale, zero = _native.quant_i4(w.cuda(), group=32, zeros=True)
    f = w.double().view(6, 2, 32)
    lo, hi = f.amin(2).clamp(max=0), f.amax(2).clamp(min=0)
    s = ((hi - lo) / 15).float().to(torch.bfloat16)          # the quotient in fp32, then its type
    assert bool(torch.isfinite(s).all()) and torch.equal(scale.cpu(), s.t())
    sf = s.float()
    z = torch.round(-lo.float() / sf).clamp(max=15)
    v = (torch.round(f.float() / sf[:, :, None]) + z[:, :, None]).clamp(0, 15).view(6, 64)
    assert torch.equal(zero.cpu(), z.t().to(torch.uint8)) and torch.equal(S.unpack(q, 64), v.long())
