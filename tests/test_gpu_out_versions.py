"""Calls that write into a tensor of the caller's: autograd sees that it has other values now."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, F32 = torch.float16, torch.float32


def _calls():
    """name: (the call on an out, the out's shape and type)"""
    import _native
    g = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=g).half().cuda()
    x, w = rand(5, 64), rand(32, 64)
    q4, s4, _ = _native.quant_i4(w, group=32)
    q8, s8 = _native.quant_i8(w)
    a8, sa = _native.quant_i8(x)
    wg, wu, wd = rand(16, 64), rand(16, 64), rand(64, 16)
    logits = torch.randn((5, 32), generator=g).cuda()
    return {
        "adjust_logits": (lambda out: _native.adjust_logits(logits, out=out), (5, 32), F32),
        "linear_i4": (lambda out: _native.linear_i4(x, q4, s4, group=32, out=out), (5, 32), F16),
        "linear_i8": (lambda out: _native.linear_i8(x, q8, s8, out=out), (5, 32), F16),
        "gemm_i8": (lambda out: _native.gemm_i8(a8, sa, q8, s8, out=out), (5, 32), F16),
        "ffn_forward": (lambda out: _native.ffn_forward(x, wg, wu, wd, out=out), (5, 64), F16),
    }


@pytest.mark.parametrize("name", ["adjust_logits", "linear_i4", "linear_i8", "gemm_i8", "ffn_forward"])
def test_out_saved_for_a_backward_pass(gpu, name):
    call, shape, dt = _calls()[name]
    out = torch.ones(shape, dtype=dt, device="cuda")
    a = torch.ones(shape, dtype=dt, device="cuda", requires_grad=True)
    before = out._version
    y = (a * out).sum()
    call(out)
    assert out._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        kept = torch.empty(shape, dtype=dt, device="cuda")
    call(kept)          # a tensor of an inference pass has no version
    assert torch.equal(kept, out)


def test_logits_adjusted_in_place(gpu):
    import _native
    x = torch.randn((2, 40), device="cuda")
    a = torch.ones((2, 40), device="cuda", requires_grad=True)
    y = (a * x).sum()
    ids, by = torch.zeros((2, 1), dtype=torch.int32, device="cuda"), torch.ones((2, 1), device="cuda")
    _native.adjust_logits(x, bias_ids=ids, bias=by, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
