"""What the dense operators refuse, before any device work: the C entry points by their codes and messages, the Python calls
by ValueError. No GPU needed."""
import ctypes as C

import pytest
import torch

import _native

P = 1 << 20    # an address that no refused call reads


@pytest.fixture(scope="module")
def lib():
    return _native.load()


def _refused(lib, rc, *words):
    msg = lib.gfl_last_error().decode()
    assert rc == 1 and all(w in msg for w in words), (rc, msg)


def _ffn(lib, x=P, ldx=64, wg=P, wu=P, wd=P, dtype=0, M=2, H=64, I=32, L=0.0, g=None, u=None, out=P, ldo=64, odt=0, acc=0,
         ws=P, nb=1 << 20):
    return lib.gfl_ffn_forward(x, ldx, wg, wu, wd, dtype, M, H, I, L, g, u, out, ldo, odt, acc, ws, nb, None)


def test_ffn_forward_refusals(lib):
    for kw, word in ((dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(M=-1), "M >= 0"), (dict(H=0), "H"),
                     (dict(I=0), "I"), (dict(H=1 << 22), "GFL_MAX_LD"), (dict(L=-1.0), "act_limit"),
                     (dict(L=float("nan")), "act_limit"), (dict(odt=1), "out_dtype"), (dict(odt=3), "out_dtype"),
                     (dict(acc=1), "accumulate"), (dict(x=None), "NULL"), (dict(wg=None), "NULL"), (dict(wu=None), "NULL"),
                     (dict(wd=None), "NULL"), (dict(out=None), "NULL"), (dict(g=P), "together"), (dict(u=P), "together"),
                     (dict(ldx=63), "strides"), (dict(ldo=63), "strides"), (dict(ldx=1 << 22), "strides"),
                     (dict(ws=None), "workspace"), (dict(nb=16), "workspace"), (dict(ws=P + 8), "workspace")):
        _refused(lib, _ffn(lib, **kw), word)
    assert _ffn(lib, M=0, x=None, wg=None, wu=None, wd=None, out=None, ws=None, nb=0) == 0


def _bwd(lib, dy=P, lddy=64, x=P, ldx=64, g=P, u=P, wg=P, wu=P, wd=P, dtype=0, M=2, H=64, I=32, L=0.0, dx=P, lddx=64,
         dwg=P, dwu=P, dwd=P, ws=P, nb=1 << 20):
    return lib.gfl_ffn_backward(dy, lddy, x, ldx, g, u, wg, wu, wd, dtype, M, H, I, L, dx, lddx, dwg, dwu, dwd, ws, nb, None)


def test_ffn_backward_refusals(lib):
    for kw, word in ((dict(dtype=2), "dtype"), (dict(M=-1), "M >= 0"), (dict(L=-0.5), "act_limit"), (dict(dy=None), "NULL"),
                     (dict(g=None), "NULL"), (dict(u=None), "NULL"), (dict(wd=None), "NULL"), (dict(lddy=63), "strides"),
                     (dict(lddx=63), "strides"), (dict(ws=None), "workspace"), (dict(nb=16), "workspace")):
        _refused(lib, _bwd(lib, **kw), word)
    assert _bwd(lib, dx=None, dwg=None, dwu=None, dwd=None) == 0    # nothing wanted, nothing launched


def test_i8_refusals(lib):
    def gemm(a=P, lda=64, sa=P, b=P, ldb=64, sb=P, M=2, N=8, K=64, out=P, ldo=8, odt=0, ws=P, nb=1 << 24):
        return lib.gfl_gemm_i8(a, lda, sa, b, ldb, sb, M, N, K, out, ldo, odt, ws, nb, None)

    def linear(x=P, ldx=64, dtype=0, b=P, ldb=64, sb=P, M=2, N=8, K=64, out=P, ldo=8, odt=0, ws=P, nb=1 << 24):
        return lib.gfl_linear_i8(x, ldx, dtype, b, ldb, sb, M, N, K, out, ldo, odt, ws, nb, None)

    for f in (gemm, linear):
        for kw, word in ((dict(M=-1), "M >= 0"), (dict(N=0), "N"), (dict(K=0), "K"), (dict(K=131072), "131071"),
                         (dict(b=None), "NULL"), (dict(sb=None), "NULL"), (dict(out=None), "NULL"), (dict(ldb=63), "strides"),
                         (dict(ldo=7), "strides"), (dict(odt=3), "out_dtype")):
            _refused(lib, f(**kw), word)
    _refused(lib, gemm(a=None), "NULL")
    _refused(lib, gemm(lda=63), "stride")
    _refused(lib, linear(dtype=2), "dtype")
    _refused(lib, linear(ldx=63), "stride")
    _refused(lib, linear(nb=16), "workspace")
    _refused(lib, lib.gfl_quant_i8(P, 64, 2, 2, 64, P, P, None), "dtype")
    _refused(lib, lib.gfl_quant_i8(P, 63, 0, 2, 64, P, P, None), "stride")
    _refused(lib, lib.gfl_quant_i8(None, 64, 0, 2, 64, P, P, None), "NULL")
    assert gemm(M=0, a=None, b=None) == 0 and lib.gfl_quant_i8(None, 64, 0, 0, 64, None, None, None) == 0


def test_sample_refusals(lib):
    def call(logits=P, ld=100, dtype=2, B=2, V=100, u=P, token=P, ws=P, nb=1 << 24):
        return lib.gfl_sample(logits, ld, dtype, B, V, None, None, None, None, u, token, None, ws, nb, None)

    for kw, word in ((dict(dtype=3), "dtype"), (dict(B=-1), "B"), (dict(V=0), "V"), (dict(V=(1 << 20) + 1, ld=1 << 21), "V"),
                     (dict(ld=99), "stride"), (dict(logits=None), "NULL"), (dict(u=None), "NULL"), (dict(token=None), "NULL")):
        _refused(lib, call(**kw), word)
    assert call(B=0, logits=None, u=None, token=None) == 0


def test_workspace_sizes(lib):
    """A workspace query answers for every size and never shrinks with the tokens; the empty call needs none."""
    f, b = C.c_size_t(), C.c_size_t()
    assert lib.gfl_ffn_workspace(0, 0, 64, 64, C.byref(f), C.byref(b)) == 0 and f.value == b.value == 0
    for M in (1, 16, 17, 64, 65, 200, 5000):
        for H, I in ((1, 1), (131, 77), (5120, 1536), (4096, 11008)):
            assert lib.gfl_ffn_workspace(1, M, H, I, C.byref(f), C.byref(b)) == 0
            assert f.value >= 2 * M * I and b.value >= 6 * M * I
            assert lib.gfl_i8_workspace(M, I, H, C.byref(f), C.byref(b)) == 0 and b.value >= M * H + 4 * M
    assert lib.gfl_ffn_workspace(2, 1, 64, 64, C.byref(f), None) == 1
    assert lib.gfl_sample_workspace(3, 1 << 21, C.byref(f)) == 1


def test_python_calls_refuse_what_does_not_fit():
    h = lambda *s: torch.zeros(s, dtype=torch.float16)
    x, wg, wu, wd = h(2, 64), h(32, 64), h(32, 64), h(64, 32)
    for args in ((h(2, 60), wg, wu, wd), (x, h(32, 60), wu, wd), (x, wg, h(30, 64), wd), (x, wg, wu, h(32, 64)),
                 (x.float(), wg, wu, wd), (x, wg.bfloat16(), wu, wd), (x, wg, wu, h(32, 64).t()),
                 (h(64, 2).t(), wg, wu, wd), (x[:1].expand(2, 64), wg, wu, wd), (x, wg, wu, wd)):   # the last: not on a device
        with pytest.raises(ValueError):
            _native.ffn_forward(*args)
    i8 = lambda *s: torch.zeros(s, dtype=torch.int8)
    f = lambda *s: torch.zeros(s)
    for args in ((x, f(2), i8(8, 64), f(8)), (i8(2, 64), f(3), i8(8, 64), f(8)), (i8(2, 64), f(2), i8(8, 60), f(8)),
                 (i8(2, 64), f(2), i8(8, 64), f(7)), (i8(2, 64), f(2), i8(8, 64), f(8))):
        with pytest.raises(ValueError):
            _native.gemm_i8(*args)
    for args, kw in (((f(2, 9), f(3)), {}), ((f(9), f(1)), {}), ((f(2, 9).double(), f(2)), {}),
                     ((f(2, 9), f(2)), dict(top_k=torch.zeros(2, dtype=torch.int64))), ((f(2, 9), f(2)), dict(top_p=f(1))),
                     ((f(2, 9), f(2)), {})):
        with pytest.raises(ValueError):
            _native.sample(*args, **kw)


def test_sizes_past_a_launch(lib):
    """What a grid could not hold is refused by size."""
    _refused(lib, _ffn(lib, M=1 << 24), "GFL_MAX_ROWS")
    _refused(lib, _bwd(lib, M=1 << 24), "GFL_MAX_ROWS")
    _refused(lib, lib.gfl_quant_i8(P, 64, 0, 1 << 24, 64, P, P, None), "GFL_MAX_ROWS")
    for M, N in ((1 << 24, 8), (1, 1 << 26)):
        _refused(lib, lib.gfl_gemm_i8(P, 64, P, P, 64, P, M, N, 64, P, N, 0, P, 1 << 24, None), "GFL_MAX")
        _refused(lib, lib.gfl_linear_i8(P, 64, 0, P, 64, P, M, N, 64, P, N, 0, P, 1 << 24, None), "GFL_MAX")
        _refused(lib, lib.gfl_i8_workspace(M, N, 64, None, None), "GFL_MAX")
