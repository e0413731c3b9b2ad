"""What the choice of experts, the products with 4-bit weights and the adjusting of logits refuse, before any device work: the C
entry points by their codes and messages, the Python calls by ValueError. No GPU needed."""
import ctypes as C

import pytest
import torch

import _native

P = 1 << 20    # an address that no refused call reads
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def lib():
    return _native.load()


def _refused(lib, rc, *words):
    msg = lib.gfl_last_error().decode()
    assert rc == 1 and all(w in msg for w in words), (rc, msg)


def test_linear_i4_refusals(lib):
    def linear(x=P, ldx=200, dtype=0, q=P, scale=P, sdt=0, zero=None, M=2, N=8, K=200, group=128, out=P, ldo=8, odt=0, ws=P, nb=1 << 24):
        return lib.gfl_linear_i4(x, ldx, dtype, q, scale, sdt, zero, M, N, K, group, out, ldo, odt, ws, nb, None)

    def dx(x=P, ldx=8, dtype=0, q=P, scale=P, sdt=0, zero=None, M=2, N=8, K=200, group=128, out=P, ldo=200, ws=P, nb=1 << 24):
        return lib.gfl_linear_i4_dx(x, ldx, dtype, q, scale, sdt, zero, M, N, K, group, out, ldo, ws, nb, None)

    for f in (linear, dx):
        for kw, word in ((dict(dtype=2), "dtype"), (dict(sdt=2), "scale_dtype"), (dict(M=-1), "M >= 0"), (dict(M=1 << 24), "GFL_MAX_ROWS"),
                         (dict(N=0), "N"), (dict(K=0), "K"), (dict(N=1 << 22), "GFL_MAX_LD"), (dict(K=1 << 22), "GFL_MAX_LD"),
                         (dict(N=1 << 20, K=4097), "2^32"), (dict(group=16), "group"), (dict(group=256), "group"), (dict(group=0), "group"),
                         (dict(q=None), "NULL"), (dict(scale=None), "NULL"), (dict(x=None), "NULL"), (dict(out=None), "NULL"),
                         (dict(q=P + 8), "aligned"), (dict(ldx=7), "stride"), (dict(ldo=7), "stride"), (dict(ldx=1 << 22), "stride")):
            _refused(lib, f(**kw), word)
        assert f(M=0, x=None, out=None, ws=None, nb=0) == 0
    _refused(lib, linear(odt=3), "out_dtype")
    _refused(lib, linear(ldo=1 << 30), "stride")
    for kw in (dict(ws=None), dict(nb=16), dict(ws=P + 8)):
        # 16-bit weights for 8192 tokens, parts of the sums for 40
        _refused(lib, linear(M=8192, N=4096, K=4096, ldx=4096, ldo=4096, **kw), "workspace")
        _refused(lib, linear(M=40, N=512, K=4096, ldx=4096, ldo=512, **kw), "workspace")
        _refused(lib, dx(M=8192, N=4096, K=4096, ldx=4096, ldo=4096, **kw), "workspace")
        _refused(lib, dx(M=40, N=4096, K=512, ldx=4096, ldo=512, **kw), "workspace")
        _refused(lib, dx(N=7, **kw), "workspace")   # too few rows of the weight for the kernel that needs none


def test_quant_and_pack_i4_refusals(lib):
    def quant(w=P, ld=200, dtype=0, N=8, K=200, group=128, q=P, scale=P):
        return lib.gfl_quant_i4(w, ld, dtype, N, K, group, q, scale, None, None)

    def pack(w=P, ld=200, N=8, K=200, q=P):
        return lib.gfl_pack_i4(w, ld, N, K, q, None)

    for f in (quant, pack):
        for kw, word in ((dict(N=0), "N"), (dict(K=0), "K"), (dict(w=None), "NULL"), (dict(q=None), "NULL"), (dict(q=P + 4), "aligned"),
                         (dict(ld=199), "stride"), (dict(ld=1 << 22), "stride"), (dict(N=1 << 20, K=4097), "2^32")):
            _refused(lib, f(**kw), word)
    _refused(lib, quant(dtype=2), "dtype")
    _refused(lib, quant(group=48), "group")
    _refused(lib, quant(scale=None), "NULL")


def test_i4_workspace(lib):
    f, b = C.c_size_t(), C.c_size_t()
    for M in (0, 1, 64, 65, 5000):
        for N, K in ((1, 1), (77, 131), (12288, 5120)):
            assert lib.gfl_i4_workspace(1, 1, M, N, K, 64, C.byref(f), C.byref(b)) == 0
            assert f.value <= 64 * M * (N + 4) if M <= 64 else N < 12288 or M < 5000 or f.value >= 2 * N * K
            assert b.value <= 64 * M * (K + 4) if N >= 8 and M <= 65 else M == 0 or b.value >= 2 * N * K or (N, K) == (77, 131)
            assert lib.gfl_i4_workspace(1, 2, M, N, K, 32, C.byref(f), None) == 0 and f.value <= 64 * M * (N + 4)
    _refused(lib, lib.gfl_i4_workspace(2, 2, 1, 8, 8, 32, C.byref(f), None), "dtype")
    _refused(lib, lib.gfl_i4_workspace(0, 0, 1, 8, 8, 16, C.byref(f), None), "group")
    _refused(lib, lib.gfl_i4_workspace(0, 0, 1, 0, 8, 32, C.byref(f), None), "N")


def test_route_experts_refusals(lib):
    def fwd(x=P, ld=64, dtype=2, bias=None, M=2, E=64, k=8, score=0, groups=1, top=1, best=1, scale=1.0, sel=P, w=P, wdt=0):
        return lib.gfl_route_experts(x, ld, dtype, bias, M, E, k, score, groups, top, best, 1, scale, sel, w, wdt, None)

    def bwd(x=P, ld=64, dtype=2, M=2, E=64, k=8, score=0, scale=1.0, sel=P, w=P, wdt=2, dx=P, ldd=64):
        return lib.gfl_route_experts_backward(w, wdt, x, ld, dtype, sel, M, E, k, score, 1, scale, dx, ldd, None)

    for f in (fwd, bwd):
        for kw, word in ((dict(dtype=3), "dtypes"), (dict(wdt=-1), "dtypes"), (dict(M=-1), "M >= 0"), (dict(M=1 << 24), "GFL_MAX_ROWS"),
                         (dict(E=0), "E"), (dict(E=1025, ld=1025), "1024"), (dict(k=0), "topk"), (dict(k=65, E=100, ld=100), "topk"),
                         (dict(E=4, k=5), "topk"), (dict(score=2), "score"), (dict(scale=NAN), "scale"), (dict(scale=INF), "scale"),
                         (dict(x=None), "NULL"), (dict(sel=None), "NULL"), (dict(w=None), "NULL"), (dict(ld=63), "stride")):
            _refused(lib, f(**kw), word)
        assert f(M=0, x=None, sel=None, w=None) == 0
    for kw, word in ((dict(groups=0), "groups"), (dict(groups=65, E=130, ld=130), "groups"), (dict(groups=3), "divide"),
                     (dict(groups=8, top=9), "top_groups"), (dict(groups=8, top=0), "top_groups"), (dict(groups=16, top=1), "hold"),
                     (dict(best=0), "group_best"), (dict(best=3), "group_best")):
        _refused(lib, fwd(**kw), word)
    _refused(lib, bwd(dx=None), "NULL")
    _refused(lib, bwd(ldd=63), "stride")


def test_adjust_logits_refusals(lib):
    def call(x=P, ld=100, dtype=2, B=2, V=100, h=P, ldh=9, L=9, length=None, prompt=None, rep=None, freq=None, pres=None, ids=P, ldb=4,
             bias=P, ldv=4, n=4, allowed=P, lda=4, out=2 * P, ldo=100):
        return lib.gfl_adjust_logits(x, ld, dtype, B, V, h, ldh, L, length, prompt, rep, freq, pres, ids, ldb, bias, ldv, n, allowed, lda,
                                     out, ldo, None)

    for kw, word in ((dict(dtype=3), "dtype"), (dict(B=-1), "B"), (dict(B=65536), "65535"), (dict(V=0), "V"),
                     (dict(V=(1 << 20) + 1, ld=1 << 21, ldo=1 << 21), "2^20"), (dict(L=-1), "L"), (dict(L=1 << 20, ldh=1 << 20), "GFL_MAX_HISTORY"),
                     (dict(n=-1), "n_bias"), (dict(n=2048, ldb=2048, ldv=2048), "GFL_MAX_BIASES"), (dict(h=None), "history"),
                     (dict(h=None, L=0, rep=P), "history"), (dict(h=None, L=0, length=P), "history"), (dict(x=None), "NULL"),
                     (dict(out=None), "NULL"), (dict(ids=None), "NULL"), (dict(bias=None), "NULL"), (dict(ld=99), "stride"),
                     (dict(ldo=99), "stride"), (dict(ldh=8), "stride"), (dict(ldb=3), "stride"), (dict(ldv=3), "stride"),
                     (dict(lda=3), "stride"), (dict(out=P, ldo=101), "in place")):
        _refused(lib, call(**kw), word)
    assert call(B=0, x=None, out=None, ids=None) == 0


def test_python_calls_refuse_what_does_not_fit():
    f = lambda *s: torch.zeros(s)
    h = lambda *s: torch.zeros(s, dtype=torch.float16)
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    i64 = lambda *s: torch.zeros(s, dtype=torch.int64)
    # the last of each is not on a device
    for args, kw in (((f(4, 8),), {}), ((h(8),), {}), ((h(4, 8),), dict(group=8)), ((h(0, 8),), {}), ((h(8, 4).t(),), {}), ((h(4, 8),), {})):
        with pytest.raises(ValueError):
            _native.quant_i4(*args, **kw)
    for args in ((f(4, 8),), (u8(8),), (u8(8, 4).t(),), (u8(4, 8),)):
        with pytest.raises(ValueError):
            _native.pack_i4(*args)
    ok = (h(2, 200), u8(8, 128), h(2, 8))
    for args, kw in (((f(2, 200),) + ok[1:], {}), ((h(2, 300),) + ok[1:], {}), ((ok[0], u8(8, 127), ok[2]), {}),
                     ((ok[0], u8(128, 8).t(), ok[2]), {}), (ok[:2] + (h(3, 8),), {}), (ok[:2] + (h(2, 7),), {}), (ok[:2] + (f(2, 8),), {}),
                     (ok[:2] + (h(8, 2).t(),), {}), (ok, dict(zero=u8(2, 7))), (ok, dict(zero=i32(2, 8))), (ok, dict(group=64)),
                     (ok, dict(group=7)), (ok, dict(dtype=torch.int8)), (ok, dict(out=h(2, 9))), (ok, dict(out=f(2, 8), dtype=torch.half)),
                     ((h(200, 2).t(),) + ok[1:], {}), (ok, {})):
        with pytest.raises(ValueError):
            _native.linear_i4(*args, **kw)
    for args, kw in (((h(2, 9), u8(8, 128), h(2, 8), 200), {}), ((f(2, 8), u8(8, 128), h(2, 8), 200), {}),
                     ((h(2, 8), u8(8, 128), h(2, 8), 300), {}), ((h(2, 8), u8(8, 128), h(2, 8), 0), {}),
                     ((h(2, 8), u8(8, 128), h(2, 8), 200), dict(group=32)), ((h(2, 8), u8(8, 128), h(2, 8), 200), {})):
        with pytest.raises(ValueError):
            _native.linear_i4_dx(*args, **kw)
    for args, kw in (((f(8),), {}), ((f(2, 8).double(),), {}), ((f(8, 2).t(),), {}), ((f(2, 8), 0), {}), ((f(2, 100), 65), {}),
                     ((f(2, 8), 2), dict(bias=f(7))), ((f(2, 8), 2), dict(bias=h(8))), ((f(2, 8), 2), dict(score="tanh")),
                     ((f(2, 8), 2), dict(groups=0)), ((f(2, 8), 2), dict(groups=4, top_groups=5)), ((f(2, 8), 2), dict(group_best=3)),
                     ((f(2, 8), 2), dict(dtype=torch.float64)), ((f(2, 8), 2), {})):
        with pytest.raises(ValueError):
            _native.route_experts(*args, **kw)
    for args, kw in (((f(2, 3), f(2, 8), i64(2, 2)), {}), ((f(2, 2), f(2, 8), i32(2, 2)), {}), ((f(2, 2), f(3, 8), i64(2, 2)), {}),
                     ((f(2, 2).double(), f(2, 8), i64(2, 2)), {}), ((f(2, 2).t(), f(2, 8), i64(2, 2)), {}),
                     ((f(2, 2), f(2, 8), i64(2, 2)), dict(score="x")), ((f(2, 2), f(2, 8), i64(2, 2)), {})):
        with pytest.raises(ValueError):
            _native.route_experts_backward(*args, **kw)
    x = f(2, 70)
    for args, kw in (((f(70),), {}), ((x.double(),), {}), ((x,), dict(history=i64(2, 3))), ((x,), dict(history=i32(3, 3))),
                     ((x,), dict(history=i32(3))), ((x,), dict(lengths=i32(2))), ((x,), dict(repetition=f(2))),
                     ((x,), dict(history=i32(2, 3), lengths=i64(2))), ((x,), dict(history=i32(2, 3), repetition=f(3))),
                     ((x,), dict(bias=f(2, 3))), ((x,), dict(bias_ids=i32(2, 3), bias=f(2, 4))), ((x,), dict(bias_ids=i64(2, 3), bias=f(2, 3))),
                     ((x,), dict(allowed=i32(2, 2))), ((x,), dict(allowed=i64(2, 3))), ((x,), dict(out=f(2, 71))), ((x,), dict(out=h(2, 70))),
                     ((x,), dict(out=f(1, 70).expand(2, 70))), ((x,), {})):
        with pytest.raises(ValueError):
            _native.adjust_logits(*args, **kw)
