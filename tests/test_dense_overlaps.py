"""Outputs that share memory with what a call reads are refused before any device work: a workgroup would read what another has written.
No GPU needed: the calls with no overlap are those that a later check refuses, or that fail for want of a device."""
import ctypes as C

import pytest

import _native

P = 1 << 20    # an address that no refused call reads


@pytest.fixture(scope="module")
def lib():
    import torch
    if torch.cuda.is_available():
        pytest.skip("calls that pass the check would be launched on addresses that are not there")
    return _native.load()


def _overlaps(lib, rc):
    """Whether the call was refused for that; what passes reaches a launch, which fails without a device."""
    msg = lib.gfl_last_error().decode()
    assert rc != 0
    return rc == 1 and "overlaps" in msg


def _shared(p, lda, ca, q, ldb, cb, rows):
    """By every byte of every row."""
    seen = {p + i * lda + k for i in range(rows) for k in range(ca)}
    return any(q + i * ldb + k in seen for i in range(rows) for k in range(cb))


@pytest.mark.parametrize("rows", [1, 2, 5])
@pytest.mark.parametrize("ld,ldo", [(10, 10), (24, 24), (33, 33), (24, 12), (10, 31), (40, 10)])
def test_adjust_logits(lib, rows, ld, ldo):
    V = 10
    for at in list(range(-150, 151, 2)):      # bytes: fp16
        want = _shared(P, 2 * ld, 2 * V, P + at, 2 * ldo, 2 * V, rows)
        rc = lib.gfl_adjust_logits(P, ld, 0, rows, V, None, 0, 0, None, None, None, None, None, None, 0, None, 0, 0, None, 0, P + at, ldo, None)
        if at == 0 and (ld == ldo or rows == 1):
            assert not _overlaps(lib, rc)     # in place
        elif at == 0:
            assert rc == 1 and "in place" in lib.gfl_last_error().decode()
        else:
            assert _overlaps(lib, rc) == want, at


@pytest.mark.parametrize("odt", [0, 2])
def test_linear_i4(lib, odt):
    M, N, K = 4, 6, 8
    for ldx, ldo in ((8, 6), (8, 8), (32, 32), (64, 16), (9, 40)):
        for at in range(-400, 401, 2):
            want = _shared(P, 2 * ldx, 2 * K, P + at, ldo * (4 if odt == 2 else 2), N * (4 if odt == 2 else 2), M)
            rc = lib.gfl_linear_i4(P, ldx, 0, 2 * P, 3 * P, 0, None, M, N, K, 32, P + at, ldo, odt, 4 * P, 1 << 20, None)
            assert _overlaps(lib, rc) == want, (ldx, ldo, at)
            if odt == 0:
                rc = lib.gfl_linear_i4_dx(P + at, ldo, 0, 2 * P, 3 * P, 0, None, M, N, K, 32, P, ldx, 4 * P, 1 << 20, None)
                assert _overlaps(lib, rc) == want, (ldx, ldo, at)
