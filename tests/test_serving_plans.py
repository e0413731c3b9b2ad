"""Which form a product with a 4-bit weight and its gradient take (q4_plan, q4_exact and q4_dx_plan of csrc/gfl_gemm_plan.hpp,
compiled for the CPU), on both sides of each change, and the bytes of workspace that gfl_i4_workspace asks for them."""
import ctypes as C
import os
import subprocess

import pytest

import _native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

SOURCE = """
#include "gfl_gemm_plan.hpp"
extern "C" void plan(int M, int N, int K, int group, long long* o)
{
    const gfl::Q4Plan p = gfl::q4_plan(M, N, K);
    o[0] = gfl::q4_exact(M, N, K, group), o[1] = p.few, o[2] = p.tt, o[3] = p.nt, o[4] = p.parts;
}
extern "C" void dx(int M, int N, int K, long long* o)
{
    const gfl::Q4DxPlan p = gfl::q4_dx_plan(M, N, K);
    o[0] = p.direct, o[1] = p.tt, o[2] = p.parts;
}
extern "C" long long gemm_part(int form, int M, int N, int K)
{
    const long long a = gfl::gm_plan(form, gfl::EP_OUT, 0, 0, M, N, K, 1).part_bytes, b = gfl::gm_plan(form, gfl::EP_OUT, 0, 1, M, N, K, 1).part_bytes;
    return a > b ? a : b;
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    clang = os.path.join(ROCM, "llvm", "bin", "clang++")
    if not os.path.exists(clang):
        pytest.skip("no clang++")
    d = tmp_path_factory.mktemp("plans")
    (d / "p.cpp").write_text(SOURCE)
    subprocess.run([clang, "-O1", "-std=c++17", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-w",
                    "-I" + os.path.join(ROOT, "glm-flash-lite_amd", "csrc"), "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROCM, "include"), str(d / "p.cpp"), "-o", str(d / "libp.so")], check=True)
    lib = C.CDLL(str(d / "libp.so"))
    lib.gemm_part.restype = C.c_longlong
    o = (C.c_longlong * 5)()

    def forward(M, N, K, group=128):
        """"few", (tokens / 16, channels / 128, parts) of a tile, or "16 bits" """
        lib.plan(M, N, K, group, o)
        return "few" if o[1] else tuple(o[2:5]) if o[0] else "16 bits"

    def backward(M, N, K):
        """(tokens / 16, parts) straight from the packed weights, or "16 bits" """
        lib.dx(M, N, K, o)
        return tuple(o[1:3]) if o[0] else "16 bits"
    return forward, backward, lib.gemm_part


# (M, N, K, group): the form. A GPU test (test_gpu_linear4_forms.py) sees by their results which of them keep the weights exact.
FORMS = {
    (1, 5120, 5120, 128): "few", (14, 640, 5120, 128): "few", (100, 40, 7, 128): "few",
    (15, 640, 5120, 128): (1, 1, 10), (16, 40, 5000, 128): (1, 1, 10), (17, 640, 5120, 64): (2, 1, 10), (32, 5120, 5120, 32): (2, 1, 6),
    (33, 640, 5120, 32): (4, 1, 10), (64, 5120, 12288, 32): (4, 2, 12), (64, 12288, 5120, 128): (4, 2, 5), (128, 1024, 1024, 128): (4, 1, 4),
    (200, 264, 1000, 64): (4, 1, 4), (513, 77, 131, 32): (4, 1, 1), (300, 1032, 520, 32): (4, 1, 3), (1024, 2048, 2048, 128): (4, 2, 2),
    (256, 12288, 5120, 32): (4, 2, 1), (65, 129, 384, 32): "16 bits", (300, 1000, 264, 128): "16 bits", (2050, 2304, 1040, 64): "16 bits",
    (400, 12288, 5120, 32): "16 bits", (1030, 12288, 5120, 128): "16 bits",
}
# (M, N, K): the gradient's
GRADIENTS = {
    (1, 11008, 4096): (1, 8), (16, 11008, 4096): (1, 8), (17, 11008, 4096): (2, 8), (64, 11008, 4096): (4, 8), (100, 11008, 4096): (4, 4),
    (300, 11008, 4096): (4, 1), (64, 1024, 1024): (4, 2), (256, 2048, 2048): (4, 4), (1, 8, 300): (1, 1), (1, 7, 128): "16 bits",
    (700, 11008, 4096): "16 bits", (1001, 11008, 4096): "16 bits", (4096, 12288, 5120): "16 bits", (2048, 2048, 2048): "16 bits",
}


@pytest.mark.parametrize("size", FORMS)
def test_forward(plans, size):
    assert plans[0](*size) == FORMS[size]


@pytest.mark.parametrize("size", GRADIENTS)
def test_backward(plans, size):
    assert plans[1](*size) == GRADIENTS[size]


def _up(n):
    return (n + 255) // 256 * 256


def _asked(M, N, K, group, out_dtype=1):
    f, b = C.c_size_t(), C.c_size_t()
    assert _native.load().gfl_i4_workspace(1, out_dtype, M, N, K, group, C.byref(f), C.byref(b)) == 0
    return f.value, b.value


def _parts(form, M, cols):
    """Bytes of the parts' sums: fp32, rows of whole 16 bytes; none for one part."""
    parts = 1 if form == "few" else form[-1]
    return _up(parts * M * ((cols + 3) // 4 * 4) * 4) if parts > 1 else 0


@pytest.mark.parametrize("size", FORMS)
def test_forward_workspace(plans, size):
    M, N, K, group = size
    form = FORMS[size]
    weight = _up(N * ((K + 7) // 8 * 8) * 2)
    want = weight + _up(plans[2](0, M, N, K)) if form == "16 bits" else _parts(form, M, N)
    assert _asked(*size)[0] == want
    if form == "16 bits":       # for an fp32 result the weights stay exact: tiles of 64 tokens
        want = _parts(_tile(M, N, K), M, N)
    assert _asked(*size, out_dtype=2)[0] == want


def _tile(M, N, K):
    """q4_plan's tiles of more than 32 tokens, by its rule."""
    blocks, tall = (K + 127) // 128, (M + 63) // 64
    nt = 1 if tall * ((N + 255) // 256) * (blocks // 4) < 256 else 2
    wg = tall * ((N + 128 * nt - 1) // (128 * nt))
    most = max(blocks // 4, min((blocks + 1) // 2, 4))
    return (4, nt, max(1, min(most, 16, 256 // wg)))


@pytest.mark.parametrize("size", GRADIENTS)
def test_backward_workspace(plans, size):
    M, N, K = size
    form = GRADIENTS[size]
    weight = _up(N * ((K + 7) // 8 * 8) * 2)
    assert _asked(M, N, K, 64)[1] == (weight + _up(plans[2](1, M, K, N)) if form == "16 bits" else _parts(form, M, K))
    assert _asked(0, N, K, 64)[1] == 0
