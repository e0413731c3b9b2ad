"""Which products of the GPU tests take the largest tiles: gm_plan (csrc/gfl_gemm_plan.hpp) compiled for the CPU, at the sizes
that those tests name."""
import ctypes as C
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
NT, NN, TN = range(3)
OUT, GATE, DACT, I8 = range(4)

SOURCE = """
#include "gfl_gemm_plan.hpp"
extern "C" void plan(int form, int ep, int dual, int aligned, int M, int N, int K, int segs, int nz, int* o)
{
    const gfl::GmPlan p = gfl::gm_plan(form, ep, dual, aligned, M, N, K, segs, nz);
    o[0] = p.tm, o[1] = p.first, o[2] = p.parts;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    clang = os.path.join(ROCM, "llvm", "bin", "clang++")
    if not os.path.exists(clang):
        pytest.skip("no clang++")
    d = tmp_path_factory.mktemp("plan")
    (d / "p.cpp").write_text(SOURCE)
    subprocess.run([clang, "-O1", "-std=c++17", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-w",
                    "-I" + os.path.join(ROOT, "glm-flash-lite_amd", "csrc"), "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROCM, "include"), str(d / "p.cpp"), "-o", str(d / "libp.so")], check=True)
    lib = C.CDLL(str(d / "libp.so"))

    def f(form, ep, M, N, K, dual=0, segs=1, nz=1):
        """(tile rows, columns of a first launch or 0)"""
        o = (C.c_int * 3)()
        lib.plan(form, ep, dual, 1, M, N, K, segs, nz, o)
        return o[0], o[1]
    return f


def _products(plan, M, H, I):
    return dict(gate_up=plan(NT, GATE, M, I, H, dual=1), down=plan(NT, OUT, M, H, I), dh=plan(NN, DACT, M, I, H),
                dx=plan(NN, OUT, M, H, I, segs=2), dwg_dwu=plan(TN, OUT, I, H, M, nz=2), dwd=plan(TN, OUT, H, I, M))


def test_training_pass_in_large_tiles(plan):
    import test_gpu_dense_tiles as T
    for M, H, I in [T.ALL] + T.RAGGED:
        p = _products(plan, M, H, I)
        assert all(tm == 256 for tm, _ in p.values()), p
        assert p["gate_up"][1] and p["dwd"][1]
        assert M % 32 and H % 32 and I % 32 and H % 256 and I % 256
    assert [s[1] % 8 == s[2] % 8 == 0 for s in [T.ALL] + T.RAGGED] == [True, False, False]
    assert [s[2] % 4 == 0 for s in T.RAGGED] == [True, False]


def test_last_columns_in_a_launch_of_their_own(plan):
    import test_gpu_dense_tiles as T
    for name, (M, H, I) in T.REST.items():
        p = _products(plan, M, H, I)[name]
        assert p[0] == 256 and p[1] and M % 32 and H % 32 and I % 32, (name, p)


def test_gemm_i8_in_large_tiles(plan):
    import test_gpu_dense_tiles as T
    p = [plan(NT, I8, *s) for s in T.I8]
    assert all(tm == 256 for tm, _ in p) and [bool(f) for _, f in p] == [False, False, True, True], p
    assert all(K % 64 and N % 256 for _, N, K in T.I8) and T.I8[1][2] % 4
