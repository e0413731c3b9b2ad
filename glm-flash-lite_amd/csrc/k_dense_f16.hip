// Tile products of the dense operators, f16 inputs.
#include "gfl_gemm_launch.hpp"

namespace gfl {

int launch_gemm_f16(int form, int ep, int dual, int aligned, GmArgs& a, void* ws, size_t ws_bytes, int nz, hipStream_t st)
{
    return launch_gemm<GmF16>(form, ep, dual, aligned, a, ws, ws_bytes, nz, st);
}

}  // namespace gfl
