// Products with 4-bit weights (k_quant4.hip has their layout): y[m][n] = sum over groups of s[g][n] * sum_k x[m][k] (v[n][k] - z[g][n]).
//
// The values go into the MFMAs as they are: 16 + v in the type of x is one shift and one mask and-or for two of them (v in the
// mantissa's upper bits, exact), and a second MFMA by ones sums the tokens' inputs, so that a group adds
// s * (sum x (16 + v) - (16 + z) sum x) to the fp32 sums, with no rounding of a weight.
#include "gfl_gemm.hpp"
#include "gfl_quant.hpp"

#include <algorithm>

namespace gfl {

__device__ __forceinline__ gm_i4 q4_frag(GmBF16, uint32_t w)
{
    constexpr uint32_t M = 0x00780078, O = 0x41804180;
    return gm_i4{ (int)((w << 3 & M) | O), (int)((w >> 1 & M) | O), (int)((w >> 5 & M) | O), (int)((w >> 9 & M) | O) };
}
__device__ __forceinline__ gm_i4 q4_frag(GmF16, uint32_t w)
{
    constexpr uint32_t M = 0x03C003C0, O = 0x4C004C00;
    return gm_i4{ (int)((w << 6 & M) | O), (int)((w << 2 & M) | O), (int)((w >> 2 & M) | O), (int)((w >> 6 & M) | O) };
}
__device__ __forceinline__ gm_i4 q4_ones(GmBF16) { return gm_i4{ 0x3F803F80, 0x3F803F80, 0x3F803F80, 0x3F803F80 }; }
__device__ __forceinline__ gm_i4 q4_ones(GmF16) { return gm_i4{ 0x3C003C00, 0x3C003C00, 0x3C003C00, 0x3C003C00 }; }

// 16 channels and 16 TT tokens by NW waves that take the blocks of 128 inputs in turn and join their sums in LDS. GB: groups of a
// block.
template <typename T, int GB, int TT, int NW>
__global__ __launch_bounds__(NW * 64) void q4_kernel(Q4Args a)
{
    constexpr int WG = 4 / GB;   // words of a group
    __shared__ gm_f4 red[NW][TT][64];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    const int n = min((int)blockIdx.x * 16 + r, a.N - 1), m0 = blockIdx.y * 16 * TT;
    const char* w = reinterpret_cast<const char*>(a.q) + (int64_t)n * a.blocks * 64 + g * 16;
    const char* x[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) x[t] = a.x + (int64_t)min(m0 + t * 16 + r, a.M - 1) * a.ldx + g * 16;
    const int groups = (a.K + a.group - 1) / a.group;
    gm_f4 acc[TT] = {};
    for (int c = wave; c < a.blocks; c += NW)
    {
        gm_i4 v;
        __builtin_memcpy(&v, w + (int64_t)c * 64, 16);
        const bool whole = (c + 1) * 128 <= a.K;
#pragma unroll
        for (int i = 0; i < GB; ++i)
        {
            const int64_t at = (int64_t)min(c * GB + i, groups - 1) * a.N + n;
            const float s = q4_scale(a, at), z = a.zero ? 16.0f + (float)a.zero[at] : 24.0f;
            gm_f4 sum[TT] = {}, xs[TT] = {};
#pragma unroll
            for (int j = i * WG; j < (i + 1) * WG; ++j)
            {
                const gm_i4 b = q4_frag(T{}, (uint32_t)v[j]);
#pragma unroll
                for (int t = 0; t < TT; ++t)
                {
                    const char* p = x[t] + (c * 128 + j * 32) * 2;
                    gm_i4 f;
                    if (whole) __builtin_memcpy(&f, p, 16);
                    else f = gm_masked<2>(p, (a.K - c * 128 - j * 32 - g * 8) * 2);
                    sum[t] = T::mfma(f, b, sum[t]);
                    xs[t] = T::mfma(f, q4_ones(T{}), xs[t]);
                }
            }
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(s, fmaf(-z, xs[t][e], sum[t][e]), acc[t][e]);
        }
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) red[wave][t][lane] = acc[t];
    __syncthreads();
    for (int t = wave; t < TT; t += NW)
    {
        gm_f4 v = red[0][t][lane];
        for (int k = 1; k < NW; ++k) v += red[k][t][lane];
        if ((int)blockIdx.x * 16 + r >= a.N) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            const int m = m0 + t * 16 + g * 4 + e;
            if (m < a.M) gm_put1(a.out, a.odt, (int64_t)m * a.ldo + n, v[e]);
        }
    }
}

template <typename T, int GB>
static void q4_go(const Q4Args& a, hipStream_t st)
{
    const int tt = a.M > 32 ? 4 : a.M > 16 ? 2 : 1, wide = (a.N + 15) / 16;
    auto* kern = tt == 4 ? &q4_kernel<T, GB, 4, 8> : tt == 2 ? &q4_kernel<T, GB, 2, 8> : &q4_kernel<T, GB, 1, 8>;
    // a launch has fewer than 2^32 threads (512 a workgroup) and 65536 workgroups in y
    const int rows = std::max(1, std::min(65535, (1 << 22) / wide)) * 16 * tt;
    for (int m = 0; m < a.M; m += rows)
    {
        Q4Args b = a;
        b.x += (int64_t)m * a.ldx;
        b.M = std::min(rows, a.M - m);
        b.out = static_cast<char*>(a.out) + (int64_t)m * a.ldo * (a.odt == 2 ? 4 : 2);
        hipLaunchKernelGGL(kern, dim3(wide, (b.M + 16 * tt - 1) / (16 * tt)), dim3(512), 0, st, b);
    }
}

void launch_linear_i4(const Q4Args& a, int bf16, hipStream_t st)
{
    if (bf16) (a.group == 32 ? &q4_go<GmBF16, 4> : a.group == 64 ? &q4_go<GmBF16, 2> : &q4_go<GmBF16, 1>)(a, st);
    else (a.group == 32 ? &q4_go<GmF16, 4> : a.group == 64 ? &q4_go<GmF16, 2> : &q4_go<GmF16, 1>)(a, st);
}

}  // namespace gfl
