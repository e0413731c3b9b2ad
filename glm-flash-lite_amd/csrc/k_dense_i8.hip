// Tile products of the dense operators, i8 inputs.
#include "gfl_gemm_launch.hpp"
#include "gfl_quant.hpp"

namespace gfl {

int launch_gemm_i8(int form, int ep, int dual, int aligned, GmArgs& a, void* ws, size_t ws_bytes, int nz, hipStream_t st)
{
    return launch_gemm<GmI8>(form, ep, dual, aligned, a, ws, ws_bytes, nz, st);
}

// gfl_linear_i8 of one or two tokens in one launch: every workgroup quantises the tokens itself (into LDS, while the first of its
// weights are on their way), then takes columns as gm_row_kernel does, U KB of a row at a time. K is a multiple of 8 from 1024 to
// LQ_K, token rows are 16-byte aligned. Loads have no condition but a place to read: behind a branch the compiler waits for all
// that may be under way (9.5 us instead of 8.2 below). Weights from HBM, us, against gfl_quant_i8's launch and then the product's: one
// token 5120 x 5120 8.2 and 10.9, 8192 x 8192 14.6 and 18.9, 4096 -> 65536 47 and 50; two tokens 11.7 and 11.9, 47 and 50.
template <bool BF, int MM, int U>
__global__ __launch_bounds__(256) void linear_row_kernel(GmArgs a)
{
    constexpr int NC = LQ_K / 2048;   // chunks of 8 elements a thread holds of a token
    __shared__ __align__(16) int8_t xq[MM][LQ_K];
    __shared__ uint32_t red[MM][4];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, kb = a.K, whole = kb / 1024;
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    u16x8 keep[MM][NC];
#pragma unroll
    for (int m = 0; m < MM; ++m)
#pragma unroll
        for (int s = 0; s < NC; ++s)
        {
            const int k = (s * 256 + (int)threadIdx.x) * 8;
            keep[m][s] = *reinterpret_cast<const u16x8*>(a.A[0] + m * a.lda + min(k, kb - 8) * 2);
        }
    int row = (blockIdx.x * 4 + wave) * 2;
    const char *w0, *w1;
    gm_i4 f0[U], f1[U];
    auto aim = [&]() {
        w0 = a.B[0] + (int64_t)min(row, a.N - 1) * a.ldb + lane * 16;
        w1 = row + 1 < a.N ? w0 + a.ldb : w0;
    };
    auto load = [&](int c) {
#pragma unroll
        for (int j = 0; j < U; ++j)
        {
            __builtin_memcpy(&f0[j], w0 + min(c + j, whole - 1) * 1024, 16);
            __builtin_memcpy(&f1[j], w1 + min(c + j, whole - 1) * 1024, 16);
        }
    };
    aim();
    load(0);
    __builtin_amdgcn_sched_barrier(0);   // (the loads would move behind the waits for the tokens)
#pragma unroll
    for (int m = 0; m < MM; ++m)
    {
        uint32_t top = 0;   // (chunks past the end repeat the last one)
#pragma unroll
        for (int s = 0; s < NC; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, (uint32_t)(keep[m][s][i] & 0x7FFF));
#pragma unroll
        for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
        if (lane == 0) red[m][wave] = top;
    }
    gm_barrier();   // (waits for LDS alone: the weights stay under way)
    float scale[MM];
#pragma unroll
    for (int m = 0; m < MM; ++m)
    {
        const QRow<BF> r(max(max(red[m][0], red[m][1]), max(red[m][2], red[m][3])));
        scale[m] = r.scale;
#pragma unroll
        for (int s = 0; s < NC; ++s)
        {
            const int k = (s * 256 + (int)threadIdx.x) * 8;
            if (k >= (kb + 1023) / 1024 * 1024) continue;   // zeros up to the end of the last 1024
            uint16_t e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = keep[m][s][i];
            *reinterpret_cast<uint64_t*>(&xq[m][k]) = k < kb ? r.eight(e) : 0;
        }
    }
    gm_barrier();
    while (row < a.N)
    {
        int acc[2][MM] = {};
        auto dot = [&](const gm_i4& g0, const gm_i4& g1, int c) {
#pragma unroll
            for (int m = 0; m < MM; ++m)
            {
                const gm_i4 v = *reinterpret_cast<const gm_i4*>(&xq[m][c * 1024 + lane * 16]);
                acc[0][m] = gm_dot(GmI8{}, g0, v, acc[0][m]);
                acc[1][m] = gm_dot(GmI8{}, g1, v, acc[1][m]);
            }
        };
        for (int c = 0; c < whole;)
        {
#pragma unroll
            for (int j = 0; j < U; ++j)
                if (c + j < whole) dot(f0[j], f1[j], c + j);
            c += U;
            if (c < whole) load(c);
        }
        if (kb % 1024)
        {
            const int nb = kb - whole * 1024 - lane * 16;
            dot(gm_masked<1>(w0 + whole * 1024, nb), gm_masked<1>(w1 + whole * 1024, nb), whole);
        }
        const int n = row;
        row += (int)gridDim.x * 8;
        aim();
        if (row < a.N) load(0);
#pragma unroll
        for (int m = 0; m < MM; ++m)
        {
            int s0 = acc[0][m], s1 = acc[1][m];
#pragma unroll
            for (int o = 32; o; o >>= 1) s0 += __shfl_xor(s0, o), s1 += __shfl_xor(s1, o);
            if (lane != m) continue;
            const int left = min(2, a.N - n);
            float v[4] = { (float)s0 * scale[m] * a.sb[n], (float)s1 * scale[m] * a.sb[n + left - 1], 0.f, 0.f };
            gm_put4(a.out[0], a.odt, (int64_t)m * a.ldo + n, v, left, 0);
        }
    }
}

void launch_linear_row_i8(const GmArgs& a, int bf16, hipStream_t st)
{
    const int wg = std::min((a.N + 7) / 8, LQ_WG);
    auto* kern = bf16 ? (a.M == 1 ? &linear_row_kernel<true, 1, 5> : &linear_row_kernel<true, 2, 5>)
                      : (a.M == 1 ? &linear_row_kernel<false, 1, 5> : &linear_row_kernel<false, 2, 5>);
    hipLaunchKernelGGL(kern, dim3(wg), dim3(256), 0, st, a);
}

}  // namespace gfl
