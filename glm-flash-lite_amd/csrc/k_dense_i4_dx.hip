// The gradient of a product with 4-bit weights (k_quant4.hip has their layout) with respect to its input:
// dx[m][k] = sum_n dy[m][n] w[n][k], w = (v - z) s rounded to the type of dy.
//
// The sum runs over the weight's rows. A lane's word of a row holds 8 neighbouring k, so the words of 8 rows make one value of each of 8
// MFMAs' fragments for 8 neighbouring columns: 16 lanes take a block of 128 columns, and no weight goes through LDS or memory. A weight
// costs a conversion, a multiply-add (z s, kept for a row, is finite up to scales of 2^119) and half a rounding of two; up to 64 tokens share
// it. That is what bounds 64 tokens (1.6 us a step, of which 0.8 are these and 0.4 the MFMAs), and few tokens the weight's way from memory:
// 11008 -> 4096 1 token 13.0 us, 24 16.0, 64 21.3; through weights of 16 bits in memory 45, 45 and 47.
#include "gfl_device.hpp"
#include "gfl_gemm.hpp"
#include "gfl_gemm_plan.hpp"
#include "gfl_open.hpp"
#include "gfl_quant.hpp"

namespace gfl {

// 16 TT tokens and a block of 128 columns by 8 waves, 32 rows of the weight a wave and step, over a part of the rows. The waves share
// nothing until their sums are joined in LDS.
template <typename T, int GB, bool ZERO, int TT>
__global__ __launch_bounds__(512, TT >= 2 ? 2 : 4) void q4_dx_kernel(Q4Args a)
{
    constexpr int LDR = 132;   // floats of a row of sums in LDS
    extern __shared__ __align__(16) float dx_red[];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64), lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    int tm, block, part;
    {
        // workgroups of the same weights lie 8 apart, on one XCD
        const int tall = (a.M + 16 * TT - 1) / (16 * TT), np = a.blocks * a.parts, eights = np / 8 * 8;
        int id = blockIdx.x;
        if (id < eights * tall)
        {
            const int k = id / 8;
            tm = k % tall;
            id = k / tall * 8 + id % 8;
        }
        else
        {
            id -= eights * tall;
            tm = id % tall;
            id = eights + id / tall;
        }
        // and the two blocks of a 128-byte line of the weight too
        if (id < np / 16 * 16) id = id / 16 * 16 + id % 8 * 2 + id / 8 % 2;
        block = id % a.blocks;
        part = id / a.blocks;
    }
    const int m0 = tm * 16 * TT, steps = (a.N + 31) / 32, share = (steps + a.parts - 1) / a.parts;
    const int first = part * share + wave, end = min((part + 1) * share, steps);

    // offsets from uniform addresses: a weight has up to 2^31 bytes, scales up to 2^28, a tile's rows of dy lie within 2^29
    const uint32_t stride = (uint32_t)a.blocks * 64;
    const uint8_t* q = a.q + block * 64;
    const int groups = (a.K + 128 / GB - 1) / (128 / GB);
    const uint32_t of = (uint32_t)min(block * GB + r % 4 * GB / 4, groups - 1) * (uint32_t)a.N;
    const char* dy = a.x + (int64_t)m0 * a.ldx;
    uint32_t row[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) row[t] = (uint32_t)min(t * 16 + r, a.M - 1 - m0) * (uint32_t)a.ldx;

    struct Step
    {
        uint32_t w[8];
        uint32_t s[4], z[2];
        gm_i4 dy[TT];
    } even, odd;
    // the 8 rows of lane group g in step s; at the weight's end, its last 8
    auto rows = [&](int s) { return min(min(s, end - 1) * 32 + g * 8, a.N - 8); };
    auto weights = [&](int s, Step& o) {
        const uint32_t n = (uint32_t)rows(s);
        __builtin_memcpy(o.s, static_cast<const uint16_t*>(a.scale) + (of + n), 16);
        if constexpr (ZERO) __builtin_memcpy(o.z, a.zero + (of + n), 8);
        const uint32_t at = n * stride + r * 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) __builtin_memcpy(&o.w[i], q + i * (int64_t)stride + at, 4);
    };
    auto tokens = [&](int s, Step& o) {
        const uint32_t n = (uint32_t)rows(s) * 2;
#pragma unroll
        for (int t = 0; t < TT; ++t) __builtin_memcpy(&o.dy[t], dy + (row[t] + n), 16);
    };
    gm_f4 acc[8][TT] = {};
    auto step = [&](int s, Step& o) {
        uint32_t half[2][8];
        float sc[8], off[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                half[h][i] = o.w[i] >> (4 * h) & 0x0F0F0F0F;
                asm volatile("" : "+v"(half[h][i]));   // (opaque: a byte is then one conversion, and not cut out first)
            }
            const uint16_t bits = (uint16_t)(o.s[i / 2] >> (i % 2 * 16));
            sc[i] = a.scale_bf ? q_val<true>(bits) : q_val<false>(bits);
            off[i] = (ZERO ? -(float)(o.z[i / 4] >> (i % 4 * 8) & 255) : -8.0f) * sc[i];
            asm volatile("" : "+v"(off[i]));   // (and z s is kept for the row)
        }
        if (s * 32 + 32 > a.N)
        {
            // rows before this lane group's are another's, or there are none left
            const int over = s * 32 + g * 8 - (a.N - 8);
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o.dy[t][i] = over > 2 * i + 1 ? 0 : over > 2 * i ? o.dy[t][i] & (int)0xFFFF0000 : o.dy[t][i];
        }
        weights(s + 16, o);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int b = 0; b < 4; ++b)
            {
                gm_i4 f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
                    typedef typename T::elem pair __attribute__((ext_vector_type(2)));
                    float v[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k)   // exact: one rounding, of at most 13 bits
                        v[k] = fmaf((float)(half[h][2 * i + k] >> (8 * b) & 255), sc[2 * i + k], off[2 * i + k]);
                    const pair p = { static_cast<typename T::elem>(v[0]), static_cast<typename T::elem>(v[1]) };
                    f[i] = __builtin_bit_cast(int, p);
                }
                const int k = h * 2 + b % 2 * 4 + b / 2;   // the column of a word's byte
#pragma unroll
                for (int t = 0; t < TT; ++t) acc[k][t] = T::mfma(o.dy[t], f, acc[k][t]);
            }
        tokens(s + 16, o);
    };
    weights(first, even);
    tokens(first, even);
    weights(first + 8, odd);
    tokens(first + 8, odd);
    int s = first;
    for (; s + 8 < end; s += 16)
    {
        step(s, even);
        step(s + 8, odd);
    }
    if (s < end) step(s, even);

    float* mine = dx_red + wave * 16 * LDR;
    const int m = threadIdx.x / 32, c = threadIdx.x % 32 * 4;
#pragma unroll
    for (int t = 0; t < TT; ++t)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            float* p = mine + (g * 4 + e) * LDR + r % 4 * 32 + r / 4 * 8;
            *reinterpret_cast<gm_f4*>(p) = gm_f4{ acc[0][t][e], acc[1][t][e], acc[2][t][e], acc[3][t][e] };
            *reinterpret_cast<gm_f4*>(p + 4) = gm_f4{ acc[4][t][e], acc[5][t][e], acc[6][t][e], acc[7][t][e] };
        }
        gm_barrier();
        gm_f4 sum = {};
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += *reinterpret_cast<const gm_f4*>(dx_red + (w * 16 + m) * LDR + c);
        gm_barrier();
        const int token = m0 + t * 16 + m, col = block * 128 + c;
        if (token >= a.M || col >= a.K) continue;   // (the barriers are behind)
        if (a.parts > 1) *reinterpret_cast<gm_f4*>(a.part + ((int64_t)part * a.M + token) * a.ldp + col) = sum;
        else
        {
            const float v[4] = { sum[0], sum[1], sum[2], sum[3] };
            gm_put4(a.out, a.odt, (int64_t)token * a.ldo + col, v, a.K - col, 0);
        }
    }
}

template <typename T, int GB, bool ZERO, int TT>
static void q4_dx_go(const Q4Args& a, hipStream_t st)
{
    constexpr int lds = 8 * 16 * 132 * 4;
    auto* kern = &q4_dx_kernel<T, GB, ZERO, TT>;
    static std::atomic<uint64_t> opened{ 0 };
    gm_open(reinterpret_cast<const void*>(kern), lds, opened);
    const int64_t wg = (int64_t)((a.M + 16 * TT - 1) / (16 * TT)) * a.blocks * a.parts;
    hipLaunchKernelGGL(kern, dim3((unsigned)wg), dim3(512), lds, st, a);
    if (a.parts == 1) return;
    GmArgs j;
    j.M = a.M; j.N = a.K;
    j.out[0] = a.out; j.ldo = a.ldo; j.odt = a.odt;
    const int64_t n = (int64_t)a.M * ((a.K + 3) / 4);
    hipLaunchKernelGGL((gm_join_kernel<T, false, EP_OUT>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, j, (const void*)a.part,
                       a.ldp, a.parts);
}

template <typename T, bool ZERO>
static void q4_dx_group(const Q4Args& a, int tt, hipStream_t st)
{
    auto by = [&](auto gb) {
        constexpr int GB = decltype(gb)::value;
        (tt == 1 ? &q4_dx_go<T, GB, ZERO, 1> : tt == 2 ? &q4_dx_go<T, GB, ZERO, 2> : &q4_dx_go<T, GB, ZERO, 4>)(a, st);
    };
    if (a.group == 32) by(std::integral_constant<int, 4>{});
    else if (a.group == 64) by(std::integral_constant<int, 2>{});
    else by(std::integral_constant<int, 1>{});
}

void launch_linear_i4_dx(Q4Args& a, int bf16, void* ws, hipStream_t st)
{
    const Q4DxPlan p = q4_dx_plan(a.M, a.N, a.K);
    a.parts = p.parts;
    a.part = static_cast<float*>(ws);
    a.ldp = p.ldp;
    if (bf16) (a.zero ? &q4_dx_group<GmBF16, true> : &q4_dx_group<GmBF16, false>)(a, p.tt, st);
    else (a.zero ? &q4_dx_group<GmF16, true> : &q4_dx_group<GmF16, false>)(a, p.tt, st);
}

}  // namespace gfl
