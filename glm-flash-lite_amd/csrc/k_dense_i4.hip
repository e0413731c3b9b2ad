// Products with 4-bit weights (k_quant4.hip has their layout): y[m][n] = sum over groups of s[g][n] * sum_k x[m][k] (v[n][k] - z[g][n]).
//
// The values go into the MFMAs as they are: 16 + v in the type of x is one shift and one mask and-or for two of them (v in the
// mantissa's upper bits, exact), and a second MFMA by ones sums the tokens' inputs, so that a group adds
// s * (sum x (16 + v) - (16 + z) sum x) to the fp32 sums, with no rounding of a weight.
#include "gfl_device.hpp"
#include "gfl_gemm.hpp"
#include "gfl_gemm_plan.hpp"
#include "gfl_open.hpp"
#include "gfl_quant.hpp"

#include <algorithm>

namespace gfl {

// a fragment of which the first n values (0..7; else as it is) are dropped and zeros follow
__device__ __forceinline__ gm_i4 q4_shift(gm_i4 v, int n)
{
    n = n > 0 && n < 8 ? n : 0;
    const bool four = n & 4, two = n & 2, one = n & 1;
    v = gm_i4{ four ? v[2] : v[0], four ? v[3] : v[1], four ? 0 : v[2], four ? 0 : v[3] };
    v = gm_i4{ two ? v[1] : v[0], two ? v[2] : v[1], two ? v[3] : v[2], two ? 0 : v[3] };
    auto half = [](int hi, int lo) { return (int)(((uint32_t)hi << 16) | ((uint32_t)lo >> 16)); };
    return one ? gm_i4{ half(v[1], v[0]), half(v[2], v[1]), half(v[3], v[2]), half(0, v[3]) } : v;
}

// 16 + v of a word's 8 values. The constants are asked into registers of their own (opaque, so that they stay there): a shift and
// a v_and_or_b32 for two values, where literals take a shift, an and and an or.
template <typename T>
struct Q4Frag
{
    static constexpr bool BF = std::is_same_v<T, GmBF16>;
    uint32_t mask = BF ? 0x00780078 : 0x03C003C0, off = BF ? 0x41804180 : 0x4C004C00;
    __device__ __forceinline__ Q4Frag() { asm volatile("" : "+s"(mask), "+v"(off)); }
    __device__ __forceinline__ gm_i4 operator()(uint32_t w) const
    {
        if constexpr (BF) return gm_i4{ (int)((w << 3 & mask) | off), (int)((w >> 1 & mask) | off), (int)((w >> 5 & mask) | off), (int)((w >> 9 & mask) | off) };
        else return gm_i4{ (int)((w << 6 & mask) | off), (int)((w << 2 & mask) | off), (int)((w >> 2 & mask) | off), (int)((w >> 6 & mask) | off) };
    }
};
__device__ __forceinline__ gm_i4 q4_ones(GmBF16) { return gm_i4{ 0x3F803F80, 0x3F803F80, 0x3F803F80, 0x3F803F80 }; }
__device__ __forceinline__ gm_i4 q4_ones(GmF16) { return gm_i4{ 0x3C003C00, 0x3C003C00, 0x3C003C00, 0x3C003C00 }; }

// Up to 16 tokens, the inputs of which fit the LDS. A tile of 16 channels is formed by KS waves that share its inputs out among
// themselves (ks has the blocks of 128 from ks * share on) and join their sums in LDS; a workgroup of NW waves is at NW / KS tiles at
// a time. The tokens are put into LDS once for all the channels that the workgroup takes; a wave's weights come straight from memory,
// U blocks of them while it is at the U before. GB: groups of a block.
//
// Loads return in order, and what is loaded first is needed first: the tokens, then scales, then weights.
//
// Bound by the weights' bytes from 65536 channels on (9 tokens of 4096 29 us, 4.8 TB/s); one token of 5120 -> 5120 takes 6.0 us, 2.2 of
// them a launch's, 2.8 its bytes.
template <typename T, int GB, bool ZERO, int U, int KS, int NW>
__global__ __launch_bounds__(NW * 64) void q4_few_kernel(Q4Args a)
{
    constexpr int WG = 4 / GB, G = 128 / GB, NS = (U * GB + 3) / 4, NP = 4;   // words of a group, its size, loads of scales, of tokens
    extern __shared__ __align__(16) char q4_lds[];   // tokens, rows of blocks * 256 + 16 bytes (which spreads them over the banks)
    __shared__ float red[KS > 1 ? 2 : 1][KS > 1 ? NW : 1][4][64];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64), lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    const int groups = (a.K + G - 1) / G, tiles = (a.N + 15) / 16, last = a.blocks - 1;
    const int share = (a.blocks + KS - 1) / KS, c0 = wave % KS * share, batches = (share + U - 1) / U;
    const int m0 = blockIdx.y * 16, M = min(a.M - m0, 16);
    const int pieces = a.blocks * 16, total = pieces * M, ldr = a.blocks * 256 + 16;   // of 16 bytes
    const char* xg = a.x + (int64_t)m0 * a.ldx;
    const Q4Frag<T> frag;

    gm_i4 w[U], wn[U], xp[NP];
    uint16_t s[NS], sn[NS];
    uint8_t z[NS], zn[NS];
    // the blocks from c on of a tile; what lies past the wave's share is loaded from its end (and has no scale)
    const int end = min(c0 + share, a.blocks);
    auto load = [&](int tile, int c, gm_i4 (&v)[U], uint16_t (&sc)[NS], uint8_t (&zr)[NS]) {
        const int n = min(tile * 16 + r, a.N - 1);
        // lane group g has the scale of slot 4 l + g: of group slot % GB of the wave's block slot / GB
#pragma unroll
        for (int l = 0; l < NS; ++l)
        {
            const uint32_t at = (uint32_t)min(c * GB + 4 * l + g, groups - 1) * a.N + n;
            sc[l] = static_cast<const uint16_t*>(a.scale)[at];
            if constexpr (ZERO) zr[l] = a.zero[at];
        }
        const uint32_t row = (uint32_t)n * a.blocks * 64 + g * 16;   // (a weight has up to 2^31 bytes)
#pragma unroll
        for (int i = 0; i < U; ++i) __builtin_memcpy(&v[i], a.q + (row + min(c + i, last) * 64), 16);
    };
    // piece p of the tokens: 8 inputs of token p / pieces
    auto token_at = [&](int p, int& m, int& k) {
        m = (int)__umulhi((uint32_t)p, a.magic);
        k = (p - m * pieces) * 8;
    };
    auto fetch = [&](int p0) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
        {
            int m, k;
            token_at(min(p0 + i * NW * 64, total - 1), m, k);
            __builtin_memcpy(&xp[i], xg + ((uint32_t)m * (uint32_t)a.ldx + min(k, a.K - 8) * 2), 16);
        }
    };
    auto keep = [&](int p0) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
        {
            const int p = p0 + i * NW * 64;
            int m, k;
            token_at(p, m, k);
            if (p < total) *reinterpret_cast<gm_i4*>(q4_lds + m * ldr + k * 2) = k < a.K ? xp[i] : gm_i4{ 0, 0, 0, 0 };
        }
    };
    int tile = blockIdx.x * (NW / KS) + wave / KS;
    const int step = gridDim.x * (NW / KS);
    if (a.K % 8 == 0)
    {
        fetch(threadIdx.x);
        load(tile, c0, w, s, z);
        keep(threadIdx.x);
        for (int p = threadIdx.x + NP * NW * 64; p < total; p += NP * NW * 64)
        {
            fetch(p);
            keep(p);
        }
    }
    else
    {
        load(tile, c0, w, s, z);
        for (int p = threadIdx.x; p < total; p += NW * 64)
        {
            int m, k;
            token_at(p, m, k);
            *reinterpret_cast<gm_i4*>(q4_lds + m * ldr + k * 2) = gm_masked<2>(xg + m * a.ldx + k * 2, (a.K - k) * 2);
        }
    }
    gm_barrier();   // (waits for LDS alone: the weights stay under way)
    const char* x = q4_lds + min(r, M - 1) * ldr + g * 16;
    // whole rounds of the workgroup, so that its waves meet as often as each other
    for (int it = 0, first = blockIdx.x * (NW / KS); first < tiles; ++it, first += step, tile += step)
    {
        gm_f4 acc = {};
        for (int b = 0; b < batches; ++b)
        {
            const int c = c0 + b * U;
            load(b + 1 < batches ? tile : tile + step, b + 1 < batches ? c + U : c0, wn, sn, zn);
            float sf[NS], zf[NS];
#pragma unroll
            for (int l = 0; l < NS; ++l)
            {
                sf[l] = c * GB + 4 * l + g >= min(groups, end * GB) ? 0.0f : a.scale_bf ? q_val<true>(s[l]) : q_val<false>(s[l]);
                if constexpr (ZERO) zf[l] = 16.0f + (float)z[l];
            }
#pragma unroll
            for (int i = 0; i < U; ++i)
            {
                const char* xb = x + min(c + i, last) * 256;
#pragma unroll
                for (int q = 0; q < GB; ++q)
                {
                    gm_f4 sum = {}, xs = {};
#pragma unroll
                    for (int j = q * WG; j < (q + 1) * WG; ++j)
                    {
                        const gm_i4 f = *reinterpret_cast<const gm_i4*>(xb + j * 64);
                        sum = T::mfma(f, frag((uint32_t)w[i][j]), sum);
                        xs = T::mfma(f, q4_ones(T{}), xs);
                    }
                    const int slot = i * GB + q;
                    const float sv = __shfl(sf[slot / 4], slot % 4 * 16 + r);
                    const float zv = ZERO ? __shfl(zf[slot / 4], slot % 4 * 16 + r) : 24.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[e] = fmaf(sv, fmaf(-zv, xs[e], sum[e]), acc[e]);
                }
            }
#pragma unroll
            for (int i = 0; i < U; ++i) w[i] = wn[i];
#pragma unroll
            for (int l = 0; l < NS; ++l) s[l] = sn[l], z[l] = zn[l];
        }
        if constexpr (KS == 1)
        {
            const int n = tile * 16 + r;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (g * 4 + e < M && n < a.N) gm_put1(a.out, a.odt, (int64_t)(m0 + g * 4 + e) * a.ldo + n, acc[e]);
        }
        else
        {
#pragma unroll
            for (int e = 0; e < 4; ++e) red[it % 2][wave][e][lane] = acc[e];
            gm_barrier();
            for (int o = threadIdx.x % (KS * 64); o < 256; o += KS * 64)
            {
                const int w0 = wave / KS * KS, e = o / 64, l = o % 64, m = l / 16 * 4 + e, n = tile * 16 + l % 16;
                float v = 0.0f;
#pragma unroll
                for (int k = 0; k < KS; ++k) v += red[it % 2][w0 + k][e][l];
                if (m < M && n < a.N) gm_put1(a.out, a.odt, (int64_t)(m0 + m) * a.ldo + n, v);
            }
        }
    }
}

template <typename T, int GB, bool ZERO, int U, int KS>
static void q4_few_go(Q4Args a, hipStream_t st)
{
    constexpr int NW = 8;
    auto* kern = &q4_few_kernel<T, GB, ZERO, U, KS, NW>;
    static std::atomic<uint64_t> opened{ 0 };
    gm_open(reinterpret_cast<const void*>(kern), Q4_TOKENS, opened);
    a.magic = (uint32_t)((1ull << 32) / (a.blocks * 16) + 1);
    const int lds = std::min(a.M, 16) * (a.blocks * 256 + 16), tiles = (a.N + 15) / 16, wg = (tiles + NW / KS - 1) / (NW / KS);
    hipLaunchKernelGGL(kern, dim3(std::min(wg, 256 * std::min(LDS_LIMIT / (lds + (KS > 1 ? NW * 2048 : 0)), 3)), (a.M + 15) / 16),
                       dim3(NW * 64), lds, st, a);
}

// Two blocks on their way while a wave is at two, one where a share of few blocks would be padded: us, U = 1, 2, 3 and 4, 5120 -> 5120 1
// token (shares of 10) 6.7, 6.4, 7.1 and 7.3, 4072 -> 11007 5 tokens (16) 10.5, 9.9, 11.4 and 10.6, 4096 -> 65536 9 tokens (32) 39.9,
// 34.7, 36.5 and 35.0; shares of 3, 3000 -> 3000 3 tokens, 4.3 and 4.9 by 1 and 2.
template <typename T, int GB, bool ZERO, int KS>
static void q4_few_u(const Q4Args& a, hipStream_t st)
{
    const int share = (a.blocks + KS - 1) / KS;
    if (share % 2 == 0 || share > 6) q4_few_go<T, GB, ZERO, 2, KS>(a, st);
    else q4_few_go<T, GB, ZERO, 1, KS>(a, st);
}

// Waves to a tile: the fewer, the longer a wave's own chain; the more, the more workgroups beyond a CU's. us by 1, 2, 4 and 8 waves, 1 and 8
// tokens of 5120:
//    256 tiles  14.3 9.0 6.3 5.0, 16.0 10.6 7.7 6.6     319  14.5 9.1 6.5 6.7, 16.1 10.7 7.9 8.8     320  14.5 9.2 6.4 6.8, 16.1 10.7 7.8 8.9
//    512        14.5 9.3 6.7 7.2, 16.1 10.8 8.3 9.3     639  14.6 9.3 9.0 8.8, 16.4 11.2 11.6 11.3   640  14.6 9.3 9.1 8.7, 16.3 11.1 11.7 11.5
//   1024        14.6 9.6 9.3 10.3, 16.6 11.6 11.8 14.0  1280  14.7 14.2 12.5 12.3, 16.8 18.1 15.1 16.2  2048  16.9 15.7 16.5 19.6, 18.9 19.3 19.8 25.6
// and 4096 -> 65536 (4096 tiles) 9 tokens 34, 39, 39, 40. Of 2048 inputs the order is the same: 256 tiles 7.0 5.0 3.9 3.4, 1280 7.6 7.6 7.2
// 6.9. Between the edges the best is missed by up to 10% from 257 to 319 tiles, and by 15% from 1280 to some 2000.
template <typename T, int GB, bool ZERO>
static void q4_few(const Q4Args& a, hipStream_t st)
{
    const int tiles = (a.N + 15) / 16;
    (tiles >= 1280 ? &q4_few_u<T, GB, ZERO, 1> : tiles >= 640 ? &q4_few_u<T, GB, ZERO, 2> : tiles >= 320 ? &q4_few_u<T, GB, ZERO, 4>
                                                                                         : &q4_few_u<T, GB, ZERO, 8>)(a, st);
}

// More tokens, or tokens that do not fit the LDS whole: 16 TT tokens and 128 NT channels by a workgroup of 8 waves, 16 NT channels each,
// over a part of the inputs. Two blocks of 128 inputs a step: the tokens' inputs of a step lie in LDS, the next step's on their way
// to registers like the wave's weights, which go from memory into its MFMAs. The sums of the tokens' inputs by groups, without
// which a group's 16 and zero point cannot leave its sums, are formed where the tokens are put into LDS, once for all channels, and
// enter as the MFMAs' first accumulators: a group then costs one multiply-add a result.
//
// A step of 64 tokens and 256 channels takes 2.0 us without its loads and the tokens' way to LDS, 2.7 with them (256 tokens of 5120 ->
// 12288 57 us): MFMAs, LDS reads and VALU take some 0.85 each, and two waves a SIMD overlap them little. Loads two steps ahead
// instead of one changed nothing. In 50 tokens of 12288 -> 5120 (23 us and 5 to join 12 parts) most is the ends of 4 steps: 6 parts
// 36 us, tiles of 128 channels in 6 parts 30.
template <typename T, int GB, bool ZERO, int TT, int NT>
__global__ __launch_bounds__(512, TT * NT >= 8 ? 2 : 4) void q4_tile_kernel(Q4Args a)
{
    constexpr int WG = 4 / GB, G = 128 / GB, SG = 2 * GB, NS = (NT * SG + 3) / 4;   // words of a group, its size, groups of a step
    constexpr int LDR = 528, XB = TT * 16 * LDR, SB = SG * TT * 16 * 4;             // bytes of a token's row, of a step's tokens, sums
    extern __shared__ __align__(16) char q4_lds[];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64), lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    const int groups = (a.K + G - 1) / G, last = a.blocks - 1;
    int tm, tn, part;
    {
        // workgroups of the same weights lie 8 apart, on one XCD
        const int wide = (a.N + 128 * NT - 1) / (128 * NT), tall = (a.M + 16 * TT - 1) / (16 * TT), np = wide * a.parts;
        int id = blockIdx.x;
        const int eights = np / 8 * 8;
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
        tn = id % wide;
        part = id / wide;
    }
    const int m0 = tm * 16 * TT, nw = tn * 128 * NT + wave * 16 * NT;   // the wave's first channel
    const int share = ((a.blocks + a.parts - 1) / a.parts + 1) / 2 * 2, b0 = part * share, end = min(b0 + share, a.blocks);
    const Q4Frag<T> frag;

    // all offsets from uniform addresses: a tile's rows of x lie within 2^29 bytes, a weight has up to 2^31, scales up to 2^28
    const char* xg = a.x + (int64_t)m0 * a.ldx;
    uint32_t wo[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) wo[t] = (uint32_t)min(nw + t * 16 + r, a.N - 1) * a.blocks * 64 + g * 16;
    uint16_t s[NS], s1[NS];
    uint8_t z[NS], z1[NS];
    gm_i4 w[NT][2], w1[NT][2], xv[TT];
    // lane group g has the scale of slot 4 l + g: of channel tile slot / SG and group slot % SG of the step
    auto scales = [&](int b) {
#pragma unroll
        for (int l = 0; l < NS; ++l)
        {
            const int n = min(nw + min((4 * l + g) / SG, NT - 1) * 16 + r, a.N - 1);
            const uint32_t at = (uint32_t)min(b * GB + (4 * l + g) % SG, groups - 1) * a.N + n;
            s1[l] = static_cast<const uint16_t*>(a.scale)[at];
            if constexpr (ZERO) z1[l] = a.zero[at];
        }
    };
    auto weights = [&](int b) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) __builtin_memcpy(&w1[t][i], a.q + (wo[t] + min(b + i, last) * 64), 16);
    };
    // a thread's pieces of the tokens: 8 inputs of one token each, 32 pieces a token. K >= 8: a piece that ends past the row is
    // loaded from the row's last 8 inputs and shifted
    const int col = threadIdx.x % 32, row = threadIdx.x / 32;
    uint32_t xo[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) xo[t] = (uint32_t)min(row + 16 * t, a.M - 1 - m0) * (uint32_t)a.ldx;
    auto fetch = [&](int b) {
        const uint32_t k = (uint32_t)min(b * 128 + col * 8, a.K - 8) * 2;
#pragma unroll
        for (int t = 0; t < TT; ++t) __builtin_memcpy(&xv[t], xg + (xo[t] + k), 16);
    };
    auto keep = [&](int b, int buf) {
        const int k = b * 128 + col * 8, over = k + 8 - a.K;
        if (a.K % 8)
#pragma unroll
            for (int t = 0; t < TT; ++t) xv[t] = q4_shift(xv[t], over);
        const bool there = k < a.K;
        char* xl = q4_lds + buf * (XB + SB);
        float* sl = reinterpret_cast<float*>(xl + XB);
#pragma unroll
        for (int t = 0; t < TT; ++t)
        {
            if (!there) xv[t] = gm_i4{ 0, 0, 0, 0 };
            *reinterpret_cast<gm_i4*>(xl + (row + 16 * t) * LDR + col * 16) = xv[t];
            float v = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const int u = xv[t][i];
                if constexpr (Q4Frag<T>::BF) v += __int_as_float(u << 16) + __int_as_float(u & 0xFFFF0000);
                else
                {
                    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                    const h2 p = __builtin_bit_cast(h2, u);
                    v += (float)p[0] + (float)p[1];
                }
            }
            v += lane_xor<1>(v);
            v += lane_xor<2>(v);
            if constexpr (GB <= 2) v += lane_xor<4>(v);
            if constexpr (GB == 1) v += lane_xor<8>(v);
            if (col % (G / 8) == 0) sl[col / (G / 8) * (TT * 16) + row + 16 * t] = ZERO ? -v : -24.0f * v;
        }
    };

    gm_f4 acc[NT][TT] = {};
    scales(b0);
    fetch(b0);
    weights(b0);
    keep(b0, 0);
    gm_barrier();
    for (int b = b0, it = 0; b < end; b += 2, ++it)
    {
#pragma unroll
        for (int l = 0; l < NS; ++l) s[l] = s1[l], z[l] = z1[l];
#pragma unroll
        for (int t = 0; t < NT; ++t) w[t][0] = w1[t][0], w[t][1] = w1[t][1];
        const bool more = b + 2 < end;
        const int next = more ? b + 2 : b;
        scales(next);
        fetch(next);
        weights(next);
        __builtin_amdgcn_sched_barrier(0);   // the compiler would issue them half a step later (2% of 16 to 64 tokens)
        float sf[NS], zf[NS];
#pragma unroll
        for (int l = 0; l < NS; ++l)
        {
            const int q = b * GB + (4 * l + g) % SG;
            sf[l] = q >= min(groups, end * GB) ? 0.0f : a.scale_bf ? q_val<true>(s[l]) : q_val<false>(s[l]);
            if constexpr (ZERO) zf[l] = 16.0f + (float)z[l];
        }
        const char* xl = q4_lds + it % 2 * (XB + SB);
        const float* sl = reinterpret_cast<const float*>(xl + XB);
        const char* xr = xl + r * LDR + g * 16;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < GB; ++q)
            {
                gm_f4 sum[NT][TT], xs[TT];
                float sv[NT], zv[NT];
#pragma unroll
                for (int t = 0; t < TT; ++t) xs[t] = *reinterpret_cast<const gm_f4*>(sl + (i * GB + q) * (TT * 16) + t * 16 + g * 4);
#pragma unroll
                for (int n = 0; n < NT; ++n)
                {
                    const int slot = n * SG + i * GB + q;
                    sv[n] = __shfl(sf[slot / 4], slot % 4 * 16 + r);
                    zv[n] = ZERO ? __shfl(zf[slot / 4], slot % 4 * 16 + r) : 1.0f;
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int t = 0; t < TT; ++t)
                    {
                        sum[n][t] = xs[t];
                        if constexpr (ZERO)
#pragma unroll
                            for (int e = 0; e < 4; ++e) sum[n][t][e] *= zv[n];
                    }
#pragma unroll
                for (int j = q * WG; j < (q + 1) * WG; ++j)
                {
                    gm_i4 f[TT];
#pragma unroll
                    for (int t = 0; t < TT; ++t) f[t] = *reinterpret_cast<const gm_i4*>(xr + t * 16 * LDR + i * 256 + j * 64);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                    {
                        const gm_i4 v = frag((uint32_t)w[n][i][j]);
#pragma unroll
                        for (int t = 0; t < TT; ++t) sum[n][t] = T::mfma(f[t], v, sum[n][t]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int t = 0; t < TT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[n][t][e] = fmaf(sv[n], sum[n][t][e], acc[n][t][e]);
                // here and not later: all groups' MFMAs first, which is how the compiler would have it, take more registers than there are
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int t = 0; t < TT; ++t) asm volatile("" : "+v"(acc[n][t]));
            }
        if (more) keep(next, 1 - it % 2);
        gm_barrier();
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
    {
        const int c = nw + n * 16 + r;
        if (c >= a.N) continue;
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                const int m = m0 + t * 16 + g * 4 + e;
                if (m >= a.M) continue;
                if (a.parts > 1) a.part[((int64_t)part * a.M + m) * a.ldp + c] = acc[n][t][e];
                else gm_put1(a.out, a.odt, (int64_t)m * a.ldo + c, acc[n][t][e]);
            }
    }
}

template <typename T, int GB, bool ZERO, int TT, int NT>
static void q4_tile_go(const Q4Args& a, hipStream_t st)
{
    constexpr int lds = 2 * (TT * 16 * 528 + 2 * GB * TT * 16 * 4);
    auto* kern = &q4_tile_kernel<T, GB, ZERO, TT, NT>;
    if constexpr (lds > 65536)
    {
        static std::atomic<uint64_t> opened{ 0 };
        gm_open(reinterpret_cast<const void*>(kern), lds, opened);
    }
    const int64_t wg = (int64_t)((a.N + 128 * NT - 1) / (128 * NT)) * ((a.M + 16 * TT - 1) / (16 * TT)) * a.parts;
    hipLaunchKernelGGL(kern, dim3((unsigned)wg), dim3(512), lds, st, a);
    if (a.parts == 1) return;
    GmArgs j;
    j.M = a.M; j.N = a.N;
    j.out[0] = a.out; j.ldo = a.ldo; j.odt = a.odt;
    const int64_t n = (int64_t)a.M * ((a.N + 3) / 4);
    hipLaunchKernelGGL((gm_join_kernel<T, false, EP_OUT>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, j, (const void*)a.part,
                       a.ldp, a.parts);
}

template <typename T, int GB, bool ZERO>
static void q4_tiles(const Q4Args& a, const Q4Plan& p, hipStream_t st)
{
    (p.tt == 1 ? p.nt == 1 ? &q4_tile_go<T, GB, ZERO, 1, 1> : &q4_tile_go<T, GB, ZERO, 1, 2>
     : p.tt == 2 ? p.nt == 1 ? &q4_tile_go<T, GB, ZERO, 2, 1> : &q4_tile_go<T, GB, ZERO, 2, 2>
     : p.nt == 1 ? &q4_tile_go<T, GB, ZERO, 4, 1> : &q4_tile_go<T, GB, ZERO, 4, 2>)(a, st);
}

template <typename T, int GB, bool ZERO>
static void q4_run(Q4Args& a, void* ws, hipStream_t st)
{
    const Q4Plan p = q4_plan(a.M, a.N, a.K);
    // a launch has fewer than 2^32 threads, and fewer than 2^16 workgroups in y: the rows in as many launches as it takes
    const int64_t wide = p.few ? 768 : (int64_t)((a.N + 128 * p.nt - 1) / (128 * p.nt)) * p.parts;
    const int tt = p.few ? 1 : p.tt, M = a.M;
    const int rows = (int)std::max<int64_t>(1, std::min<int64_t>((1 << 22) / wide, 65535)) * 16 * tt;
    for (int m = 0; m < M; m += rows)
    {
        Q4Args b = a;
        b.x += (int64_t)m * a.ldx;
        b.M = std::min(rows, M - m);
        b.out = static_cast<char*>(a.out) + (int64_t)m * a.ldo * (a.odt == 2 ? 4 : 2);
        b.parts = p.parts;
        b.part = static_cast<float*>(ws);
        b.ldp = p.ldp;
        if (p.few) q4_few<T, GB, ZERO>(b, st);
        else q4_tiles<T, GB, ZERO>(b, p, st);
    }
}

template <typename T, bool ZERO>
static void q4_group(Q4Args& a, void* ws, hipStream_t st)
{
    (a.group == 32 ? &q4_run<T, 4, ZERO> : a.group == 64 ? &q4_run<T, 2, ZERO> : &q4_run<T, 1, ZERO>)(a, ws, st);
}

void launch_linear_i4(Q4Args& a, int bf16, void* ws, hipStream_t st)
{
    if (bf16) (a.zero ? &q4_group<GmBF16, true> : &q4_group<GmBF16, false>)(a, ws, st);
    else (a.zero ? &q4_group<GmF16, true> : &q4_group<GmF16, false>)(a, ws, st);
}

}  // namespace gfl
