// The tile GEMM of the dense operators (gated feed-forward block and its gradients, 8-bit integer product):
//   D[m][n] = sum_k A(m, k) * B(n, k), in fp32 (f16, bf16 inputs) or int32 (i8).
//
// A workgroup of WM x WN waves forms a TM x TN tile over K steps of SB = 128 or 64 bytes a row (128: 64 16-bit elements, 128
// of i8). Each operand is stored either with K contiguous ("KC": [rows][K], as activations and nn.Linear weights are) or
// with K as the rows ("KS": [K][cols], the transposed products of the gradients):
//   KC tiles lie in LDS as [rows][SB / 16 chunks of 16 bytes], chunk c of row r at place c ^ kc_swz(r), which spreads 16
//   neighbouring rows over all banks; a fragment is one ds_read_b128 per lane;
//   KS tiles (16-bit types) lie as [k][cols], chunk c of row k at place c ^ ks_swz(k); a fragment is two
//   ds_read_b64_tr_b16, which hand lane i of each 16 the 4 k values of column i.
// MFMA operands are (B rows, A rows), so that a lane's 4 accumulators are 4 neighbouring n of one m: vector stores.
//
// AL = 1 (rows start at multiples of 4 bytes) loads tiles by LDS-direct buffer loads, NST - 1 steps ahead; rows past
// the matrix are clamped to its last (their results are not stored), k past the end is read as zero through the
// buffer's bounds. Where rows end inside a chunk of 16 bytes (GmArgs::ragged) the last K step, whose chunks may reach past
// the matrix, goes through registers, masked per element: what other steps read past a row is the next row's, in
// columns that are not stored. AL = 0 takes any strides and alignment: every chunk goes through registers.
#pragma once
#include "gfl_internal.hpp"

#include <type_traits>
#include <utility>

namespace gfl {

typedef __attribute__((address_space(3))) void gm_lds_void;
typedef int gm_i4 __attribute__((ext_vector_type(4)));
typedef float gm_f4 __attribute__((ext_vector_type(4)));
typedef _Float16 gm_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 gm_b8 __attribute__((ext_vector_type(8)));
typedef short gm_s4 __attribute__((ext_vector_type(4)));

struct GmF16
{
    typedef _Float16 elem;
    typedef gm_f4 acc;
    typedef float scalar;
    static __device__ __forceinline__ acc mfma(gm_i4 a, gm_i4 b, acc c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gm_h8, a), __builtin_bit_cast(gm_h8, b), c, 0, 0,
                                                      0);
    }
    static __device__ __forceinline__ void mfma_agpr(gm_i4 a, gm_i4 b, acc& c)
    {
        asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    }
};
struct GmBF16
{
    typedef __bf16 elem;
    typedef gm_f4 acc;
    typedef float scalar;
    static __device__ __forceinline__ acc mfma(gm_i4 a, gm_i4 b, acc c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gm_b8, a), __builtin_bit_cast(gm_b8, b), c, 0,
                                                       0, 0);
    }
    static __device__ __forceinline__ void mfma_agpr(gm_i4 a, gm_i4 b, acc& c)
    {
        asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    }
};
struct GmI8
{
    typedef int8_t elem;
    typedef gm_i4 acc;
    typedef int scalar;
    static __device__ __forceinline__ acc mfma(gm_i4 a, gm_i4 b, acc c)
    {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ void mfma_agpr(gm_i4 a, gm_i4 b, acc& c)
    {
        asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    }
};

template <int N>
__device__ __forceinline__ void gm_wait_vmcnt()
{
    static_assert(N <= 63, "vmcnt has 6 bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void gm_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ const char* gm_uniform(const char* p)
{
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
    return reinterpret_cast<const char*>(((uint64_t)hi << 32) | lo);
}

// buffer descriptor of 2 GiB from p on (uniform)
__device__ __forceinline__ gm_i4 gm_rsrc(const char* p, int bytes = 0x7FFFFFFF)
{
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    return gm_i4{ __builtin_amdgcn_readfirstlane((int)(uint32_t)v), __builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32) & 0xFFFF),
                  __builtin_amdgcn_readfirstlane(bytes), 0x00020000 };
}
// LDS-direct load: lane l's 16 bytes at byte offset v of the buffer go to LDS address lds + 16 l (lds the same for the wave). In asm, because
// after the builtin the compiler waits for all outstanding loads before each ds_read_b64_tr (it takes that builtin for a possible
// write to the loads' LDS), which leaves nothing in flight; it holds no result register, and the waits for it are explicit
// everywhere. An s_nop between the write of M0 and its use.
__device__ __forceinline__ int gm_lds_at(char* lds) { return (int)(uint32_t)reinterpret_cast<uintptr_t>((gm_lds_void*)lds); }
__device__ __forceinline__ void gm_load_lds(gm_i4 r, int lds, uint32_t v)
{
    const int at = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(at), "v"(v), "s"(r) : "memory", "m0");
}

constexpr uint32_t GM_OUT = 0x80000000u;   // a lane offset past every buffer: reads as zero

// the 16 bytes at p of which the first nb (a multiple of ES, at most 16; may be <= 0) exist; the rest is zero
template <int ES>
__device__ __forceinline__ gm_i4 gm_masked(const char* p, int nb)
{
    gm_i4 r = { 0, 0, 0, 0 };
    if (nb >= 16)
    {
        __builtin_memcpy(&r, p, 16);
        return r;
    }
    uint32_t w[4] = { 0, 0, 0, 0 };
#pragma unroll
    for (int i = 0; i < 16 / ES; ++i)
        if (i * ES < nb)
        {
            const uint32_t e = ES == 2 ? (uint32_t)*reinterpret_cast<const uint16_t*>(p + i * ES)
                                       : (uint32_t)*reinterpret_cast<const uint8_t*>(p + i * ES);
            w[i * ES / 4] |= e << (i * ES % 4 * 8);
        }
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (int)w[i];
    return r;
}

template <int CH>
__device__ __forceinline__ int gm_kc_swz(int r)
{
    return CH == 8 ? (r >> 1) & 7 : (r >> 1) & 3;
}
__device__ __forceinline__ int gm_ks_swz(int k, int chunks) { return (2 * ((k & 3) | ((k >> 1) & 4))) & (chunks - 1); }

// One operand of a tile: R rows (KC) or columns (KS) from r0 on of a matrix with `rows` of them.
// p points at the tile's first k; advance by step() bytes per K step.
template <typename T, int R, bool KS, bool DUAL, int NW, int SB = 128>
struct GmSide
{
    static constexpr int ES = sizeof(typename T::elem);
    static constexpr int BK = SB / ES;                   // elements per K step
    static constexpr int CH = KS ? R * ES / 16 : SB / 16;   // chunks of 16 bytes per LDS row
    static constexpr int LROWS = 64 / CH;                // LDS rows per load of a wave
    static constexpr int NI = R * SB / 1024;             // wave loads per K step
    static constexpr int NV = (NI + NW - 1) / NW;        // per wave (waves past NI repeat others' loads)
    static constexpr int BYTES = R * SB;
    static_assert(CH <= 64, "an LDS row is at most one wave load");

    uint32_t voff[NV];                                   // AL: this lane's byte offset from the base in load j
    const char* p0;
    const char* p1;                                      // DUAL: the second matrix (rows 16..31 of every 32)
    int64_t ld;
    int nrow;                                            // rows (KC) or columns (KS) from r0 to the matrix's end

    __device__ __forceinline__ void init(int wave, int lane, const char* a, const char* b, int64_t ld_, int r0, int rows)
    {
        ld = ld_;
        nrow = rows - r0;
        p0 = gm_uniform(KS ? a + (int64_t)r0 * ES : a + (int64_t)r0 * ld);
        p1 = DUAL ? gm_uniform(b + (int64_t)r0 * ld) : p0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
        {
            const int r = lrow(wave, lane, j), c = chunk(lane, r);
            if constexpr (KS) voff[j] = (uint32_t)(r * (int)ld + min(c * 16, ((nrow + 7) / 8 - 1) * 16));
            else voff[j] = (uint32_t)(min(src_row(r), nrow - 1) * (int)ld + c * 16);
        }
    }
    // LDS row of this lane in load j, and the source chunk that belongs to its place in row r
    static __device__ __forceinline__ int lrow(int wave, int lane, int j) { return (wave + NW * j) % NI * LROWS + lane / CH; }
    static __device__ __forceinline__ int chunk(int lane, int r)
    {
        return (lane % CH) ^ (KS ? gm_ks_swz(r, CH) : gm_kc_swz<CH>(r));
    }
    // row of the matrix that LDS row r holds (DUAL: rows 16..31 of every 32 come from the second matrix)
    static __device__ __forceinline__ int src_row(int r) { return DUAL ? (r >> 5) * 16 + (r & 15) : r; }
    static __device__ __forceinline__ bool second(int wave, int j) { return DUAL && ((((wave + NW * j) % NI) * LROWS >> 4) & 1); }
    __device__ __forceinline__ int64_t step() const { return KS ? (int64_t)BK * ld : SB; }
    __device__ __forceinline__ void advance(int64_t n)
    {
        p0 += n * step();
        if (DUAL) p1 += n * step();
    }

    // load j of a whole K step, LDS-direct, from the descriptors of p0 and p1
    __device__ __forceinline__ void issue_whole(int j, int lds, int wave, gm_i4 r0, gm_i4 r1) const
    {
        gm_load_lds(second(wave, j) ? r1 : r0, lds + (wave + NW * j) % NI * 1024, voff[j]);
    }
    // LDS-direct loads of one K step of which `rem` elements exist
    __device__ __forceinline__ void issue(char* lds, int wave, int lane, int rem) const
    {
        const int at = gm_lds_at(lds);
        const gm_i4 r0 = gm_rsrc(p0), r1 = DUAL ? gm_rsrc(p1) : r0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
        {
            uint32_t v = voff[j];
            if (rem < BK)
            {
                const int r = lrow(wave, lane, j);
                v = (KS ? r : chunk(lane, r) * (16 / ES)) < rem ? v : GM_OUT;
            }
            gm_load_lds(second(wave, j) ? r1 : r0, at + (wave + NW * j) % NI * 1024, v);
        }
    }
    // the same chunks through registers
    __device__ __forceinline__ void fetch(gm_i4 (&b)[NV], int wave, int lane, int rem) const
    {
#pragma unroll
        for (int j = 0; j < NV; ++j)
        {
            const char* base = second(wave, j) ? p1 : p0;
            const int r = lrow(wave, lane, j), c = chunk(lane, r) * (16 / ES);
            if constexpr (KS) b[j] = gm_masked<ES>(base + r * ld + c * ES, r < rem ? (nrow - c) * ES : 0);
            else b[j] = gm_masked<ES>(base + (int64_t)min(src_row(r), nrow - 1) * ld + c * ES, (rem - c) * ES);
        }
    }
    // one K step through registers at once
    __device__ __forceinline__ void carry(char* lds, int wave, int lane, int rem) const
    {
        gm_i4 b[NV];
        fetch(b, wave, lane, rem);
        commit(b, lds, wave, lane);
    }
    __device__ __forceinline__ void commit(const gm_i4 (&b)[NV], char* lds, int wave, int lane) const
    {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            *reinterpret_cast<gm_i4*>(lds + (wave + NW * j) % NI * 1024 + lane * 16) = b[j];
    }

    // fragment f (rows 16f..16f+15), 64 bytes kk of the K step's rows
    static __device__ __forceinline__ gm_i4 frag(const char* lds, int lane, int f, int kk)
    {
        const int i = lane & 15, q = lane >> 4;
        if constexpr (!KS)
            return *reinterpret_cast<const gm_i4*>(lds + (f * 16 + i) * SB + (((kk * 4 + q) ^ gm_kc_swz<CH>(i)) << 4));
        else
        {
            union { gm_i4 v; gm_s4 h[2]; } r;
#pragma unroll
            for (int j = 0; j < 2; ++j)
            {
                const int k = kk * 32 + q * 8 + j * 4 + (i >> 2);
                const int off = k * (CH * 16) + (((f * 2 + ((i & 3) >> 1)) ^ gm_ks_swz(k, CH)) << 4) + (i & 1) * 8;
                r.h[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((gm_s4 __attribute__((address_space(3)))*)(lds + off));
            }
            return r.v;
        }
    }
};

// p[i] by a select: an index into the arguments would put them into memory
template <typename P>
__device__ __forceinline__ P gm_pick(P const (&p)[2], int i)
{
    return i ? p[1] : p[0];
}

template <typename E>
__device__ __forceinline__ float gm_silu(float g, float& s)
{
    s = __builtin_amdgcn_rcpf(1.0f + __expf(-g));
    return g * s;
}

// v = 4 neighbouring elements at p of which the first n exist
template <typename E>
__device__ __forceinline__ void gm_store4(E* p, const float (&v)[4], int n)
{
    typedef E vec __attribute__((ext_vector_type(4)));
    if (n >= 4 && (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(E) - 1)) == 0)
    {
        vec o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = static_cast<E>(v[i]);
        *reinterpret_cast<vec*>(p) = o;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) p[i] = static_cast<E>(v[i]);
}
template <typename E>
__device__ __forceinline__ void gm_load4(const E* p, float (&v)[4], int n)
{
    typedef E vec __attribute__((ext_vector_type(4)));
    if (n >= 4 && (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(E) - 1)) == 0)
    {
        const vec o = *reinterpret_cast<const vec*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(o[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? static_cast<float>(p[i]) : 0.f;
}

__device__ __forceinline__ void gm_put4(void* out, int odt, int64_t at, const float (&v)[4], int n, int accumulate)
{
    if (odt == 2)
    {
        float* p = static_cast<float*>(out) + at;
        if (accumulate)
        {
            float o[4];
            gm_load4(p, o, n);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += v[i];
            gm_store4(p, o, n);
        }
        else gm_store4(p, v, n);
    }
    else if (odt == 1) gm_store4(static_cast<__bf16*>(out) + at, v, n);
    else gm_store4(static_cast<_Float16*>(out) + at, v, n);
}

__device__ __forceinline__ void gm_put1(void* out, int odt, int64_t at, float v)
{
    if (odt == 2) static_cast<float*>(out)[at] = v;
    else if (odt == 1) static_cast<__bf16*>(out)[at] = static_cast<__bf16>(v);
    else static_cast<_Float16*>(out)[at] = static_cast<_Float16>(v);
}

// The clamps of silu(g) and u, by comparison: a NaN stays one (fminf and fmaxf would give the limit for it).
__device__ __forceinline__ float gm_clamp_gate(float t, float limit) { return t > limit ? limit : t; }
__device__ __forceinline__ float gm_clamp_up(float v, float limit) { return v > limit ? limit : v < -limit ? -limit : v; }

// the block's forward epilogue for 4 neighbouring columns: h, and g and u of a training pass in fp32 (16-bit ones doubled the
// gradients' error: 2.0 against 1.4 roundings in the root mean square; their traffic is 2% of a training step). h (like dg and du
// of the backward pass) is rounded to the inputs' type, as the next product's MFMAs take it: y is off by 1.4 of the one rounding that it
// has with an fp32 h (root mean square, relative: bf16 2.3e-3 and 1.7e-3, fp16 2.9e-4 and 2.1e-4). An h in two halves would give that
// back for twice the MFMAs and bytes of down's product.
template <typename E>
__device__ __forceinline__ void gm_gate_of(float limit, const float (&g)[4], const float (&u)[4], float (&h)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        float s, t = gm_silu<E>(g[i], s), v = u[i];
        if (limit != 0.f)
        {
            t = gm_clamp_gate(t, limit);
            v = gm_clamp_up(v, limit);
        }
        h[i] = t * v;
    }
}
template <typename E>
__device__ __forceinline__ void gm_gate4(const GmArgs& a, int m, int n, const float (&g)[4], const float (&u)[4], int left)
{
    float h[4];
    gm_gate_of<E>(a.limit, g, u, h);
    gm_store4(static_cast<E*>(a.out[0]) + (int64_t)m * a.ldo + n, h, left);
    if (a.g)
    {
        gm_store4(a.g + (int64_t)m * a.ldg + n, g, left);
        gm_store4(a.u + (int64_t)m * a.ldg + n, u, left);
    }
}

// dh -> dg = dh * clamp(u) * [silu(g) <= L] * silu'(g), du = dh * min(silu(g), L) * [|u| <= L], h, for 4 neighbouring columns
template <typename E>
__device__ __forceinline__ void gm_dact_of(float limit, const float (&dh)[4], const float (&g)[4], const float (&u)[4],
                                           float (&dg)[4], float (&du)[4], float (&h)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        float s, t = gm_silu<E>(g[i], s), v = u[i];
        float kg = s + t * (1.0f - s), ku = 1.0f;
        if (limit != 0.f)
        {
            if (t > limit) kg = 0.f;
            if (fabsf(v) > limit) ku = 0.f;
            t = gm_clamp_gate(t, limit);
            v = gm_clamp_up(v, limit);
        }
        dg[i] = dh[i] * v * kg;
        du[i] = dh[i] * t * ku;
        h[i] = t * v;
    }
}
template <typename E>
__device__ __forceinline__ void gm_dact4(const GmArgs& a, int m, int n, const float (&dh)[4], const float (&g)[4],
                                         const float (&u)[4], int left)
{
    float dg[4], du[4], h[4];
    gm_dact_of<E>(a.limit, dh, g, u, dg, du, h);
    const int64_t at = (int64_t)m * a.ldo + n;
    gm_store4(static_cast<E*>(a.dg) + at, dg, left);
    gm_store4(static_cast<E*>(a.du) + at, du, left);
    gm_store4(static_cast<E*>(a.out[0]) + at, h, left);
}

// Work of a workgroup: consecutive workgroups go to the 8 XCDs in turn, and each XCD takes a run of neighbouring work, K parts
// first (a part's slice of the operands then stays in one XCD's L2), then tiles in groups of GM_GROUP tile rows, so that the
// tiles that an XCD's CUs work on at once share their operands.
constexpr int GM_GROUP = 4;
__device__ __forceinline__ void gm_tile(int b, int tm, int tn, int parts, int& part, int& im, int& in)
{
    const int tiles = tm * tn, total = tiles * parts, per = total / 8, extra = total % 8;
    const int x = b % 8, s = b / 8;
    int p = x * per + min(x, extra) + s;
    part = p / tiles;
    p -= part * tiles;
    const int wide = GM_GROUP * tn, grp = p / wide, first = grp * GM_GROUP;
    const int rows = min(GM_GROUP, tm - first), r = p - grp * wide;
    im = first + r % rows;
    in = r / rows;
}

// f(integral_constant 0), ..., f(integral_constant N - 1)
template <typename F, int... I>
__device__ __forceinline__ void gm_each(F&& f, std::integer_sequence<int, I...>)
{
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void gm_each(F&& f)
{
    gm_each(f, std::make_integer_sequence<int, N>{});
}

// A wave's tile of MI x NI fragments (tokens x columns, from m0 and n0 on) to where it goes.
template <typename T, int EP, bool DUAL, int MI, int NI>
__device__ __forceinline__ void gm_epilogue(const GmArgs& a, const typename T::acc (&acc)[NI][MI], int lane, int m0, int n0, int part,
                                            int z)
{
    const int i16 = lane & 15, q = lane >> 4;
    if constexpr (EP == EP_DACT)
    {
        // g and u of 4 fragments are loaded together, and the next 4's under these ones' arithmetic (clamped into
        // the matrix): one by one they cost 15 us of a 50 us launch (333 x 5504)
        const bool quads = a.N % 4 == 0;   // then 4 neighbouring columns are all inside or all outside
        const int nw = n0 + q * 4;
        constexpr int NB = NI < 4 ? NI : 4, HB = NI / NB;   // fragments of a load, loads of a tile row
        gm_f4 g[2][NB], u[2][NB];
        auto fetch = [&](auto kc) {
            constexpr int k = decltype(kc)::value;
            const int64_t row = (int64_t)min(m0 + k / HB * 16 + i16, a.M - 1) * a.ldg;
#pragma unroll
            for (int i = 0; i < NB; ++i)
            {
                const int64_t at = row + min(nw + (k % HB * NB + i) * 16, a.N - 4);
                g[k & 1][i] = *reinterpret_cast<const gm_f4*>(a.g + at);
                u[k & 1][i] = *reinterpret_cast<const gm_f4*>(a.u + at);
            }
        };
        if (quads) fetch(std::integral_constant<int, 0>{});
        gm_each<MI * HB>([&](auto kc) {
            constexpr int k = decltype(kc)::value, j = k / HB;
            if constexpr (k + 1 < MI * HB)
                if (quads) fetch(std::integral_constant<int, k + 1>{});
            const int m = m0 + j * 16 + i16;
            if (m >= a.M) return;
#pragma unroll
            for (int i = 0; i < NB; ++i)
            {
                const int n = nw + (k % HB * NB + i) * 16;
                if (n >= a.N) continue;
                float v[4], gv[4], uv[4];
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    v[r] = static_cast<float>(acc[k % HB * NB + i][j][r]), gv[r] = g[k & 1][i][r], uv[r] = u[k & 1][i][r];
                if (!quads)
                {
                    gm_load4(a.g + (int64_t)m * a.ldg + n, gv, a.N - n);
                    gm_load4(a.u + (int64_t)m * a.ldg + n, uv, a.N - n);
                }
                gm_dact4<typename T::elem>(a, m, n, v, gv, uv, a.N - n);
            }
        });
        return;
    }
    gm_each<MI>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        const int m = m0 + j * 16 + i16;
        if (m >= a.M) return;
        gm_each<NI / (DUAL ? 2 : 1)>([&](auto ic) {
            constexpr int i = decltype(ic)::value * (DUAL ? 2 : 1);
            const int n = n0 + decltype(ic)::value * 16 + q * 4;
            if (n >= a.N) return;
            if constexpr (EP == EP_PART)
            {
                typename T::scalar* p = static_cast<typename T::scalar*>(a.out[0]) +
                                        ((int64_t)part * (DUAL ? 2 : 1) * a.M + m) * a.ldo + n;
                // ldo is a multiple of 4 and rows are padded to it: whole vectors
                *reinterpret_cast<typename T::acc*>(p) = acc[i][j];
                if (DUAL) *reinterpret_cast<typename T::acc*>(p + (int64_t)a.M * a.ldo) = acc[i + DUAL][j];
            }
            else
            {
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = static_cast<float>(acc[i][j][r]);
                if constexpr (EP == EP_GATE)
                {
                    float w[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) w[r] = static_cast<float>(acc[i + DUAL][j][r]);
                    gm_gate4<typename T::elem>(a, m, n, v, w, a.N - n);
                }
                else
                {
                    if constexpr (EP == EP_I8)
                    {
                        float sn[4];
                        gm_load4(a.sb + n, sn, a.N - n);
                        const float sm = a.sa[m];
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] = v[r] * sm * sn[r];
                    }
                    gm_put4(gm_pick(a.out, z), a.odt, (int64_t)m * a.ldo + n, v, a.N - n, a.accumulate);
                }
            }
        });
    });
}

template <typename T, int TM, int TN, int WM, int WN, bool AKS, bool BKS, bool DUAL, int NST, bool AL, int EP>
__global__ __launch_bounds__(WM* WN * 64, (WM * WN + 3) / 4) void gm_kernel(GmArgs a)
{
    constexpr int NW = WM * WN;
    typedef GmSide<T, TM, AKS, false, NW> SA;
    typedef GmSide<T, TN, BKS, DUAL, NW> SB;
    constexpr int MI = TM / WM / 16, NI = TN / WN / 16;
    constexpr int STAGE = SA::BYTES + SB::BYTES;
    constexpr int BK = SA::BK;
    static_assert(!DUAL || NI % 2 == 0, "gate and up fragments alternate");
    extern __shared__ __align__(16) char gm_lds[];

    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64), lane = threadIdx.x % 64;
    const int wm = wave / WN, wn = wave % WN;
    int part, im, in;
    gm_tile(blockIdx.x, a.tm, a.tn, a.parts, part, im, in);
    constexpr int TNC = DUAL ? TN / 2 : TN;   // columns of a tile
    const int m0 = im * TM, n0 = in * TNC;
    const int z = blockIdx.z;

    // K steps of this part, over the segments
    const int steps1 = (a.K + BK - 1) / BK;
    int t0 = 0, t1 = steps1 * a.segs;
    if (a.parts > 1)
    {
        t0 = (int)((int64_t)t1 * part / a.parts);
        t1 = (int)((int64_t)t1 * (part + 1) / a.parts);
    }
    SA sa;
    SB sb;
    const int seg0 = t0 >= steps1 && a.segs > 1 ? 1 : 0;   // the segment that the part starts in (z: one segment)
    sa.init(wave, lane, gm_pick(a.A, z + seg0), nullptr, a.lda, m0, a.M);
    sb.init(wave, lane, DUAL ? a.B[0] : gm_pick(a.B, z + seg0), a.B[1], a.ldb, n0, a.N);
    sa.advance(t0 - seg0 * steps1);
    sb.advance(t0 - seg0 * steps1);
    // the step whose loads are issued next
    int ti = t0;
    auto rem_of = [&](int t) { return a.K - (t < steps1 ? t : t - steps1) * BK; };
    auto next = [&]() {
        ++ti;
        if (a.segs > 1 && ti == steps1)   // the second segment from its start
        {
            sa.p0 = gm_uniform(AKS ? a.A[1] + (int64_t)m0 * SA::ES : a.A[1] + (int64_t)m0 * a.lda);
            sb.p0 = gm_uniform(BKS ? a.B[1] + (int64_t)n0 * SB::ES : a.B[1] + (int64_t)n0 * a.ldb);
        }
        else
        {
            sa.advance(1);
            sb.advance(1);
        }
    };

    typename T::acc acc[NI][MI];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) acc[i][j] = typename T::acc{ 0, 0, 0, 0 };

    auto compute = [&](const char* st) {
        const char* la = st + (AKS ? 0 : wm * (TM / WM) * 128);
        const char* lb = st + SA::BYTES + (BKS ? 0 : wn * (TN / WN) * 128);
        const int fa = AKS ? wm * MI : 0, fb = BKS ? wn * NI : 0;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
        {
            gm_i4 fa_[MI], fb_[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) fb_[i] = SB::frag(lb, lane, fb + i, kk);
#pragma unroll
            for (int j = 0; j < MI; ++j) fa_[j] = SA::frag(la, lane, fa + j, kk);
#pragma unroll
            for (int j = 0; j < MI; ++j)
#pragma unroll
                for (int i = 0; i < NI; ++i) acc[i][j] = T::mfma(fb_[i], fa_[j], acc[i][j]);
        }
    };

    if constexpr (AL)
    {
        constexpr int NV = SA::NV + SB::NV;
        auto issue = [&](int slot) {
            char* st = gm_lds + slot * STAGE;
            const int rem = rem_of(ti);
            if (a.ragged && rem <= BK)
            {
                // (its loads are waited for here, and with them all earlier ones: the counted waits below stay true)
                sa.carry(st, wave, lane, rem);
                sb.carry(st + SA::BYTES, wave, lane, rem);
            }
            else
            {
                sa.issue(st, wave, lane, rem);
                sb.issue(st + SA::BYTES, wave, lane, rem);
            }
            next();
        };
        for (int s = 0; s < NST - 1; ++s)
            if (ti < t1) issue(s);
        int cur = 0, fill = NST - 1;
        for (int t = t0; t < t1; ++t)
        {
            if (t + NST - 2 < t1) gm_wait_vmcnt<(NST - 2) * NV>();   // this wave's loads of step t have landed
            else gm_wait_vmcnt<0>();
            gm_barrier();                     // every wave's have, and every wave is done with step t - 1
            if (ti < t1) issue(fill);         // into the slot of step t - 1
            compute(gm_lds + cur * STAGE);
            cur = cur + 1 == NST ? 0 : cur + 1;
            fill = fill + 1 == NST ? 0 : fill + 1;
        }
    }
    else
    {
        gm_i4 ba[SA::NV], bb[SB::NV];
        if (ti < t1)
        {
            sa.fetch(ba, wave, lane, rem_of(ti));
            sb.fetch(bb, wave, lane, rem_of(ti));
            next();
        }
        for (int t = t0; t < t1; ++t)
        {
            __syncthreads();   // every wave is done with step t - 1
            sa.commit(ba, gm_lds, wave, lane);
            sb.commit(bb, gm_lds + SA::BYTES, wave, lane);
            __syncthreads();
            if (ti < t1)
            {
                sa.fetch(ba, wave, lane, rem_of(ti));
                sb.fetch(bb, wave, lane, rem_of(ti));
                next();
            }
            compute(gm_lds);
        }
    }

    gm_epilogue<T, EP, DUAL, MI, NI>(a, acc, lane, m0 + wm * (TM / WM), n0 + wn * (TNC / WN), part, z);
}

// A wave's 16-bit results by way of LDS: lanes put 4 neighbouring columns each, then whole runs of a row go out (a fragment's own
// stores are 16 rows x 32 bytes; with them a 4096 x 12288 output of 256 x 256 tiles took 80 us at K = 128). Rows are padded by 16
// bytes, so that 16 neighbouring rows' puts spread over the banks.
template <typename E, int C>
__device__ __forceinline__ void gm_put_row(char* lds, int row, int col, const float (&v)[4])
{
    typedef E vec __attribute__((ext_vector_type(4)));
    vec o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = static_cast<E>(v[i]);
    *reinterpret_cast<vec*>(lds + row * (C * 2 + 16) + col * 2) = o;
}
template <int ROWS, int C>
__device__ __forceinline__ void gm_flush_rows(const char* lds, int lane, void* out, int64_t ldo, int m0, int n0, int M, int N)
{
    constexpr int LPR = C / 8, RPI = 64 / LPR;   // lanes of a row, rows of a store
    const int r0 = lane / LPR, c = lane % LPR * 8;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // this wave's puts
    if (n0 + c < N)
#pragma unroll
        for (int i = 0; i < ROWS / RPI; ++i)
        {
            const int r = i * RPI + r0;
            if (m0 + r < M)
                *reinterpret_cast<gm_i4*>(static_cast<uint16_t*>(out) + (int64_t)(m0 + r) * ldo + n0 + c) =
                    *reinterpret_cast<const gm_i4*>(lds + r * (C * 2 + 16) + c * 2);
        }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read, before the next puts
}

constexpr int GM_BIG_LDS = 4 * 128 * 272;   // 4 waves' rows on the way out; the K steps' ring takes 128 KB of it

// gm_epilogue of a wave's 128 x 128 results (DUAL: 128 x 64 of each matrix) where whole chunks of 16 bytes can be stored
template <typename T, int EP, bool DUAL>
__device__ __forceinline__ void gm_big_epilogue(const GmArgs& a, const typename T::acc (&acc)[8][8], char* lds, int lane, int m0, int n0,
                                                int z)
{
    typedef typename T::elem E;
    const int i16 = lane & 15, q = lane >> 4;
    if constexpr (EP == EP_GATE)
    {
        gm_each<8>([&](auto jc) {
            constexpr int j = decltype(jc)::value;
            const int m = m0 + j * 16 + i16;
            gm_each<4>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                float g[4], u[4], h[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) g[r] = acc[2 * i][j][r], u[r] = acc[2 * i + 1][j][r];
                gm_gate_of<E>(a.limit, g, u, h);
                gm_put_row<E, 64>(lds, j * 16 + i16, i * 16 + q * 4, h);
                const int n = n0 + i * 16 + q * 4;
                if (a.g && m < a.M && n < a.N)
                {
                    gm_store4(a.g + (int64_t)m * a.ldg + n, g, 4);
                    gm_store4(a.u + (int64_t)m * a.ldg + n, u, 4);
                }
            });
        });
        gm_flush_rows<128, 64>(lds, lane, a.out[0], a.ldo, m0, n0, a.M, a.N);
    }
    else if constexpr (EP == EP_DACT)
    {
        constexpr int R = 32, REG = R * 272;   // rows at a time, of three outputs
        gm_f4 g[2][4], u[2][4];
        auto fetch = [&](auto kc) {            // 4 fragments' g and u, clamped into the matrix
            constexpr int k = decltype(kc)::value;
            const int64_t row = (int64_t)min(m0 + k / 2 * 16 + i16, a.M - 1) * a.ldg;
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const int64_t at = row + min(n0 + q * 4 + (k % 2 * 4 + i) * 16, a.N - 4);
                g[k & 1][i] = *reinterpret_cast<const gm_f4*>(a.g + at);
                u[k & 1][i] = *reinterpret_cast<const gm_f4*>(a.u + at);
            }
        };
        fetch(std::integral_constant<int, 0>{});
        gm_each<16>([&](auto kc) {
            constexpr int k = decltype(kc)::value, j = k / 2, b = k % 2 * 4;
            if constexpr (k + 1 < 16) fetch(std::integral_constant<int, k + 1>{});
            gm_each<4>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                float v[4], gv[4], uv[4], dg[4], du[4], h[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = acc[b + i][j][r], gv[r] = g[k & 1][i][r], uv[r] = u[k & 1][i][r];
                gm_dact_of<E>(a.limit, v, gv, uv, dg, du, h);
                const int row = j % 2 * 16 + i16, col = (b + i) * 16 + q * 4;
                gm_put_row<E, 128>(lds, row, col, dg);
                gm_put_row<E, 128>(lds + REG, row, col, du);
                gm_put_row<E, 128>(lds + 2 * REG, row, col, h);
            });
            if constexpr (k % 4 == 3)
            {
                const int at = m0 + j / 2 * R;
                gm_flush_rows<R, 128>(lds, lane, a.dg, a.ldo, at, n0, a.M, a.N);
                gm_flush_rows<R, 128>(lds + REG, lane, a.du, a.ldo, at, n0, a.M, a.N);
                gm_flush_rows<R, 128>(lds + 2 * REG, lane, a.out[0], a.ldo, at, n0, a.M, a.N);
            }
        });
    }
    else
    {
        float sn[8][4];
        if constexpr (EP == EP_I8)
#pragma unroll
            for (int i = 0; i < 8; ++i) gm_load4(a.sb + min(n0 + i * 16 + q * 4, a.N - 4), sn[i], 4);
        gm_each<8>([&](auto jc) {
            constexpr int j = decltype(jc)::value;
            float sm = 0.f;
            if constexpr (EP == EP_I8) sm = a.sa[min(m0 + j * 16 + i16, a.M - 1)];
            gm_each<8>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r)
                {
                    v[r] = static_cast<float>(acc[i][j][r]);
                    if constexpr (EP == EP_I8) v[r] = v[r] * sm * sn[i][r];
                }
                if (a.odt == 1) gm_put_row<__bf16, 128>(lds, j * 16 + i16, i * 16 + q * 4, v);
                else gm_put_row<_Float16, 128>(lds, j * 16 + i16, i * 16 + q * 4, v);
            });
        });
        gm_flush_rows<128, 128>(lds, lane, gm_pick(a.out, z), a.ldo, m0, n0, a.M, a.N);
    }
}

// The largest products: 256 x 256 by 4 waves of 128 x 128, one to a SIMD. Bound by LDS reads: 8 waves of 128 x 64 read 192 KB for
// a tile's 64 k (1536 cycles of 128 bytes, beside 512 of writes and 2048 of MFMA), these 128 KB. A wave's accumulators
// are all 256 AGPRs (by asm constraint; left to itself the compiler copied or spilled them), its fragments of this step and of the
// next 128 VGPRs. In the K loop nothing is spilled; around it 16 to 25 VGPRs are in the forms but dh's and i8's. K steps of 64 bytes a
// row, NST slots of 32 KB: a step's MFMAs run under the reads of the next step's fragments and the loads of the step NST - 1 ahead,
// one barrier a step. bf16 4096 x 12288 x 5120: 384 us (1.34 PFLOP/s) against 466 by 8 waves on one card; 8192 x 8192 x
// 8192: 785 (1.40) against 914. Under it clocks are 1.9 to 2.1 GHz, and MFMAs fill 50 to 62% of the SIMDs' cycles (37 in the form
// of dh, whose epilogue is the longest). A fifth slot and other orders of the reads made no difference.
template <typename T, bool AKS, bool BKS, bool DUAL, int EP>
__global__ __launch_bounds__(256, 1) void gm_big_kernel(GmArgs a)
{
    constexpr int NST = 4;
    typedef GmSide<T, 256, AKS, false, 4, 64> SA;
    typedef GmSide<T, 256, BKS, DUAL, 4, 64> SB;
    constexpr int STAGE = SA::BYTES + SB::BYTES, BK = SA::BK, NV = SA::NV + SB::NV;
    static_assert(SA::NV == 4 && SB::NV == 4, "a load for every second group of MFMAs");
    extern __shared__ __align__(16) char gm_lds[];

    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64), lane = threadIdx.x % 64;
    const int wm = wave / 2, wn = wave % 2, z = blockIdx.z;
    int part, im, in;
    gm_tile(blockIdx.x, a.tm, a.tn, 1, part, im, in);
    constexpr int TNC = DUAL ? 128 : 256;
    const int m0 = im * 256, n0 = in * TNC;
    // whole steps by the pipeline; a segment's last step that is not whole comes after it, through registers
    // (where rows end inside a chunk of 16 bytes the last step of whole rows does too: its last row's chunk would reach past the matrix)
    const int steps1 = (a.K - (a.ragged && (AKS || BKS) ? 1 : 0)) / BK, steps = steps1 * a.segs, tail = a.K - steps1 * BK;
    SA sa;
    SB sb;
    sa.init(wave, lane, gm_pick(a.A, z), nullptr, a.lda, m0, a.M);
    sb.init(wave, lane, DUAL ? a.B[0] : gm_pick(a.B, z), a.B[1], a.ldb, n0, a.N);
    auto segment = [&](int s) {
        sa.p0 = gm_uniform(AKS ? gm_pick(a.A, s) + (int64_t)m0 * SA::ES : gm_pick(a.A, s) + (int64_t)m0 * a.lda);
        sb.p0 = gm_uniform(BKS ? gm_pick(a.B, s) + (int64_t)n0 * SB::ES : gm_pick(a.B, s) + (int64_t)n0 * a.ldb);
    };
    int ti = 0;   // the step whose loads are issued next
    auto next = [&]() {
        ++ti;
        if (a.segs > 1 && ti == steps1) segment(1);
        else if (ti < steps)
        {
            sa.advance(1);
            sb.advance(1);
        }
    };

    typename T::acc acc[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = typename T::acc{ 0, 0, 0, 0 };
    gm_i4 fa[2][8], fb[2][8];
    auto slot_a = [&](int s) { return gm_lds + s * STAGE + (AKS ? 0 : wm * 128 * 64); };
    auto slot_b = [&](int s) { return gm_lds + s * STAGE + SA::BYTES + (BKS ? 0 : wn * 128 * 64); };
    const int f0a = AKS ? wm * 8 : 0, f0b = BKS ? wn * 8 : 0, lds0 = gm_lds_at(gm_lds);

    for (int s = 0; s < NST - 1; ++s)
    {
        const int live = ti < steps ? 0x7FFFFFFF : 0;   // past the end nothing is read (zeros are written)
        const gm_i4 ra = gm_rsrc(sa.p0, live), rb = gm_rsrc(sb.p0, live), rb1 = DUAL ? gm_rsrc(sb.p1, live) : rb;
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            sa.issue_whole(j, lds0 + s * STAGE, wave, ra, ra);
            sb.issue_whole(j, lds0 + s * STAGE + SA::BYTES, wave, rb, rb1);
        }
        next();
    }
    gm_wait_vmcnt<(NST - 2) * NV>();
    gm_barrier();
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        fb[0][i] = SB::frag(slot_b(0), lane, f0b + i, 0);
        fa[0][i] = SA::frag(slot_a(0), lane, f0a + i, 0);
    }
    // what a step's reads and loads need, worked out during the step before: its descriptors, the slot its loads go to, the slot its
    // reads come from (the next step's)
    int nxt = 1, fill = NST - 1;
    gm_i4 ra, rb, rb1;
    auto prepare = [&]() {
        const int live = ti < steps ? 0x7FFFFFFF : 0;
        ra = gm_rsrc(sa.p0, live);
        rb = gm_rsrc(sb.p0, live);
        rb1 = DUAL ? gm_rsrc(sb.p1, live) : rb;
    };
    prepare();
    // one step on fragment set c
    auto step = [&](auto set) {
        constexpr int c = decltype(set)::value;
        gm_wait_vmcnt<(NST - 3) * NV>();   // this wave's loads of the next step have landed
        gm_barrier();                      // every wave's have; every wave has read this step's slot and the one before
        const int to = lds0 + fill * STAGE;
        const char *la = slot_a(nxt), *lb = slot_b(nxt);
        // the next step's fragment r, the columns' first
        auto read = [&](auto rc) {
            constexpr int r = decltype(rc)::value;
            if constexpr (r < 8) fb[c ^ 1][r] = SB::frag(lb, lane, f0b + r, 0);
            else fa[c ^ 1][r - 8] = SA::frag(la, lane, f0a + r - 8, 0);
        };
        // 4 MFMAs, then what goes out under them: the reads end some 250 cycles before the barrier that waits for them
        gm_each<16>([&](auto gc) {
            constexpr int g = decltype(gc)::value;
#pragma unroll
            for (int k = 0; k < 4; ++k)
            {
                const int e = g * 4 + k;
                T::mfma_agpr(fb[c][e % 8], fa[c][e / 8], acc[e % 8][e / 8]);
            }
            if constexpr (g < 4)
            {
                read(std::integral_constant<int, 2 * g>{});
                read(std::integral_constant<int, 2 * g + 1>{});
            }
            else if constexpr (g < 12) read(std::integral_constant<int, g + 4>{});
            if constexpr (g % 2 == 0)
            {
                if constexpr (g < 8) sa.issue_whole(g / 2, to, wave, ra, ra);
                else sb.issue_whole(g / 2 - 4, to + SA::BYTES, wave, rb, rb1);
            }
            if constexpr (g == 14) next();
            if constexpr (g == 15)
            {
                prepare();
                nxt = nxt + 1 == NST ? 0 : nxt + 1;
                fill = fill + 1 == NST ? 0 : fill + 1;
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    for (int p = 0; p < steps / 2; ++p)
    {
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
    }
    if (steps & 1) step(std::integral_constant<int, 0>{});
    gm_wait_vmcnt<0>();
    if (tail)
        for (int s = 0; s < a.segs; ++s)
        {
            if (a.segs > 1) segment(s);
            else
            {
                sa.p0 = gm_uniform(AKS ? gm_pick(a.A, z) + (int64_t)m0 * SA::ES : gm_pick(a.A, z) + (int64_t)m0 * a.lda);
                sb.p0 = gm_uniform(DUAL ? a.B[0] + (int64_t)n0 * a.ldb : BKS ? gm_pick(a.B, z) + (int64_t)n0 * SB::ES : gm_pick(a.B, z) + (int64_t)n0 * a.ldb);
                if (DUAL) sb.p1 = gm_uniform(a.B[1] + (int64_t)n0 * a.ldb);
            }
            sa.advance(steps1);
            sb.advance(steps1);
            gm_barrier();   // the slot is read
            sa.carry(gm_lds, wave, lane, tail);
            sb.carry(gm_lds + SA::BYTES, wave, lane, tail);
            gm_barrier();
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                fb[0][i] = SB::frag(slot_b(0), lane, f0b + i, 0);
                fa[0][i] = SA::frag(slot_a(0), lane, f0a + i, 0);
            }
#pragma unroll
            for (int e = 0; e < 64; ++e) T::mfma_agpr(fb[0][e % 8], fa[0][e / 8], acc[e % 8][e / 8]);
        }
    // The last MFMAs' results: the compiler puts no wait between an MFMA in asm and a read of what it writes, so these 32 wait
    // states, more than any MFMA needs, come before every read: each accumulator passes an asm after them. (By themselves they
    // hold nothing back: the reads were moved up to 5 instructions behind the MFMA.)
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) asm volatile("" : "+a"(acc[i][j]));
    if (a.wide)
    {
        gm_barrier();   // the ring is done with
        gm_big_epilogue<T, EP, DUAL>(a, acc, gm_lds + wave * (GM_BIG_LDS / 4), lane, m0 + wm * 128, n0 + wn * (TNC / 2), z);
    }
    else gm_epilogue<T, EP, DUAL, 8, 8>(a, acc, lane, m0 + wm * 128, n0 + wn * (TNC / 2), 0, z);
}

// Joins the K parts of a split product and runs its epilogue: a thread per 4 neighbouring columns.
template <typename T, bool DUAL, int EP>
__global__ __launch_bounds__(256) void gm_join_kernel(GmArgs a, const void* part, int64_t ldp, int parts)
{
    const int cols = (a.N + 3) / 4;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= (int64_t)a.M * cols) return;
    const int m = (int)(at / cols), n = (int)(at % cols) * 4;
    const typename T::scalar* p = static_cast<const typename T::scalar*>(part) + (int64_t)m * ldp + n;
    typename T::acc s0 = { 0, 0, 0, 0 }, s1 = { 0, 0, 0, 0 };
    const int64_t mat = (int64_t)a.M * ldp;
    for (int k = 0; k < parts; ++k)
    {
        s0 += *reinterpret_cast<const typename T::acc*>(p);
        if (DUAL) s1 += *reinterpret_cast<const typename T::acc*>(p + mat);
        p += (DUAL ? 2 : 1) * mat;
    }
    float v[4], w[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = static_cast<float>(s0[r]), w[r] = static_cast<float>(s1[r]);
    if constexpr (EP == EP_GATE) gm_gate4<typename T::elem>(a, m, n, v, w, a.N - n);
    else if constexpr (EP == EP_DACT)
    {
        float g[4], u[4];
        gm_load4(a.g + (int64_t)m * a.ldg + n, g, a.N - n);
        gm_load4(a.u + (int64_t)m * a.ldg + n, u, a.N - n);
        gm_dact4<typename T::elem>(a, m, n, v, g, u, a.N - n);
    }
    else
    {
        if constexpr (EP == EP_I8)
        {
            float sn[4];
            gm_load4(a.sb + n, sn, a.N - n);
            const float sm = a.sa[m];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = v[r] * sm * sn[r];
        }
        gm_put4(a.out[0], a.odt, (int64_t)m * a.ldo + n, v, a.N - n, a.accumulate);
    }
}

// ---- few tokens (M <= 16): bound by the weights' bytes, one launch per product, no parts to join ----

// Results of 4 neighbouring columns (n..n+3, the first `left` of them wanted) of token m.
template <typename T, bool DUAL, int EP>
__device__ __forceinline__ void gm_finish4(const GmArgs& a, int m, int n, float (&v)[4], const float (&up)[4], int left)
{
    if constexpr (EP == EP_GATE) gm_gate4<typename T::elem>(a, m, n, v, up, left);
    else
    {
        if constexpr (EP == EP_I8)
        {
            float sn[4];
            gm_load4(a.sb + n, sn, left);
            const float sm = a.sa[m];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = v[k] * sm * sn[k];
        }
        gm_put4(a.out[0], a.odt, (int64_t)m * a.ldo + n, v, left, a.accumulate);
    }
}

// sum over a fragment's 16 bytes of products
__device__ __forceinline__ float gm_dot(GmF16, gm_i4 a, gm_i4 b, float c)
{
    const gm_h8 x = __builtin_bit_cast(gm_h8, a), y = __builtin_bit_cast(gm_h8, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) c = fmaf((float)x[i], (float)y[i], c);
    return c;
}
__device__ __forceinline__ float gm_dot(GmBF16, gm_i4 a, gm_i4 b, float c)
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        c = fmaf(__int_as_float(a[i] << 16), __int_as_float(b[i] << 16), c);
        c = fmaf(__int_as_float(a[i] & 0xFFFF0000), __int_as_float(b[i] & 0xFFFF0000), c);
    }
    return c;
}
__device__ __forceinline__ int gm_dot(GmI8, gm_i4 a, gm_i4 b, int c)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_sdot4(a[i], b[i], c, false);
    return c;
}

// One or two tokens: a wave forms two dot products (a gate and an up row, or two neighbouring rows), 1 KB of a row a load, U
// loads of each in flight. With the MFMA fragments of the kernels below 16 rows share a load, 64 or 128 bytes of each: 5120 x
// 1536 fp16 gate|up, weights from HBM, 9.4 and 8.4 us against 7.9 here (4.0 TB/s with the launch; a large copy reaches 4.8).
template <typename T, bool DUAL, int EP, int MM, int U>
__global__ __launch_bounds__(256) void gm_row_kernel(GmArgs a)
{
    constexpr int ES = sizeof(typename T::elem);
    const int lane = threadIdx.x % 64, row = (blockIdx.x * 4 + threadIdx.x / 64) * (DUAL ? 1 : 2);
    if (row >= a.N) return;
    const int kb = a.K * ES, whole = kb / 1024;
    const char* w0 = a.B[0] + (int64_t)row * a.ldb + lane * 16;
    const char* w1 = DUAL ? a.B[1] + (int64_t)row * a.ldb + lane * 16 : row + 1 < a.N ? w0 + a.ldb : w0;
    const char* x = a.A[0] + lane * 16;
    typename T::scalar acc[2][MM] = {};
    auto ld = [](const char* p) {
        gm_i4 v;
        __builtin_memcpy(&v, p, 16);
        return v;
    };
    int c = 0;
    for (; c + U <= whole; c += U)
    {
        gm_i4 f0[U], f1[U];
#pragma unroll
        for (int j = 0; j < U; ++j) f0[j] = ld(w0 + (c + j) * 1024), f1[j] = ld(w1 + (c + j) * 1024);
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int m = 0; m < MM; ++m)
            {
                const gm_i4 v = ld(x + m * a.lda + (c + j) * 1024);
                acc[0][m] = gm_dot(T{}, f0[j], v, acc[0][m]);
                acc[1][m] = gm_dot(T{}, f1[j], v, acc[1][m]);
            }
    }
    for (; c * 1024 < kb; ++c)
    {
        const int nb = kb - c * 1024 - lane * 16;
        const gm_i4 f0 = gm_masked<ES>(w0 + c * 1024, nb), f1 = gm_masked<ES>(w1 + c * 1024, nb);
#pragma unroll
        for (int m = 0; m < MM; ++m)
        {
            const gm_i4 v = gm_masked<ES>(x + m * a.lda + c * 1024, nb);
            acc[0][m] = gm_dot(T{}, f0, v, acc[0][m]);
            acc[1][m] = gm_dot(T{}, f1, v, acc[1][m]);
        }
    }
#pragma unroll
    for (int m = 0; m < MM; ++m)
    {
        typename T::scalar s0 = acc[0][m], s1 = acc[1][m];
#pragma unroll
        for (int o = 32; o; o >>= 1) s0 += __shfl_xor(s0, o), s1 += __shfl_xor(s1, o);
        if (lane != m) continue;
        float v[4] = { (float)s0, DUAL ? 0.f : (float)s1, 0.f, 0.f }, up[4] = { (float)s1, 0.f, 0.f, 0.f };
        gm_finish4<T, DUAL, EP>(a, m, row, v, up, DUAL ? 1 : min(2, a.N - row));
    }
}

// the waves' partial 16 x 16 tiles (rows of B x tokens) joined in LDS by wave 0
template <typename T, bool DUAL, int EP, int NW>
__device__ __forceinline__ void gm_join_waves(const GmArgs& a, typename T::acc acc, typename T::acc (*red)[16][4], int n0)
{
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    red[wave][lane & 15][lane >> 4] = acc;
    __syncthreads();
    if (wave) return;
    const int m = lane / 4, r = lane % 4;
    typename T::acc sum = red[0][m][r];
#pragma unroll
    for (int k = 1; k < NW; ++k) sum += red[k][m][r];
    float v[4], up[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
    {
        v[k] = static_cast<float>(sum[k]);
        up[k] = DUAL ? __shfl_down(v[k], 2) : 0.f;
    }
    const int n = n0 + r * 4;
    if (m >= a.M || (DUAL && r >= 2) || n >= a.N) return;
    gm_finish4<T, DUAL, EP>(a, m, n, v, up, a.N - n);
}

// 3 to 16 tokens, B's rows from 4-byte aligned addresses: 16 rows of B (DUAL: 8 of each matrix) by a workgroup of NW waves that
// take the K steps of 128 bytes a row in turn. Each wave keeps S steps in flight, its rows in an LDS ring of its own
// (loads of 8 rows x 128 bytes, no barrier before the join) and the tokens' fragments in registers.
template <typename T, bool DUAL, int EP, int NW, int S>
__global__ __launch_bounds__(NW * 64) void gm_ring_kernel(GmArgs a)
{
    constexpr int ES = sizeof(typename T::elem), NR = DUAL ? 8 : 16;
    extern __shared__ __align__(16) char gm_lds[];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64), lane = threadIdx.x % 64;
    const int i = lane & 15, q = lane >> 4, n0 = blockIdx.x * NR;
    char* ring = gm_lds + wave * S * 2048;
    const int last = a.N - 1 - n0;   // >= 0
    const char* base0 = gm_uniform(a.B[0] + (int64_t)n0 * a.ldb);
    const char* base1 = DUAL ? gm_uniform(a.B[1] + (int64_t)n0 * a.ldb) : base0;
    const int lr = lane / 8;
    const uint32_t v0 = (uint32_t)(min(lr, last) * (int)a.ldb + (((lane & 7) ^ ((lr >> 1) & 7)) << 4));
    const uint32_t v1 = (uint32_t)(min(DUAL ? lr : lr + 8, last) * (int)a.ldb + (((lane & 7) ^ (((lr + 8) >> 1) & 7)) << 4));
    const char* x = a.A[0] + (int64_t)min(i, a.M - 1) * a.lda + q * 16;
    const bool live = i < a.M;
    const int kb = a.K * ES, steps = kb / 128;   // whole steps
    typename T::acc acc = { 0, 0, 0, 0 };
    gm_i4 fx[S][2];
    auto issue = [&](int t, int s) {
        const gm_i4 r0 = gm_rsrc(base0 + (int64_t)t * 128), r1 = gm_rsrc(base1 + (int64_t)t * 128);
        gm_load_lds(r0, gm_lds_at(ring) + s * 2048, v0);
        gm_load_lds(r1, gm_lds_at(ring) + s * 2048 + 1024, v1);
        fx[s][0] = fx[s][1] = gm_i4{ 0, 0, 0, 0 };
        if (live)
        {
            __builtin_memcpy(&fx[s][0], x + (int64_t)t * 128, 16);
            __builtin_memcpy(&fx[s][1], x + (int64_t)t * 128 + 64, 16);
        }
    };
#pragma unroll
    for (int s = 0; s < S; ++s)
        if (wave + s * NW < steps) issue(wave + s * NW, s);
    for (int t = wave; t < steps; t += S * NW)
    {
#pragma unroll
        for (int s = 0; s < S; ++s)
        {
            if (t + s * NW >= steps) break;
            // this step's loads have landed: those of the S - 1 steps after it are younger
            if (t + (s + S - 1) * NW < steps) gm_wait_vmcnt<4 * (S - 1)>();
            else gm_wait_vmcnt<0>();
            gm_i4 fw[2];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
                fw[kk] = *reinterpret_cast<const gm_i4*>(ring + s * 2048 + i * 128 + (((kk * 4 + q) ^ ((i >> 1) & 7)) << 4));
            acc = T::mfma(fw[0], fx[s][0], acc);
            acc = T::mfma(fw[1], fx[s][1], acc);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the slot is read
            if (t + (s + S) * NW < steps) issue(t + (s + S) * NW, s);
        }
    }
    if (kb % 128 && wave == steps % NW)
    {
        const char* w = (DUAL && i >= 8 ? a.B[1] : a.B[0]) + (int64_t)min(n0 + (DUAL ? i & 7 : i), a.N - 1) * a.ldb + q * 16;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
        {
            const int at = steps * 128 + kk * 64, nb = kb - at - q * 16;
            acc = T::mfma(gm_masked<ES>(w + at, nb), gm_masked<ES>(x + at, live ? nb : 0), acc);
        }
    }
    __syncthreads();   // the rings are done with
    gm_join_waves<T, DUAL, EP, NW>(a, acc, reinterpret_cast<typename T::acc(*)[16][4]>(gm_lds), n0);
}

// The same from rows of any alignment: an MFMA fragment's 16 bytes a lane come straight from memory, U loads in flight.
// 8 tokens, int8 12288 x 4096: 26 us, the ring 10.
template <typename T, bool DUAL, int EP, int NW>
__global__ __launch_bounds__(NW * 64) void gm_skinny_kernel(GmArgs a)
{
    constexpr int ES = sizeof(typename T::elem), U = 8;
    __shared__ typename T::acc red[NW][16][4];   // [wave][token][4 rows]
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, i = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * (DUAL ? 8 : 16);
    const char* w = DUAL && i >= 8 ? a.B[1] : a.B[0];
    w += (int64_t)min(n0 + (DUAL ? i & 7 : i), a.N - 1) * a.ldb + q * 16;
    const char* x = a.A[0] + (int64_t)min(i, a.M - 1) * a.lda + q * 16;
    const bool live = i < a.M;
    const int kb = a.K * ES, whole = kb / 64;   // whole steps
    typename T::acc acc = { 0, 0, 0, 0 };
    auto ld = [](const char* p) {
        gm_i4 v;
        __builtin_memcpy(&v, p, 16);
        return v;
    };
    for (int t = wave; t < whole; t += U * NW)
    {
        gm_i4 fw[U], fx[U];
#pragma unroll
        for (int j = 0; j < U; ++j)
        {
            const bool in = t + j * NW < whole;
            fw[j] = in ? ld(w + (int64_t)(t + j * NW) * 64) : gm_i4{ 0, 0, 0, 0 };
            fx[j] = in && live ? ld(x + (int64_t)(t + j * NW) * 64) : gm_i4{ 0, 0, 0, 0 };
        }
#pragma unroll
        for (int j = 0; j < U; ++j) acc = T::mfma(fw[j], fx[j], acc);
    }
    if (kb % 64 && wave == whole % NW)
    {
        const int nb = kb - whole * 64 - q * 16;
        acc = T::mfma(gm_masked<ES>(w + (int64_t)whole * 64, nb), gm_masked<ES>(x + (int64_t)whole * 64, live ? nb : 0), acc);
    }
    gm_join_waves<T, DUAL, EP, NW>(a, acc, red, n0);
}

}  // namespace gfl
