// Tile choice and launches of the tile GEMM for one input type; included by one translation unit per type.
#pragma once
#include "gfl_gemm.hpp"
#include "gfl_gemm_plan.hpp"

#include <atomic>

namespace gfl {

// Allows a kernel its LDS, once on each device (the attribute belongs to the device's copy of the kernel; `opened`: a bit for each).
static inline void gm_open(const void* kern, int lds, std::atomic<uint64_t>& opened)
{
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return;   // the launch reports it
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (bit && (opened.load(std::memory_order_relaxed) & bit)) return;
    if (hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds) == hipSuccess) opened.fetch_or(bit);
}

template <typename T, int TM, int TN, int WM, int WN, bool AKS, bool BKS, bool DUAL, int NST, bool AL, int EP>
static int gm_go(const GmArgs& a, int nz, hipStream_t st)
{
    constexpr int lds = (AL ? NST : 1) * (TM + TN) * 128;
    static_assert(lds <= LDS_LIMIT, "tiles fit the LDS");
    auto* kern = gm_kernel<T, TM, TN, WM, WN, AKS, BKS, DUAL, NST, AL, EP>;
    static std::atomic<uint64_t> opened{ 0 };
    gm_open(reinterpret_cast<const void*>(kern), lds, opened);
    hipLaunchKernelGGL(kern, dim3((unsigned)(a.tm * a.tn * a.parts), 1, nz), dim3(WM * WN * 64), lds, st, a);
    return 0;
}

static int gm_wide(const GmArgs& a, int ep, int nz)
{
    auto ok = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    if (a.N % 8 || a.ldo % 8 || !ok(a.out[0]) || (nz > 1 && !ok(a.out[1]))) return 0;
    if (ep == EP_DACT) return ok(a.dg) && ok(a.du);
    return ep == EP_GATE || a.odt != 2;
}

template <typename T, bool AKS, bool BKS, bool DUAL, int EP>
static int gm_tiles(GmArgs& a, const GmPlan& p, int aligned, int nz, hipStream_t st)
{
    a.parts = p.parts;
    a.tm = (a.M + p.tm - 1) / p.tm;
    a.tn = (a.N + p.tn - 1) / p.tn;
    if (!aligned)
    {
        if constexpr (BKS && !AKS)
            if (p.tm == 16) return gm_go<T, 16, 128, 1, 4, AKS, BKS, DUAL, 2, false, EP>(a, nz, st);
        return gm_go<T, 128, 128, 2, 2, AKS, BKS, DUAL, 2, false, EP>(a, nz, st);
    }
    if constexpr (BKS && !AKS)
        if (p.tm == 16) return gm_go<T, 16, 128, 1, 4, AKS, BKS, DUAL, 4, true, EP>(a, nz, st);
    if constexpr (!AKS)
    {
        if (p.tm == 64) return gm_go<T, 64, 128, 1, 4, AKS, BKS, DUAL, 3, true, EP>(a, nz, st);
        if (p.deep) return gm_go<T, 128, 128, 2, 4, AKS, BKS, DUAL, 5, true, EP>(a, nz, st);
    }
    if (p.tm == 128) return gm_go<T, 128, 128, 2, 2, AKS, BKS, DUAL, 2, true, EP>(a, nz, st);
    if constexpr (EP == EP_PART) return -1;   // not split (gm_plan)
    else
    {
        a.wide = gm_wide(a, EP, nz);
        constexpr int lds = GM_BIG_LDS;
        auto* kern = &gm_big_kernel<T, AKS, BKS, DUAL, EP>;
        static std::atomic<uint64_t> opened{ 0 };
        gm_open(reinterpret_cast<const void*>(kern), lds, opened);
        hipLaunchKernelGGL(kern, dim3((unsigned)(a.tm * a.tn), 1, nz), dim3(256), lds, st, a);
        return 0;
    }
}

template <typename T, bool DUAL, int EP, int NW>
static void gm_ring(const GmArgs& a, int wg, hipStream_t st)
{
    constexpr int S = 4, lds = NW * S * 2048;
    auto* kern = gm_ring_kernel<T, DUAL, EP, NW, S>;
    static std::atomic<uint64_t> opened{ 0 };
    gm_open(reinterpret_cast<const void*>(kern), lds, opened);
    hipLaunchKernelGGL(kern, dim3(wg), dim3(NW * 64), lds, st, a);
}

// up to 16 tokens, B [N][K]
template <typename T, bool DUAL, int EP>
static int gm_few(const GmArgs& a, int aligned, hipStream_t st)
{
    if (a.M <= 2)
    {
        const int wg = (a.N + (DUAL ? 3 : 7)) / (DUAL ? 4 : 8);
        if (a.M == 1) hipLaunchKernelGGL((gm_row_kernel<T, DUAL, EP, 1, 5>), dim3(wg), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((gm_row_kernel<T, DUAL, EP, 2, 5>), dim3(wg), dim3(256), 0, st, a);
        return 0;
    }
    const int wg = (a.N + (DUAL ? 7 : 15)) / (DUAL ? 8 : 16);
    // 16 waves where the workgroups do not fill the CUs twice and each wave still has 3 steps (192 workgroups of 5120 fp16:
    // 8.4 us against 9.8 with 8 waves); else 8 (4096 workgroups of 4096 int8: 55 us against 63 with 4)
    const int steps = a.K * (int)sizeof(typename T::elem) / 128;
    if (!aligned) hipLaunchKernelGGL((gm_skinny_kernel<T, DUAL, EP, 8>), dim3(wg), dim3(512), 0, st, a);
    else if (wg <= 256 && steps >= 48) gm_ring<T, DUAL, EP, 16>(a, wg, st);
    else gm_ring<T, DUAL, EP, 8>(a, wg, st);
    return 0;
}

// The columns from n on, as a product of their own.
template <typename T, bool BKS>
static GmArgs gm_from(const GmArgs& a, int n)
{
    constexpr int ES = sizeof(typename T::elem);
    GmArgs b = a;
    b.N -= n;
    const int size = a.odt == 2 ? 4 : 2;   // GFL_F32
    for (int i = 0; i < 2; ++i)
    {
        if (b.B[i]) b.B[i] += (int64_t)n * (BKS ? ES : a.ldb);
        if (b.out[i]) b.out[i] = static_cast<char*>(b.out[i]) + (int64_t)n * size;
    }
    if (b.g) b.g += n;
    if (b.u) b.u += n;
    if (b.dg) b.dg = static_cast<char*>(b.dg) + (int64_t)n * 2;
    if (b.du) b.du = static_cast<char*>(b.du) + (int64_t)n * 2;
    if (b.sb) b.sb += n;
    return b;
}

template <typename T, bool AKS, bool BKS, bool DUAL, int EP>
static int gm_run(int form, int ep, int aligned, GmArgs& a, void* ws, size_t ws_bytes, int nz, hipStream_t st)
{
    if constexpr (!AKS && !BKS)
        if (a.M <= 16) return gm_few<T, DUAL, EP>(a, aligned, st);
    GmPlan p = gm_plan(form, ep, DUAL, aligned, a.M, a.N, a.K, a.segs, nz);
    if (p.part_bytes && (!ws || ws_bytes < p.part_bytes)) return -2;
    if (p.first)
    {
        GmArgs b = gm_from<T, BKS>(a, p.first);
        a.N = p.first;
        if (gm_tiles<T, AKS, BKS, DUAL, EP>(a, p, aligned, nz, st)) return -1;
        return gm_run<T, AKS, BKS, DUAL, EP>(form, ep, aligned, b, ws, ws_bytes, nz, st);
    }
    if (p.parts == 1) return gm_tiles<T, AKS, BKS, DUAL, EP>(a, p, aligned, nz, st);
    if constexpr (AKS) return -1;   // never split (gm_plan)
    else
    {
        GmArgs b = a;
        b.out[0] = ws;
        b.ldo = p.ldp;
        if (gm_tiles<T, AKS, BKS, DUAL, EP_PART>(b, p, aligned, 1, st)) return -1;
        const int64_t n = (int64_t)a.M * ((a.N + 3) / 4);
        hipLaunchKernelGGL((gm_join_kernel<T, DUAL, EP>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a,
                           (const void*)ws, p.ldp, p.parts);
        return 0;
    }
}

template <typename T>
static int launch_gemm(int form, int ep, int dual, int aligned, GmArgs& a, void* ws, size_t ws_bytes, int nz, hipStream_t st)
{
    if constexpr (sizeof(typename T::elem) == 1)
    {
        if (form == GM_NT && ep == EP_I8) return gm_run<T, false, false, false, EP_I8>(form, ep, aligned, a, ws, ws_bytes, nz, st);
    }
    else
    {
        if (form == GM_NT && ep == EP_GATE && dual) return gm_run<T, false, false, true, EP_GATE>(form, ep, aligned, a, ws, ws_bytes, nz, st);
        if (form == GM_NT && ep == EP_OUT) return gm_run<T, false, false, false, EP_OUT>(form, ep, aligned, a, ws, ws_bytes, nz, st);
        if (form == GM_NN && ep == EP_DACT) return gm_run<T, false, true, false, EP_DACT>(form, ep, aligned, a, ws, ws_bytes, nz, st);
        if (form == GM_NN && ep == EP_OUT) return gm_run<T, false, true, false, EP_OUT>(form, ep, aligned, a, ws, ws_bytes, nz, st);
        if (form == GM_TN && ep == EP_OUT) return gm_run<T, true, true, false, EP_OUT>(form, ep, aligned, a, ws, ws_bytes, nz, st);
    }
    return -1;
}

}  // namespace gfl
