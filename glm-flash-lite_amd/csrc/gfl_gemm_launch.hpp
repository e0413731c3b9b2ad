// Tile choice and launches of the tile GEMM for one input type; included by one translation unit per type.
#pragma once
#include "gfl_gemm.hpp"
#include "gfl_gemm_plan.hpp"

namespace gfl {

template <typename T, int TM, int TN, int WM, int WN, bool AKS, bool BKS, bool DUAL, int NST, bool AL, int EP>
static int gm_go(const GmArgs& a, int nz, hipStream_t st)
{
    constexpr int lds = (AL ? NST : 1) * (TM + TN) * 128;
    static_assert(lds <= LDS_LIMIT, "tiles fit the LDS");
    auto* kern = gm_kernel<T, TM, TN, WM, WN, AKS, BKS, DUAL, NST, AL, EP>;
    static const bool opened = hipFuncSetAttribute(reinterpret_cast<const void*>(kern),
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, lds) == hipSuccess;
    (void)opened;
    hipLaunchKernelGGL(kern, dim3((unsigned)(a.tm * a.tn), a.parts, nz), dim3(WM * WN * 64), lds, st, a);
    return 0;
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
    if (p.tm == 64) return gm_go<T, 64, 128, 1, 4, AKS, BKS, DUAL, 3, true, EP>(a, nz, st);
    if (p.tm == 128) return gm_go<T, 128, 128, 2, 2, AKS, BKS, DUAL, 2, true, EP>(a, nz, st);
    return gm_go<T, 256, 256, 2, 4, AKS, BKS, DUAL, 2, true, EP>(a, nz, st);
}

template <typename T, bool AKS, bool BKS, bool DUAL, int EP>
static int gm_run(int form, int ep, int aligned, GmArgs& a, void* ws, size_t ws_bytes, int nz, hipStream_t st)
{
    if constexpr (!AKS && !BKS && EP != EP_PART)
        if (a.M <= 16)
        {
            const int per = DUAL ? 8 : 16, wg = (a.N + per - 1) / per;
            // waves of a workgroup: enough loads in flight over the card's CUs, few workgroups taking more waves each
            if (wg <= 768) hipLaunchKernelGGL((gm_skinny_kernel<T, DUAL, EP, 16>), dim3(wg), dim3(1024), 0, st, a);
            else if (wg <= 2048) hipLaunchKernelGGL((gm_skinny_kernel<T, DUAL, EP, 8>), dim3(wg), dim3(512), 0, st, a);
            else hipLaunchKernelGGL((gm_skinny_kernel<T, DUAL, EP, 4>), dim3(wg), dim3(256), 0, st, a);
            return 0;
        }
    GmPlan p = gm_plan(form, ep, DUAL, aligned, a.M, a.N, a.K, a.segs);
    if (p.parts > 1 && (!ws || ws_bytes < p.part_bytes)) return -2;
    if (p.parts == 1) return gm_tiles<T, AKS, BKS, DUAL, EP>(a, p, aligned, nz, st);
    if constexpr (EP == EP_DACT || AKS) return -1;   // never split (gm_plan)
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
