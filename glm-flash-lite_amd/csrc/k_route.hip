// The choice of experts in its general form: scores (sigmoid or softmax), a bias for balance, groups, top-k, weights; and the
// gradient of the logits.
//
// Scores are fp64: a choice is a comparison of scores + bias, and in fp32 some token in every few thousand has two experts beside
// the border that fp32 cannot tell apart (or ties, which then go by index). Without a bias and groups the logits
// themselves are compared, which order as the scores do.
//
// A token takes L lanes (64 / L tokens a wave). Its E experts lie in index order over the lanes, each group over lanes of its
// own, so that among equal keys the lowest lane's lowest place is the lowest index. A pick is the maximum of the lanes' best keys:
// first of the keys' upper 32 bits, then, where two lanes share those, of the lower.
#include "gfl_device.hpp"
#include "gfl_internal.hpp"

namespace gfl {

constexpr int RT_T = 256;   // threads of a workgroup

__device__ __forceinline__ float rt_load(const void* p, int dtype, int64_t i)
{
    if (dtype == 2) return static_cast<const float*>(p)[i];
    if (dtype == 1) return static_cast<float>(static_cast<const __bf16*>(p)[i]);
    return static_cast<float>(static_cast<const _Float16*>(p)[i]);
}
__device__ __forceinline__ void rt_store(void* p, int dtype, int64_t i, double v)
{
    if (dtype == 2) static_cast<float*>(p)[i] = (float)v;
    else if (dtype == 1) static_cast<__bf16*>(p)[i] = static_cast<__bf16>((float)v);
    else static_cast<_Float16*>(p)[i] = static_cast<_Float16>((float)v);
}

// keys: unsigned integers in the order of the values, 0 for an expert that is not to be picked (NaN, -inf)
__device__ __forceinline__ uint32_t rt_key(float x)
{
    const uint32_t b = __float_as_uint(x + 0.0f);   // -0 -> +0
    return x > -INFINITY ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
}
__device__ __forceinline__ uint64_t rt_key(double x)
{
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return x > -(double)INFINITY ? (b >> 63 ? ~b : b | 1ull << 63) : 0ull;
}

template <int W>
__device__ __forceinline__ uint32_t rt_xor(uint32_t v)
{
    return __float_as_uint(lane_xor<W>(__uint_as_float(v)));
}
template <int W>
__device__ __forceinline__ double rt_xor(double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)rt_xor<W>((uint32_t)(b >> 32)) << 32 | rt_xor<W>((uint32_t)b)));
}
template <int L>
__device__ __forceinline__ uint32_t rt_max(uint32_t v)   // over a token's lanes
{
    v = max(v, rt_xor<1>(v));
    v = max(v, rt_xor<2>(v));
    v = max(v, rt_xor<4>(v));
    v = max(v, rt_xor<8>(v));
    if constexpr (L >= 32) v = max(v, rt_xor<16>(v));
    if constexpr (L >= 64) v = max(v, rt_xor<32>(v));
    return v;
}
template <int L>
__device__ __forceinline__ double rt_sum(double v)
{
    v += rt_xor<1>(v);
    v += rt_xor<2>(v);
    v += rt_xor<4>(v);
    v += rt_xor<8>(v);
    if constexpr (L >= 32) v += rt_xor<16>(v);
    if constexpr (L >= 64) v += rt_xor<32>(v);
    return v;
}

// exp(x - top) of a softmax: experts at the maximum weigh 1 (also where it is +inf), those that are not there 0
__device__ __forceinline__ double rt_soft(float x, float top)
{
    return x == top ? 1.0 : x > -INFINITY ? exp((double)x - (double)top) : 0.0;
}
__device__ __forceinline__ double rt_sigmoid(float x) { return 1.0 / (1.0 + exp(-(double)x)); }
__device__ __forceinline__ float rt_unkey(uint32_t k)
{
    return k == 0 ? -INFINITY : __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// NI: experts of a lane. FULL: the keys are scores + bias (a bias, or groups); else the logits.
template <int L, int NI, bool FULL>
__global__ __launch_bounds__(RT_T) void route_experts_kernel(RouteArgs a)
{
    constexpr int TOK = RT_T / L;
    __shared__ int pick[TOK][64];
    const int lane = threadIdx.x % 64, sub = threadIdx.x % L, tok = threadIdx.x / L;
    const int64_t t = (int64_t)blockIdx.x * TOK + tok, row = min(t, (int64_t)a.M - 1) * a.ld;
    // the lane's experts: e0 .. e0 + n - 1 of group g
    const int g = sub / a.lpg, gs = a.E / a.groups, per = (gs + a.lpg - 1) / a.lpg, s0 = sub % a.lpg * per;
    const int e0 = g * gs + s0, n = g < a.groups ? min(per, gs - s0) : 0;

    float x[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) x[i] = -INFINITY;
#pragma unroll
    for (int i = 0; i < NI; ++i)
        if (i < n) x[i] = rt_load(a.logits, a.dtype, row + e0 + i);

    float top = 0.f;
    double norm = 1.0;
    if (a.softmax)
    {
        uint32_t k = 0;
#pragma unroll
        for (int i = 0; i < NI; ++i) k = max(k, rt_key(x[i]));
        top = rt_unkey(rt_max<L>(k));
    }
    uint32_t hi[NI], lo[FULL ? NI : 1];
    if constexpr (FULL)
    {
        double s[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) s[i] = a.softmax ? rt_soft(x[i], top) : rt_sigmoid(x[i]);
        if (a.softmax)
        {
            double part = 0.0;
#pragma unroll
            for (int i = 0; i < NI; ++i) part += s[i];
            norm = rt_sum<L>(part);
#pragma unroll
            for (int i = 0; i < NI; ++i) s[i] /= norm;
        }
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (a.bias && i < n) s[i] += (double)a.bias[e0 + i];
#pragma unroll
        for (int i = 0; i < NI; ++i)
        {
            const uint64_t k = x[i] > -INFINITY ? rt_key(s[i]) : 0;
            hi[i] = (uint32_t)(k >> 32), lo[i] = (uint32_t)k;
        }
        if (a.groups > 1)
        {
            // a group is worth the sum of its one or two largest keys
            constexpr double NONE = -(double)INFINITY;
            double v1 = NONE, v2 = NONE;
#pragma unroll
            for (int i = 0; i < NI; ++i)
            {
                const double v = hi[i] | lo[i] ? s[i] : NONE;
                v2 = fmax(v2, fmin(v, v1));
                v1 = fmax(v1, v);
            }
            for (int w = 1; w < a.lpg; w *= 2)
            {
                const double o1 = __shfl_xor(v1, w), o2 = __shfl_xor(v2, w);
                v2 = fmax(fmax(v2, o2), fmin(v1, o1));
                v1 = fmax(v1, o1);
            }
            const double worth = a.group_best == 2 && v2 > NONE ? v1 + v2 : v1;
            int before = 0;
            for (int h = 0; h < a.groups; ++h)
            {
                const double o = __shfl(worth, lane / L * L + h * a.lpg);
                before += o > worth || (o == worth && h < g);
            }
            if (before >= a.top_groups)
            {
#pragma unroll
                for (int i = 0; i < NI; ++i) hi[i] = lo[i] = 0;
            }
        }
    }
    else
    {
#pragma unroll
        for (int i = 0; i < NI; ++i) hi[i] = rt_key(x[i]);
        if (a.softmax && !a.renorm)
        {
            double part = 0.0;
#pragma unroll
            for (int i = 0; i < NI; ++i) part += rt_soft(x[i], top);
            norm = rt_sum<L>(part);
        }
    }

    for (int j = 0; j < a.topk; ++j)
    {
        uint32_t bh = hi[0], bl = FULL ? lo[0] : 0;
        int at = 0;
#pragma unroll
        for (int i = 1; i < NI; ++i)
        {
            const uint32_t l = FULL ? lo[i] : 0;
            const bool more = FULL ? ((uint64_t)hi[i] << 32 | l) > ((uint64_t)bh << 32 | bl) : hi[i] > bh;
            bh = more ? hi[i] : bh;
            bl = more ? l : bl;
            at = more ? i : at;
        }
        const uint32_t m = rt_max<L>(bh);
        bool best = bh == m && m != 0;
        constexpr uint64_t MASK = L == 64 ? ~0ull : (1ull << (L % 64)) - 1;
        uint64_t all = __ballot(best) >> (lane / L * L) & MASK;
        if constexpr (FULL)
            if (__any((all & (all - 1)) != 0))
            {
                const uint32_t ml = rt_max<L>(best ? bl : 0);
                best = best && bl == ml;
                all = __ballot(best) >> (lane / L * L) & MASK;
            }
        if (all == 0 ? sub == 0 : best && (all & ((1ull << sub) - 1)) == 0)
        {
            pick[tok][j] = all ? e0 + at : -1;
#pragma unroll
            for (int i = 0; i < NI; ++i)
                if (i == at)
                {
                    hi[i] = 0;
                    if constexpr (FULL) lo[i] = 0;
                }
        }
    }
    __syncthreads();

    double w[64 / L], sum = 0.0;
#pragma unroll
    for (int r = 0; r < 64 / L; ++r)
    {
        const int j = r * L + sub, e = j < a.topk ? pick[tok][j] : -1;
        w[r] = 0.0;
        if (e >= 0)
        {
            const float v = rt_load(a.logits, a.dtype, row + e);
            w[r] = a.softmax ? rt_soft(v, top) / norm : rt_sigmoid(v);
        }
        sum += w[r];
    }
    if (a.renorm) norm = rt_sum<L>(sum);
    else norm = 1.0;
    if (t >= a.M) return;
#pragma unroll
    for (int r = 0; r < 64 / L; ++r)
    {
        const int j = r * L + sub;
        if (j >= a.topk) continue;
        a.sel[t * a.topk + j] = pick[tok][j];
        rt_store(a.w, a.wdtype, t * a.topk + j, norm > 0.0 ? (double)a.scale * w[r] / norm : 0.0);
    }
}

// With S = the sum of the picked scores s_j (1 without renormalisation) and c the scale, w_j = c s_j / S:
//   ds_j = c / S (dw_j - sum_i dw_i s_i / S), without renormalisation c dw_j;
//   sigmoid: dx = ds s (1 - s) at the picks, 0 elsewhere;
//   softmax p: dx = p (ds - sum_i ds_i p_i) everywhere; with renormalisation that sum is 0 and only ratios of the picks' exponentials
//   enter, so the row is not read.
template <int L>
__global__ __launch_bounds__(RT_T) void route_backward_kernel(RouteArgs a, const void* dw, const int64_t* sel, void* dx, int64_t ldx)
{
    constexpr int TOK = RT_T / L;
    __shared__ int pick[TOK][64];
    __shared__ float grad[TOK][64];
    const int sub = threadIdx.x % L, tok = threadIdx.x / L;
    const int64_t t = (int64_t)blockIdx.x * TOK + tok, tc = min(t, (int64_t)a.M - 1), row = tc * a.ld;
    const bool dense = a.softmax && !a.renorm;

    float top = -INFINITY, xs[64 / L];
    int es[64 / L];
    uint32_t k = 0;
#pragma unroll
    for (int r = 0; r < 64 / L; ++r)
    {
        const int j = r * L + sub;
        const int64_t e = j < a.topk ? sel[tc * a.topk + j] : -1;
        es[r] = e >= 0 && e < a.E ? (int)e : -1;
        xs[r] = es[r] >= 0 ? rt_load(a.logits, a.dtype, row + es[r]) : -INFINITY;
        k = max(k, rt_key(xs[r]));
    }
    double norm = 1.0;
    if (dense)
        for (int e = sub; e < a.E; e += L) k = max(k, rt_key(rt_load(a.logits, a.dtype, row + e)));
    if (a.softmax) top = rt_unkey(rt_max<L>(k));
    if (dense)
    {
        double part = 0.0;
        for (int e = sub; e < a.E; e += L) part += rt_soft(rt_load(a.logits, a.dtype, row + e), top);
        norm = rt_sum<L>(part);
    }
    double s[64 / L], d[64 / L], total = 0.0, dot = 0.0;
#pragma unroll
    for (int r = 0; r < 64 / L; ++r)
    {
        const int j = r * L + sub;
        s[r] = d[r] = 0.0;
        if (es[r] >= 0)
        {
            s[r] = a.softmax ? rt_soft(xs[r], top) / norm : rt_sigmoid(xs[r]);
            d[r] = (double)a.scale * rt_load(dw, a.wdtype, tc * a.topk + j);
        }
        total += s[r];
        dot += s[r] * d[r];
    }
    total = rt_sum<L>(total);
    dot = rt_sum<L>(dot);
#pragma unroll
    for (int r = 0; r < 64 / L; ++r)
    {
        const int j = r * L + sub;
        double ds = d[r];
        if (a.renorm) ds = total > 0.0 ? (ds - dot / total) / total : 0.0;
        if (j < a.topk)
        {
            pick[tok][j] = es[r];
            // softmax: what is added to -p dot; sigmoid: s (1 - s) = s sigmoid(-x)
            grad[tok][j] = es[r] < 0 ? 0.f : (float)(ds * s[r] * (a.softmax ? 1.0 : rt_sigmoid(-xs[r])));
        }
    }
    __syncthreads();
    if (t >= a.M) return;
    for (int e = sub; e < a.E; e += L)
    {
        float v = 0.f;
        if (dense) v = (float)(-dot * rt_soft(rt_load(a.logits, a.dtype, row + e), top) / norm);
        for (int j = 0; j < a.topk; ++j)
            if (pick[tok][j] == e) v += grad[tok][j];
        rt_store(dx, a.dtype, t * ldx + e, v);
    }
}

template <int L, bool FULL>
static int route_go(const RouteArgs& a, int per, hipStream_t st)
{
    const dim3 grid((unsigned)(((int64_t)a.M + RT_T / L - 1) / (RT_T / L))), block(RT_T);
#define GFL_RT(N)                                                                                   \
    if (per <= N)                                                                                   \
    {                                                                                               \
        hipLaunchKernelGGL((route_experts_kernel<L, N, FULL>), grid, block, 0, st, a);              \
        return 0;                                                                                   \
    }
    GFL_RT(1) GFL_RT(2) GFL_RT(4) GFL_RT(5) GFL_RT(8) GFL_RT(16) GFL_RT(32)
#undef GFL_RT
    return -1;
}

int launch_route_experts(RouteArgs& a, hipStream_t st)
{
    int lanes = 1;   // for each group, of 64
    while (lanes < a.groups) lanes *= 2;
    a.lpg = 64 / lanes;
    const int size = a.E / a.groups, per = (size + a.lpg - 1) / a.lpg;
    return a.bias || a.groups > 1 ? route_go<64, true>(a, per, st) : route_go<64, false>(a, per, st);
}

void launch_route_backward(const RouteArgs& a, const void* dw, const int64_t* sel, void* dx, int64_t ldx, hipStream_t st)
{
    const dim3 grid((unsigned)(((int64_t)a.M + 3) / 4));
    hipLaunchKernelGGL(route_backward_kernel<64>, grid, dim3(RT_T), 0, st, a, dw, sel, dx, ldx);
}

}  // namespace gfl
