// The choice of experts in its general form: scores (sigmoid or softmax), a bias for balance, groups, top-k, weights; and the
// gradient of the logits.
//
// The choice is that of fp64 scores: in fp32 some token in every few thousand has two experts beside the border that fp32 cannot tell
// apart (or ties, which then go by index). It is made in fp32 first, whose keys are known to within a margin; where two picks, or the
// last and what comes after it, lie closer, the candidates are ordered again by their fp64 keys, and where that does not settle it (a
// border between groups, a softmax with a bias, a crowd at the border) the token is chosen for in fp64 by the whole wave. Without a
// bias the logits themselves are compared, which order as the scores do and stay apart where those saturate; groups go by the scores.
//
// A token takes L lanes (64 / L tokens a wave). Its E experts lie in index order over the lanes, each group over lanes of its
// own, so that among equal keys the lowest lane's lowest place is the lowest index. A lane sorts its keys once; a pick is then the
// largest of the lanes' first ones, found by DPP, and a step down in one lane.
//
// Bound by the picks' chains of dependent instructions, not by bytes: 8192 tokens of 256 experts in 8 groups 11.9 to 14.5 us (bytes 1.9; some 920
// instructions a wave, 7.0 us of issue; 15.9 with a choice in fp64 throughout); 16384 tokens of 128, softmax without renormalisation in
// bf16, and their gradient 16.6 (7.6 and 9.2 by the tracer, bytes 2.2, issue 5.6 and 6.5); one token 5.0, 2.2 of them a launch's. What
// falls back to fp64 costs more: 8192 tokens of 256 experts, softmax 7.2, with a bias 16.5, with 8 groups 14.6, with both 18.8; sigmoid with
// 8 groups in fp32, fp16 and bf16, whose groups' worths tie more often, 10.0, 11.4 and 13.0.
#include "gfl_device.hpp"
#include "gfl_internal.hpp"

#include <type_traits>
#include <utility>

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

// What a token's lanes hold, joined by `op` (which is associative, commutative and, in a softmax's sum, the same in any lane): within rows of
// 16 by DPP (quads, then mirrored half rows and rows, whose quads are all equal by then), across rows by gfx950's swaps, which leave a
// lane both its own value and the other's.
template <int L, typename V, typename Op>
__device__ __forceinline__ V rt_all(V v, Op op)
{
    constexpr int N = sizeof(V) / 4;
    struct Words { uint32_t w[N]; };
    auto dpp = [&](auto ctrl) {
        Words a = __builtin_bit_cast(Words, v), b;
#pragma unroll
        for (int i = 0; i < N; ++i) b.w[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a.w[i], decltype(ctrl)::value, 0xF, 0xF, true);
        v = op(v, __builtin_bit_cast(V, b));
    };
    dpp(std::integral_constant<int, 0xB1>{});    // quad_perm 1, 0, 3, 2
    dpp(std::integral_constant<int, 0x4E>{});    // quad_perm 2, 3, 0, 1
    dpp(std::integral_constant<int, 0x141>{});   // row_half_mirror
    dpp(std::integral_constant<int, 0x140>{});   // row_mirror
    if constexpr (L >= 32)
    {
        const Words a = __builtin_bit_cast(Words, v);
        Words b, c;
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            const auto r = __builtin_amdgcn_permlane16_swap(a.w[i], a.w[i], false, false);
            b.w[i] = r[0], c.w[i] = r[1];
        }
        v = op(__builtin_bit_cast(V, b), __builtin_bit_cast(V, c));
    }
    if constexpr (L >= 64)
    {
        const Words a = __builtin_bit_cast(Words, v);
        Words b, c;
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            const auto r = __builtin_amdgcn_permlane32_swap(a.w[i], a.w[i], false, false);
            b.w[i] = r[0], c.w[i] = r[1];
        }
        v = op(__builtin_bit_cast(V, b), __builtin_bit_cast(V, c));
    }
    return v;
}
template <int L>
__device__ __forceinline__ uint32_t rt_max(uint32_t v)
{
    return rt_all<L>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int L>
__device__ __forceinline__ double rt_sum(double v)
{
    return rt_all<L>(v, [](double a, double b) { return a + b; });
}

// keys[0..N) into descending order by a merge exchange network (any N)
template <int N>
struct RtNet
{
    int a[N * 6 + 1] = {}, b[N * 6 + 1] = {}, n = 0;
    constexpr RtNet()
    {
        for (int p = 1; p < N; p *= 2)
            for (int k = p; k >= 1; k /= 2)
                for (int j = k % p; j + k < N; j += 2 * k)
                    for (int i = 0; i < k && i + j + k < N; ++i)
                        if ((i + j) / (2 * p) == (i + j + k) / (2 * p)) a[n] = i + j, b[n] = i + j + k, ++n;
    }
};
template <int N, size_t... I>
__device__ __forceinline__ void rt_sort(uint32_t (&key)[N], std::index_sequence<I...>)
{
    constexpr RtNet<N> net;
    auto swap = [&](auto at) {
        constexpr int x = net.a[decltype(at)::value], y = net.b[decltype(at)::value];
        const uint32_t hi = max(key[x], key[y]), lo = min(key[x], key[y]);
        key[x] = hi, key[y] = lo;
    };
    (swap(std::integral_constant<size_t, I>{}), ...);
}
template <int N>
__device__ __forceinline__ void rt_sort(uint32_t (&key)[N])
{
    constexpr RtNet<N> net;
    rt_sort(key, std::make_index_sequence<net.n>{});
}

// exp(x - top) of a softmax: experts at the maximum weigh 1 (also where it is +inf), those that are not there 0
__device__ __forceinline__ double rt_soft(float x, float top)
{
    return x == top ? 1.0 : x > -INFINITY ? exp((double)x - (double)top) : 0.0;
}
// The same within 2^-35, for what decides nothing: a whole row's weights and their sum. Taylor's series of degree 9 over |r| <= ln 2 / 2; an
// expert that is not there (NaN) goes to the lower end, which is 0.
__device__ __forceinline__ double rt_soft_near(float x, float top)
{
    const double d = fmax((double)x - (double)top, -750.0), n = rint(d * 1.4426950408889634), r = fma(n, -0.6931471805599453, d);
    double e = 1.0 / 362880;
    const double c[9] = { 1.0 / 40320, 1.0 / 5040, 1.0 / 720, 1.0 / 120, 1.0 / 24, 1.0 / 6, 0.5, 1.0, 1.0 };
#pragma unroll
    for (int i = 0; i < 9; ++i) e = fma(e, r, c[i]);
    return x == top ? 1.0 : ldexp(e, (int)n);
}
__device__ __forceinline__ double rt_sigmoid(float x) { return 1.0 / (1.0 + exp(-(double)x)); }
__device__ __forceinline__ float rt_unkey(uint32_t k)
{
    return k == 0 ? -INFINITY : __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// What experts of the kept groups are compared by without a bias: the logit. Beside a softmax's +inf the others' scores are all 0.
__device__ __forceinline__ float rt_rank(const RouteArgs& a, float x, float top)
{
    return a.softmax && top == INFINITY && x > -INFINITY ? (x == top ? 1.0f : 0.0f) : x;
}

__device__ __forceinline__ float rt_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// the lanes of a token in a ballot
template <int L>
__device__ __forceinline__ uint64_t rt_lanes(uint64_t all, int lane)
{
    if constexpr (L == 64) return all;
    else return all >> (lane / L * L) & ((1ull << L) - 1);
}

template <typename X, int NI>
__device__ __forceinline__ void rt_row(const X* p, int n, float (&x)[NI])   // n of NI neighbouring elements, -inf past them
{
    X e[NI] = {};
    if (n == NI) __builtin_memcpy(e, p, sizeof e);
    else if (n > 0)
#pragma unroll
        for (int i = 0; i < NI; ++i) e[i] = p[min(i, n - 1)];   // (all loads at once: behind a condition each waits for the one before)
#pragma unroll
    for (int i = 0; i < NI; ++i) x[i] = i < n ? static_cast<float>(e[i]) : -INFINITY;
}

// Which groups a lane's group is among the kept ones, by their worth (the sum of the one or two largest keys, given as v1 >= v2 of the
// lane's experts and left as the group's; -inf: none): how many come before it.
template <int L, typename V>
__device__ __forceinline__ int rt_group(const RouteArgs& a, int lpg, int lane, int g, V& v1, V& v2, V& worth)
{
    for (int w = 1; w < lpg; w *= 2)
    {
        const V o1 = __shfl_xor(v1, w), o2 = __shfl_xor(v2, w);
        v2 = fmax(fmax(v2, o2), fmin(v1, o1));
        v1 = fmax(v1, o1);
    }
    worth = a.group_best == 2 && v2 > -(V)INFINITY ? v1 + v2 : v1;
    int before = 0;
    for (int h = 0; h < a.groups; ++h)
    {
        const V o = __shfl(worth, lane / L * L + h * lpg);
        before += o > worth || (o == worth && h < g);
    }
    return before;
}

constexpr int RT_MORE = 6;   // candidates past the picks

enum
{
    RT_SURE = 0,
    RT_ORDER = 1,   // the candidates' order is to be looked at again
    RT_WIDE = 2,    // what fp32 says is not enough
};

// The choice in fp32: picks, and as many candidates more as lie within the margin of the last (`count` in all). Keys hold a place in the
// lane in their last bits and compare by the rest; a lane's are sorted once, so that its best is its first, and a pick moves
// the rest up. exact_keys: the places take no bits of the logits.
// Margins. Sigmoid: the argument's rounding and v_exp_f32 make 1.5 |x| 2^-24 + 2^-23 of exp(-x), which counts s (1 - s) times, 1 + exp
// and v_rcp_f32 1.5 2^-23 of s: below 2^-22. Softmax: the same of an exponential, 32 additions and a reciprocal of the sum: below 2^-18.
// Adding the bias takes 2^-24 of the key, the places up to PLACE 2^-23. Two keys, twice each; 2^-20 leaves as much again.
// A group's worth is off by its keys' errors, and their sum's rounding is at most 2^-24 of |v1| + |v2|, beside which the worth itself may be
// small (one expert forced by its bias, the others held off): margin + 2^-22 (|v1| + |v2|) is twice that.
template <int L, int NI, bool FULL>
__device__ __forceinline__ int rt_choose(const RouteArgs& a, int lane, int sub, int g, int e0, const float (&x)[NI], const float (&bias)[NI],
                                         float top, int* pick, bool exact_keys, int& count)
{
    constexpr uint32_t PLACE = NI > 16 ? 31 : NI > 8 ? 15 : NI > 4 ? 7 : NI > 2 ? 3 : NI > 1 ? 1 : 0;
    const float margin = a.softmax ? 0x1p-16f : 0x1p-20f;
    constexpr float STEP = (PLACE + 3) * 0x1p-23f;
    int state = RT_SURE;
    const bool by_score = FULL && a.bias;
    uint32_t key[NI];
    if constexpr (FULL)
    {
        float s[NI], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NI; ++i)
        {
            const float t = a.softmax ? (x[i] == top ? 1.0f : rt_exp(x[i] - top)) : rt_exp(-x[i]);
            s[i] = a.softmax ? t : __builtin_amdgcn_rcpf(1.0f + t);
            sum += x[i] > -INFINITY ? t : 0.0f;
        }
        if (a.softmax)
        {
            const float r = __builtin_amdgcn_rcpf((float)rt_sum<L>((double)sum));
#pragma unroll
            for (int i = 0; i < NI; ++i) s[i] *= r;
        }
#pragma unroll
        for (int i = 0; i < NI; ++i)
        {
            s[i] += bias[i];
            s[i] = x[i] > -INFINITY && s[i] == s[i] ? s[i] : -INFINITY;
        }
        bool kept = true;
        if (a.groups > 1)
        {
            float v1 = -INFINITY, v2 = -INFINITY, worth;
#pragma unroll
            for (int i = 0; i < NI; ++i)
            {
                v2 = fmaxf(v2, fminf(s[i], v1));
                v1 = fmaxf(v1, s[i]);
            }
            kept = rt_group<L, float>(a, a.lpg, lane, g, v1, v2, worth) < a.top_groups;
            const bool mine = g < a.groups;
            // (a group that has nothing is worth -inf, and no key of it is compared; of infinite sums nothing is known)
            const float off = v1 > -INFINITY ? margin + (fabsf(v1) + (a.group_best == 2 && v2 > -INFINITY ? fabsf(v2) : 0.0f)) * 0x1p-22f : 0.0f;
            const float least = worth - off, most = worth + off;
            const float in = -rt_unkey(rt_max<L>(mine && kept ? rt_key(least == least ? -least : INFINITY) : 0)),
                        out = rt_unkey(rt_max<L>(mine && !kept ? rt_key(most == most ? most : INFINITY) : 0));
            if (out > -INFINITY && !(in > out)) state = RT_WIDE;
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) key[i] = kept ? rt_key(by_score ? s[i] : rt_rank(a, x[i], top)) : 0;
    }
    else
#pragma unroll
        for (int i = 0; i < NI; ++i) key[i] = rt_key(x[i]);
#pragma unroll
    for (int i = 0; i < NI; ++i) key[i] = key[i] ? (key[i] & ~PLACE) | (PLACE - i) : 0;
    rt_sort(key);
    const int most = min(a.topk + RT_MORE, L);
    uint32_t least = 0, mine = 0;   // the last pick's key; lane i: candidate i's
    auto close = [&](uint32_t above, uint32_t m) {
        if (!by_score) return m != 0 && above == m;
        const float u = rt_unkey(above), v = rt_unkey(m);
        return m != 0 && !(u - v > margin + fmaxf(fabsf(u), fabsf(v)) * STEP);
    };
    for (count = 0;; ++count)
    {
        const uint32_t best = key[0] & ~PLACE, m = rt_max<L>(best);
        if (count >= a.topk)
        {
            const bool border = !exact_keys && close(least, m);
            if (!__any(border)) break;
            if (count >= most)
            {
                if (border) state = RT_WIDE;
                break;
            }
        }
        if (count < a.topk) least = m;
        mine = sub == count ? m : mine;
        bool win = best == m;
        const uint64_t all = __ballot(win);
        if (__popcll(all) != 64 / L || __any(m == 0))
        {
            // two lanes have it (the lower one counts), or a token has none left
            win = win && m != 0 && (rt_lanes<L>(all, lane) & ((1ull << sub) - 1)) == 0;
            if (m == 0 && sub == 0) pick[count] = -1;
        }
        if (win) pick[count] = e0 + (int)(PLACE - (key[0] & PLACE));
        // (by masks: of a select between two elements the compiler makes an index, and of that a chain of selects)
        const uint32_t gone = win ? ~0u : 0u;
#pragma unroll
        for (int i = 0; i + 1 < NI; ++i) key[i] = (key[i + 1] & gone) | (key[i] & ~gone);
        key[NI - 1] &= ~gone;
    }
    if (!exact_keys)
    {
        const uint32_t above = __shfl_up(mine, 1);
        const bool c = sub > 0 && sub < count && close(above, mine);
        if (rt_lanes<L>(__ballot(c), lane)) state |= RT_ORDER;
    }
    return state & RT_WIDE || (state && by_score && a.softmax) ? RT_WIDE : state;
}

// The choice in fp64. A pick is the maximum of the lanes' best keys: first of the upper 32 bits, then, where two lanes share those, of
// the lower.
template <int NI, bool FULL>
__device__ __forceinline__ void rt_choose_wide(const RouteArgs& a, int lpg, int lane, int g, int e0, int n, const float (&x)[NI], float top,
                                               int* pick)
{
    constexpr int L = 64;
    const int sub = lane;
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
            const double norm = rt_sum<L>(part);
#pragma unroll
            for (int i = 0; i < NI; ++i) s[i] /= norm;
        }
        constexpr double NONE = -(double)INFINITY;
        double v1 = NONE, v2 = NONE;
#pragma unroll
        for (int i = 0; i < NI; ++i)
        {
            if (a.bias && i < n) s[i] += (double)a.bias[e0 + i];
            const uint64_t k = x[i] > -INFINITY ? rt_key(s[i]) : 0;
            hi[i] = a.bias ? (uint32_t)(k >> 32) : rt_key(rt_rank(a, x[i], top)), lo[i] = a.bias ? (uint32_t)k : 0;
            const double v = k ? s[i] : NONE;
            v2 = fmax(v2, fmin(v, v1));
            v1 = fmax(v1, v);
        }
        if (a.groups > 1)
        {
            double worth;
            if (rt_group<L, double>(a, lpg, lane, g, v1, v2, worth) >= a.top_groups)
            {
#pragma unroll
                for (int i = 0; i < NI; ++i) hi[i] = lo[i] = 0;
            }
        }
    }
    else
#pragma unroll
        for (int i = 0; i < NI; ++i) hi[i] = rt_key(x[i]);
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
        uint64_t all = rt_lanes<L>(__ballot(best), lane);
        if constexpr (FULL)
            if (__any((all & (all - 1)) != 0))
            {
                const uint32_t ml = rt_max<L>(best ? bl : 0);
                best = best && bl == ml;
                all = rt_lanes<L>(__ballot(best), lane);
            }
        if (all == 0 ? sub == 0 : best && (all & ((1ull << sub) - 1)) == 0)
        {
            pick[j] = all ? e0 + at : -1;
#pragma unroll
            for (int i = 0; i < NI; ++i)
                if (i == at)
                {
                    hi[i] = 0;
                    if constexpr (FULL) lo[i] = 0;
                }
        }
    }
}

// NI: experts of a lane. FULL: scores are formed (for a bias, or groups).
template <typename X, int L, int NI, bool FULL>
__global__ __launch_bounds__(RT_T) void route_experts_kernel(RouteArgs a)
{
    constexpr int TOK = RT_T / L;
    __shared__ int picks[TOK][MAX_ROUTE_K];
    __shared__ uint64_t keys[TOK][L];
    const int lane = threadIdx.x % 64, sub = threadIdx.x % L, tok = threadIdx.x / L;
    const int64_t t = (int64_t)blockIdx.x * TOK + tok;
    const X* row = static_cast<const X*>(a.logits) + min(t, (int64_t)a.M - 1) * a.ld;
    // the lane's experts: e0 .. e0 + n - 1 of group g
    const int gs = a.E / a.groups;
    auto mine = [&](int l, int lpg, int per, int& g, int& e0, int& n) {
        const int s0 = l % lpg * per;
        g = l / lpg;
        e0 = min(g * gs + s0, a.E);
        n = g < a.groups ? min(per, max(gs - s0, 0)) : 0;
    };
    int g, e0, n;
    mine(sub, a.lpg, a.per, g, e0, n);
    float x[NI], bias[NI], top = 0.f;
    rt_row(row + e0, n, x);
#pragma unroll
    for (int i = 0; i < NI; ++i) bias[i] = 0.f;
    if (FULL && a.bias)
#pragma unroll
        for (int i = 0; i < NI; ++i) bias[i] = a.bias[min(e0 + i, a.E - 1)];   // (past the lane's experts there is no logit)
    if (a.softmax)
    {
        uint32_t k = 0;
#pragma unroll
        for (int i = 0; i < NI; ++i) k = max(k, rt_key(x[i]));
        top = rt_unkey(rt_max<L>(k));
    }
    int* pick = picks[tok];
    int count;
    const int state = rt_choose<L, NI, FULL>(a, lane, sub, g, e0, x, bias, top, pick, (!FULL || !a.bias) && sizeof(X) == 2, count);
    if (__any(state == RT_ORDER))
    {
        asm volatile("" ::: "memory");   // (LDS is read and written in order within a wave)
        const int e = sub < count ? pick[sub] : -1;
        uint64_t key = 0;
        if (e >= 0)
        {
            const float v = static_cast<float>(row[e]);
            if (FULL && a.bias) key = rt_key(rt_sigmoid(v) + (double)a.bias[e]);
            else key = rt_key((double)(FULL ? rt_rank(a, v, top) : v));
        }
        keys[tok][sub] = key;
        asm volatile("" ::: "memory");
        int before = 0;
        for (int c = 0; c < count; ++c)
        {
            const uint64_t k = keys[tok][c];
            before += k > key || (k == key && pick[c] < e);
        }
        asm volatile("" ::: "memory");
        if (state == RT_ORDER && e >= 0 && before < a.topk) pick[before] = e;
    }
    for (uint64_t left = __ballot(state == RT_WIDE && sub == 0); left; left &= left - 1)
    {
        constexpr int NW = (NI * L + 63) / 64;
        const int first = __builtin_ctzll(left), lpg = a.lpg * (64 / L);
        const int64_t tw = (int64_t)blockIdx.x * TOK + threadIdx.x / 64 * (64 / L) + first / L;
        const X* rw = static_cast<const X*>(a.logits) + min(tw, (int64_t)a.M - 1) * a.ld;
        int gw, ew, nw;
        mine(lane, lpg, (gs + lpg - 1) / lpg, gw, ew, nw);
        float xw[NW], topw = 0.f;
        rt_row(rw + ew, nw, xw);
        uint32_t k = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) k = max(k, rt_key(xw[i]));
        if (a.softmax) topw = rt_unkey(rt_max<64>(k));
        rt_choose_wide<NW, FULL>(a, lpg, lane, gw, ew, nw, xw, topw, picks[threadIdx.x / 64 * (64 / L) + first / L]);
    }
    __syncthreads();

    double norm = 1.0;
    if (a.softmax && !a.renorm)
    {
        double part = 0.0;
#pragma unroll
        for (int i = 0; i < NI; ++i) part += rt_soft_near(x[i], top);
        norm = rt_sum<L>(part);
    }
    double w[64 / L], sum = 0.0;
    float xs[64 / L];
    uint32_t k = 0;
#pragma unroll
    for (int r = 0; r < 64 / L; ++r)
    {
        xs[r] = -INFINITY;
        if (r * L >= a.topk) continue;
        const int j = r * L + sub, e = j < a.topk ? pick[j] : -1;
        if (e >= 0) xs[r] = static_cast<float>(row[e]);
        k = max(k, rt_key(xs[r]));
    }
    // Renormalised, a softmax's own sum cancels: its exponentials are taken from the picks' largest logit, as the gradient's are, so that picks
    // far below the row's (a bias can choose them) have weights too.
    if (a.softmax && a.renorm) top = rt_unkey(rt_max<L>(k));
#pragma unroll
    for (int r = 0; r < 64 / L; ++r)
    {
        w[r] = xs[r] > -INFINITY ? a.softmax ? rt_soft(xs[r], top) : rt_sigmoid(xs[r]) : 0.0;
        sum += w[r];
    }
    if (a.renorm) norm = rt_sum<L>(sum);
    if (t >= a.M) return;
    norm = norm > 0.0 ? (double)a.scale / norm : 0.0;
#pragma unroll
    for (int r = 0; r < 64 / L; ++r)
    {
        const int j = r * L + sub;
        if (j >= a.topk) continue;
        a.sel[t * a.topk + j] = pick[j];
        rt_store(a.w, a.wdtype, t * a.topk + j, w[r] * norm);
    }
}

// With S = the sum of the picked scores s_j (1 without renormalisation) and c the scale, w_j = c s_j / S:
//   ds_j = c / S (dw_j - sum_i dw_i s_i / S), without renormalisation c dw_j;
//   sigmoid: dx = ds s (1 - s) at the picks, 0 elsewhere;
//   softmax p: dx = p (ds - sum_i ds_i p_i) everywhere; with renormalisation that sum is 0 and only ratios of the picks' exponentials
//   enter, so the row is not read.
// Where one expert has nearly the whole row, ds and the sum agree in all but a few bits of its own dx: they stay in fp64 up to the result, and
// the picks' p are those of the row's pass (near exponentials are still a softmax's, so that what cancels is the same on both sides).
template <typename X, int L, int NI>
__global__ __launch_bounds__(RT_T) void route_backward_kernel(RouteArgs a, const void* dw, const int64_t* sel, X* dx, int64_t ldx)
{
    constexpr int TOK = RT_T / L;
    __shared__ int picks[TOK][MAX_ROUTE_K];
    __shared__ double grads[TOK][MAX_ROUTE_K];
    const int sub = threadIdx.x % L, tok = threadIdx.x / L;
    const int64_t t = (int64_t)blockIdx.x * TOK + tok, tc = min(t, (int64_t)a.M - 1);
    const X* row = static_cast<const X*>(a.logits) + tc * a.ld;
    const bool dense = a.softmax && !a.renorm;
    const int e0 = min(sub * a.per, a.E), n = min(a.per, a.E - e0);

    float top = -INFINITY, xs[64 / L], up[64 / L];
    int es[64 / L];
    uint32_t k = 0;
    double p[NI], norm = 1.0;
    float x[NI];
    if (dense) rt_row(row + e0, n, x);
#pragma unroll
    for (int r = 0; r < 64 / L; ++r)
    {
        es[r] = -1, xs[r] = -INFINITY, up[r] = 0.f;
        if (r * L >= a.topk) continue;
        const int j = r * L + sub;
        const int64_t e = j < a.topk ? sel[tc * a.topk + j] : -1;
        if (j < a.topk) up[r] = rt_load(dw, a.wdtype, tc * a.topk + j);
        es[r] = e >= 0 && e < a.E ? (int)e : -1;
        if (es[r] >= 0) xs[r] = static_cast<float>(row[es[r]]);
        else up[r] = 0.f;   // (a missing pick's may be anything)
        k = max(k, rt_key(xs[r]));
    }
    if (dense)
#pragma unroll
        for (int i = 0; i < NI; ++i) k = max(k, rt_key(x[i]));
    if (a.softmax) top = rt_unkey(rt_max<L>(k));
    if (dense)
    {
        norm = 0.0;
#pragma unroll
        for (int i = 0; i < NI; ++i) norm += p[i] = rt_soft_near(x[i], top);
        norm = rt_sum<L>(norm);
        norm = norm > 0.0 ? 1.0 / norm : 0.0;   // (a row of NaN has no experts)
    }
    double s[64 / L], total = 0.0, dot = 0.0;
#pragma unroll
    for (int r = 0; r < 64 / L; ++r)
    {
        s[r] = 0.0;
        if (r * L >= a.topk) continue;
        if (es[r] >= 0) s[r] = dense ? rt_soft_near(xs[r], top) * norm : a.softmax ? rt_soft(xs[r], top) : rt_sigmoid(xs[r]);
        total += s[r];
        dot += s[r] * ((double)a.scale * up[r]);
    }
    total = rt_sum<L>(total);
    dot = rt_sum<L>(dot);
    const double by = total > 0.0 ? 1.0 / total : 0.0;
#pragma unroll
    for (int r = 0; r < 64 / L; ++r)
    {
        const int j = r * L + sub;
        if (j >= a.topk) continue;
        double ds = (double)a.scale * up[r];
        if (a.renorm) ds = (ds - dot * by) * by;
        picks[tok][j] = es[r];
        // dense: ds, of the whole row's p (ds - dot); else the pick's dx (sigmoid: s (1 - s) = s sigmoid(-x))
        grads[tok][j] = es[r] < 0 ? 0.0 : dense ? ds : ds * s[r] * (a.softmax ? 1.0 : rt_sigmoid(-xs[r]));
    }
    __syncthreads();
    if (t >= a.M) return;
    double v[NI] = {};
    for (int j = 0; j < a.topk; ++j)
    {
        const int at = picks[tok][j] - e0, e = at < n ? at : -1;
        const double d = grads[tok][j];
#pragma unroll
        for (int i = 0; i < NI; ++i) v[i] += e == i ? d : 0.0;
    }
    X o[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) o[i] = static_cast<X>((float)(dense ? p[i] * norm * (v[i] - dot) : v[i]));
    X* out = dx + t * ldx + e0;
    if (n == NI) __builtin_memcpy(out, o, sizeof o);
    else
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (i < n) out[i] = o[i];
}

// Experts of a lane that kernels are made for, of each number of lanes.
template <int L>
constexpr auto rt_sizes()
{
    if constexpr (L == 16) return std::integer_sequence<int, 1, 2, 4, 8, 16>{};
    else if constexpr (L == 32) return std::integer_sequence<int, 2, 4, 8, 12, 16, 32>{};
    else return std::integer_sequence<int, 1, 2, 4, 5, 8, 16, 32>{};
}
// calls f with the first that holds `per`
template <typename F, int... N>
static bool rt_sized(int per, std::integer_sequence<int, N...>, F f)
{
    return ((per <= N ? (f(std::integral_constant<int, N>{}), true) : false) || ...);
}

template <typename X, int L>
static int route_go(const RouteArgs& a, hipStream_t st)
{
    const dim3 grid((unsigned)(((int64_t)a.M + RT_T / L - 1) / (RT_T / L))), block(RT_T);
    const bool done = rt_sized(a.per, rt_sizes<L>(), [&](auto n) {
        constexpr int N = decltype(n)::value;
        if (a.bias || a.groups > 1) hipLaunchKernelGGL((route_experts_kernel<X, L, N, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((route_experts_kernel<X, L, N, false>), grid, block, 0, st, a);
    });
    return done ? 0 : -1;
}

template <typename X, int L>
static void route_back(const RouteArgs& a, const void* dw, const int64_t* sel, void* dx, int64_t ldx, hipStream_t st)
{
    const dim3 grid((unsigned)(((int64_t)a.M + RT_T / L - 1) / (RT_T / L))), block(RT_T);
    rt_sized(a.per, rt_sizes<L>(), [&](auto n) {
        hipLaunchKernelGGL((route_backward_kernel<X, L, decltype(n)::value>), grid, block, 0, st, a, dw, sel, static_cast<X*>(dx), ldx);
    });
}

// Lanes a token. 16 or 32 do the steps of a pick for 4 or 2 tokens at once, 64 hold fewer experts each and are done sooner. us by 64, 32
// and 16 lanes (16 are 32 where a lane would hold more than 16 experts), 1024, 2048, 4096, 6144, 8192, 12288 and 16384 tokens:
//   288 experts, sigmoid and bias  6.1 7.7 -, 6.8 8.1 -, 8.5 9.9 -, 11.1 11.4 -, 13.3 12.6 -, 17.6 16.8 -, 22.4 20.3 -
//   256 in 8 groups, the same      7.6 8.6 10.4, 7.4 7.9 9.7, 10.4 11.1 11.6, 13.0 12.6 14.2, 14.8 13.2 13.7, 19.2 15.9 15.7, 24.8 20.0 19.0
//   128 experts, softmax           4.6 4.5 4.8, 4.9 4.6 4.8, 6.1 4.8 5.1, 7.4 5.2 5.0, 8.9 5.8 5.3, 11.7 7.3 5.7, 14.6 8.7 6.5
// The edges are those of the larger routers; 128 experts and fewer would take 32 lanes from 1024 tokens on and 16 from 6144 (1.3 us of 6).
template <typename X>
static int route_of(RouteArgs& a, hipStream_t st)
{
    int lanes = 1;   // for each group
    while (lanes < a.groups) lanes *= 2;
    const int size = a.E / a.groups;
    auto per = [&](int L) { return (size + L / lanes - 1) / (L / lanes); };
    int L = a.M < 6144 ? 64 : a.M < 12288 ? 32 : 16;
    while (L < 64 && (lanes > L || per(L) > L || a.topk + 1 > L)) L *= 2;
    a.lpg = L / lanes;
    a.per = per(L);
    return L == 16 ? route_go<X, 16>(a, st) : L == 32 ? route_go<X, 32>(a, st) : route_go<X, 64>(a, st);
}

int launch_route_experts(RouteArgs& a, hipStream_t st)
{
    return a.dtype == 2 ? route_of<float>(a, st) : a.dtype == 1 ? route_of<__bf16>(a, st) : route_of<_Float16>(a, st);
}

// 16 lanes a token where each then has a power of two of experts, which it stores as one vector. us by 64 and 16 lanes, sigmoid renormalised in
// fp32 and softmax not renormalised in bf16: 128 experts 4096 tokens 5.0 4.5, 5.9 5.4, 8192 7.6 5.4, 8.9 6.2, 16384 13.4 8.3, 15.5 8.9;
// 256 experts 4096 tokens 5.9 7.3, 7.0 7.5, 8192 9.3 9.1, 11.1 9.2, 16384 16.5 14.2, 20.3 15.0; 160 (10 a lane) 8192 8.9 9.5, 11.3 10.2, 16384
// 16.0 14.8, 20.3 15.3. 288 and 384 experts, more than 16 a lane, 8192 tokens by 64 lanes 10.5 and 13.1, 13.0 and 16.8.
template <typename X>
static void route_back_of(RouteArgs& a, const void* dw, const int64_t* sel, void* dx, int64_t ldx, hipStream_t st)
{
    a.per = (a.E + 15) / 16;
    if (a.M >= 8192 && a.E % 16 == 0 && (a.per & (a.per - 1)) == 0 && a.per <= 16) return route_back<X, 16>(a, dw, sel, dx, ldx, st);
    a.per = (a.E + 63) / 64;
    route_back<X, 64>(a, dw, sel, dx, ldx, st);
}

void launch_route_backward(RouteArgs& a, const void* dw, const int64_t* sel, void* dx, int64_t ldx, hipStream_t st)
{
    (a.dtype == 2 ? &route_back_of<float> : a.dtype == 1 ? &route_back_of<__bf16> : &route_back_of<_Float16>)(a, dw, sel, dx, ldx, st);
}

}  // namespace gfl
