// Token selection from logits: temperature, top-k, top-p, min-p, then the draw for a given uniform number.
//
// The three filters each keep a prefix of the logits in descending order (equal logits by index), so the kept set is the
// shortest prefix: a threshold key and the number of logits equal to it that are kept. Keys are the logits' bits as
// unsigned integers in their order. Weights exp((x - max) / T) are fp64, rounded to whole units of 2^-43: their sums are
// integer sums, the same in any order.
#include "gfl_internal.hpp"

namespace gfl {

constexpr int SM_T = 1024, SM_W = SM_T / 64, SM_BINS = 2048;
constexpr uint32_t SM_MASKED = 0x007FFFFFu;   // key of -inf: logits at or below are never drawn

__device__ __forceinline__ uint32_t sm_key(float x)
{
    if (x != x) return SM_MASKED;
    const uint32_t b = __float_as_uint(x + 0.0f);   // -0 -> +0: equal logits have equal keys
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sm_value(uint32_t key)
{
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

struct SmRow
{
    const void* p;
    int dtype;
    __device__ __forceinline__ uint32_t key(int i) const
    {
        float x;
        if (dtype == 2) x = static_cast<const float*>(p)[i];
        else if (dtype == 1) x = static_cast<float>(static_cast<const __bf16*>(p)[i]);
        else x = static_cast<float>(static_cast<const _Float16*>(p)[i]);
        return sm_key(x);
    }
};

// exp((x - max) / T) as 2^n p, n the nearest whole number to the exponent in base 2 and p by the Taylor series of e^x on
// |x| <= ln 2 / 2, whose remainder after degree 12 is below 2^-51. scale = log2(e) / T.
__device__ __forceinline__ double sm_exp(uint32_t key, uint32_t top, double scale)
{
    if (key == top) return 1.0;
    double y = ((double)sm_value(key) - (double)sm_value(top)) * scale;
    if (!(y > -1000.0)) return 0.0;   // also a NaN: finite - inf over an infinite T
    const double n = rint(y), x = (y - n) * 0.693147180559945309417;
    double p = 1.0 / 479001600;
    p = fma(p, x, 1.0 / 39916800);
    p = fma(p, x, 1.0 / 3628800);
    p = fma(p, x, 1.0 / 362880);
    p = fma(p, x, 1.0 / 40320);
    p = fma(p, x, 1.0 / 5040);
    p = fma(p, x, 1.0 / 720);
    p = fma(p, x, 1.0 / 120);
    p = fma(p, x, 1.0 / 24);
    p = fma(p, x, 1.0 / 6);
    p = fma(p, x, 0.5);
    p = fma(p, x, 1.0);
    p = fma(p, x, 1.0);
    return __longlong_as_double(__double_as_longlong(p) + ((long long)(int)n << 52));
}

// a weight in units of 2^-43 of the largest logit's: added to 2^52, the last bit of the sum is a unit
__device__ __forceinline__ uint64_t sm_units(double e)
{
    return (uint64_t)__double_as_longlong(fma(e, 0x1p43, 0x1p52)) & 0xFFFFFFFFFFFFFull;
}
__device__ __forceinline__ uint64_t sm_weight(uint32_t key, uint32_t top, double scale)
{
    return key > SM_MASKED ? sm_units(sm_exp(key, top, scale)) : 0;
}

template <typename V>
__device__ __forceinline__ V sm_wave_sum(V v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

struct SmShared
{
    uint32_t cnt[SM_BINS];
    unsigned long long mass[SM_BINS];
    uint32_t wcnt[SM_W];
    unsigned long long wmass[SM_W];
    uint32_t prefix;
    unsigned long long above;      // weight (by weight) or count (by count) above the found bin
    unsigned long long above_mass;
    uint32_t in_bin;
};

// The key at which the descending order reaches `want`: by weight (mode 1) the first key with (weight at or above it) >=
// want, by count (mode 0) the key of the want-th logit. Returns it; s.above = weight / count strictly above that key,
// s.above_mass the weight strictly above, s.in_bin how many logits have it. Three passes of 11, 11, 10 bits.
__device__ uint32_t sm_select(SmShared& s, const SmRow& row, int V, uint32_t top, double scale, int mode,
                              unsigned long long want)
{
    uint32_t prefix = 0;
    unsigned long long above = 0, above_mass = 0;
    for (int level = 0; level < 3; ++level)
    {
        const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
        for (int i = threadIdx.x; i < SM_BINS; i += SM_T) s.cnt[i] = 0, s.mass[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < V; i += SM_T)
        {
            const uint32_t k = row.key(i);
            if (level == 0 || (k >> (shift + bits)) == prefix)
            {
                const uint32_t b = (k >> shift) & ((1u << bits) - 1);
                atomicAdd(&s.cnt[b], 1u);
                const uint64_t w = sm_weight(k, top, scale);
                if (w) atomicAdd(&s.mass[b], (unsigned long long)w);
            }
        }
        __syncthreads();
        if (threadIdx.x == 0)
        {
            unsigned long long c = above, m = above_mass;
            int b = (1 << bits) - 1;
            for (; b > 0; --b)
            {
                const unsigned long long step = mode ? s.mass[b] : s.cnt[b];
                if (c + step >= want && s.cnt[b]) break;
                c += step;
                m += s.mass[b];
            }
            s.prefix = (uint32_t)b;
            s.above = c;
            s.above_mass = m;
            s.in_bin = s.cnt[b];
        }
        __syncthreads();
        prefix = (prefix << bits) | s.prefix;
        above = s.above;
        above_mass = s.above_mass;
    }
    __syncthreads();
    return prefix;
}

// The whole selection of a row by one workgroup, for rows whose threshold bin is too full for the list (many equal logits, or a
// large top-k): three-level selects over the row, which it reads some eight times.
__device__ void sm_row_slow(SmShared& s, const SampleArgs& a, int b, const SmRow& row, uint32_t top, double scale)
{
    const int V = a.V, lane = threadIdx.x % 64, wave = threadIdx.x / 64;

    // the kept prefix: keys above `cut`, and the first `ties` of those equal to it
    uint32_t cut = 0;
    unsigned long long ties = ~0ull;
    unsigned long long total = 0;   // weight of the top-k
    const int k = a.top_k ? a.top_k[b] : 0;
    if (k > 0 && k < V)
    {
        cut = sm_select(s, row, V, top, scale, 0, (unsigned long long)k);
        ties = (unsigned long long)k - s.above;
        total = s.above_mass + ties * sm_weight(cut, top, scale);
        __syncthreads();
    }
    const float p = a.top_p ? a.top_p[b] : 1.0f;
    if (p < 1.0f)
    {
        if (cut == 0)
        {
            unsigned long long m = 0;
            for (int i = threadIdx.x; i < V; i += SM_T) m += sm_weight(row.key(i), top, scale);
            m = sm_wave_sum(m);
            if (lane == 0) s.wmass[wave] = m;
            __syncthreads();
            for (int w = 0; w < SM_W; ++w) total += s.wmass[w];
            __syncthreads();
        }
        const double goal = (double)p * (double)total;
        const unsigned long long want = goal > 1.0 ? (unsigned long long)ceil(goal) : 1ull;
        const uint32_t pc = sm_select(s, row, V, top, scale, 1, want);
        const unsigned long long w = sm_weight(pc, top, scale);
        unsigned long long t = w ? (want - s.above + w - 1) / w : 1;
        if (pc > cut || (pc == cut && t < ties)) cut = pc, ties = t;
        __syncthreads();
    }
    const float mp = a.min_p ? a.min_p[b] : 0.0f;
    auto kept_by_min = [&](uint32_t key) { return !(mp > 0.0f) || key == top || sm_exp(key, top, scale) >= (double)mp; };

    // each wave takes a run of the row: weight and ties of its run, then the wave that holds the drawn token walks it
    const int per = (V + SM_W * 64 - 1) / (SM_W * 64) * 64, lo = wave * per, hi = min(V, lo + per);
    uint32_t nt = 0;
    for (int i = lo + lane; i < hi; i += 64) nt += row.key(i) == cut;
    nt = sm_wave_sum(nt);
    if (lane == 0) s.wcnt[wave] = nt;
    __syncthreads();
    unsigned long long tie0 = 0;
    for (int w = 0; w < wave; ++w) tie0 += s.wcnt[w];
    auto walk = [&](auto&& use) {   // use(index, weight or 0) over the run, in order, wave by wave of 64
        unsigned long long seen = tie0;
        for (int i0 = lo; i0 < hi; i0 += 64)
        {
            const int i = i0 + lane;
            const uint32_t key = i < hi ? row.key(i) : 0;
            const bool tie = i < hi && key == cut;
            const unsigned long long bal = __ballot(tie);
            const unsigned long long r = seen + __popcll(bal & ((1ull << lane) - 1));
            seen += __popcll(bal);
            const bool keep = i < hi && (key > cut || (tie && r < ties)) && kept_by_min(key);
            if (use(i, keep ? (unsigned long long)sm_weight(key, top, scale) : 0ull)) break;
        }
    };
    unsigned long long mine = 0;
    walk([&](int, unsigned long long w) {
        mine += w;
        return false;
    });
    mine = sm_wave_sum(mine);
    if (lane == 0) s.wmass[wave] = mine;
    __syncthreads();
    unsigned long long sum = 0, before = 0;
    int last = 0;   // the last wave with weight
    for (int w = 0; w < SM_W; ++w)
    {
        if (w < wave) before += s.wmass[w];
        if (s.wmass[w]) last = w;
        sum += s.wmass[w];
    }
    const double target = fmax((double)a.u[b] * (double)sum, 0.0);   // a NaN too becomes 0
    // this wave's run holds the first index whose cumulative weight exceeds the target (or is the last, should none)
    const bool start_le = !((double)before > target), end_gt = (double)(before + mine) > target;
    const bool hold = mine && start_le && (end_gt || wave == last);
    if (hold)
    {
        unsigned long long cum = before;
        int tok = -1;
        unsigned long long tw = 0;
        walk([&](int i, unsigned long long w) {
            unsigned long long c = w;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1)
            {
                const unsigned long long v = __shfl_up(c, o);
                if (lane >= o) c += v;
            }
            c += cum;
            const unsigned long long hit = __ballot(w && (double)c > target), any = __ballot(w != 0);
            cum = __shfl(c, 63);
            const int l = hit ? __ffsll(hit) - 1 : any ? 63 - __clzll(any) : -1;
            if (l >= 0)
            {
                tok = __shfl(i, l);
                tw = __shfl(w, l);
            }
            return hit != 0;
        });
        if (lane == 0)
        {
            a.token[b] = tok;
            if (a.prob) a.prob[b] = (float)((double)tw / (double)sum);
        }
    }
}


// ---- the launches ----
//
// A row is cut into S slices, a workgroup each, so that a few rows fill the card (B = 1, V = 131,072: 64 workgroups; the same
// work in one workgroup took 547 us). Four launches:
//   top     each slice's largest and smallest logit and the largest's index; clears the row's histogram
//   bins    2,047 bins of equal width from the largest logit down to where weights round to zero (or to the smallest), and
//           one for what lies below: logits per bin, and where the nucleus needs it their weight
//   cut     every workgroup finds the bin in which the kept prefix ends from the row's histogram. With a top-k (and few
//           logits down to its bin) all logits down to that bin go into the row's list; else the list takes the bin alone
//           and each slice sums the weight of its logits above it
//   pick    a workgroup per row sorts the list, finds the threshold in it, and draws: from the list itself (top-k), or
//           from the slice in which the target lies
constexpr int SM_LIST = 4096;         // logits a row's list holds (32 KB of LDS)
constexpr int SM_LISTK = 1024;        // top-k up to which the list is expected to hold the whole kept set
constexpr int SM_PT = 256;            // threads of the slice launches
constexpr int SM_MAXS = 256;          // slices of a row

struct SmSlice
{
    uint32_t top, low;                // largest key, smallest key above -inf (0, ~0 without any)
    int32_t arg;                      // lowest index of the largest
    int32_t pad;
    unsigned long long mass;          // weight above the cut bin (of the kept by min-p)
};
enum
{
    SM_ALL = 0,                       // every logit kept (but for min-p): draw from the slices
    SM_BIN = 1,                       // the list holds the bin where the nucleus ends
    SM_TOPK = 2,                      // the list holds everything that may be kept
    SM_SLOW = 3,
};
struct SmState                        // of a row
{
    int32_t count;                    // list entries
    int32_t mode;
    unsigned long long want, above;   // SM_BIN: weight at which the nucleus ends, weight above the bin
};
struct SmWs
{
    uint32_t* cnt;                    // [B][SM_BINS]
    unsigned long long* mass;         // [B][SM_BINS]
    unsigned long long* list;         // [B][SM_LIST] key << 32 | ~index
    SmSlice* slice;                   // [B][S]
    SmState* state;                   // [B]
    int S, len;                       // slices of a row, logits of a slice
};

static void sm_split(int B, int V, int& S, int& len)
{
    const int want = (1024 + B - 1) / B;                     // four workgroups a CU
    S = V / 2048 < 1 ? 1 : V / 2048;
    if (S > want) S = want;
    if (S > SM_MAXS) S = SM_MAXS;
    len = ((V + S - 1) / S + 3) / 4 * 4;
    S = (V + len - 1) / len;
}

static size_t sm_carve(void* base, int B, int V, SmWs& w)
{
    sm_split(B, V, w.S, w.len);
    char* p = static_cast<char*>(base);
    auto take = [&](size_t n) {
        char* r = p;
        p += (n + 255) / 256 * 256;
        return r;
    };
    w.mass = reinterpret_cast<unsigned long long*>(take((size_t)B * SM_BINS * 8));
    w.list = reinterpret_cast<unsigned long long*>(take((size_t)B * SM_LIST * 8));
    w.slice = reinterpret_cast<SmSlice*>(take((size_t)B * w.S * sizeof(SmSlice)));
    w.state = reinterpret_cast<SmState*>(take((size_t)B * sizeof(SmState)));
    w.cnt = reinterpret_cast<uint32_t*>(take((size_t)B * SM_BINS * 4));
    return (size_t)(p - static_cast<char*>(base));
}

// use(index, key) for this thread's logits of [lo, hi): 4 neighbours at a time, 4 loads in flight (`first`: the first 4, loaded
// ahead of what the launch waits for otherwise)
template <typename E, int NT>
struct SmBatch
{
    typedef E vec __attribute__((ext_vector_type(4)));
    vec v[4];
    __device__ __forceinline__ void load(const E* row, int i, int hi)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * NT * 4 + 4 <= hi) __builtin_memcpy(&v[j], row + i + j * NT * 4, sizeof(vec));
    }
};
template <typename E, int NT, typename F>
__device__ __forceinline__ void sm_each(const E* row, int lo, int hi, SmBatch<E, NT> b, F&& use)
{
    for (int i = lo + (int)threadIdx.x * 4; i < hi;)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            const int at = i + j * NT * 4;
            if (at + 4 <= hi)
            {
#pragma unroll
                for (int k = 0; k < 4; ++k) use(at + k, sm_key(static_cast<float>(b.v[j][k])));
            }
            else
                for (int k = at; k < hi; ++k) use(k, sm_key(static_cast<float>(row[k])));   // the slice's last, not whole, chunk
        }
        i += 4 * NT * 4;
        b.load(row, i, hi);
    }
}

// what every launch after the first knows of a row
struct SmHead
{
    uint32_t top, low;
    int arg;
    bool done;            // greedy, or nothing to draw from
    bool wide;            // a range past fp32: no bins
    float T, top_x, bins; // bins per unit of logit
    double scale;
    __device__ __forceinline__ int bin(uint32_t key) const
    {
        return key == top ? 0 : (int)fminf((top_x - sm_value(key)) * bins, (float)(SM_BINS - 1));
    }
};

__device__ __forceinline__ SmHead sm_head(const SampleArgs& a, const SmWs& w, int b)
{
    SmHead h;
    uint32_t top = 0, low = ~0u;
    int arg = 0x7FFFFFFF;
    const int lane = threadIdx.x % 64;
    for (int s = lane; s < w.S; s += 64)
    {
        const SmSlice& c = w.slice[(size_t)b * w.S + s];
        if (c.top > top) top = c.top, arg = c.arg;   // slices in order: the first of equals has the lowest index
        low = min(low, c.low);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1)
    {
        const uint32_t t = (uint32_t)__shfl_xor((int)top, o);
        const int f = __shfl_xor(arg, o);
        if (t > top || (t == top && f < arg)) top = t, arg = f;
        low = min(low, (uint32_t)__shfl_xor((int)low, o));
    }
    h.top = top;
    h.low = low;
    h.arg = arg;
    h.T = a.temperature ? a.temperature[b] : 1.0f;
    h.done = top <= SM_MASKED || !(h.T > 0.0f);
    h.top_x = sm_value(top);
    h.scale = 1.4426950408889634074 / (double)h.T;
    // down to the smallest logit (a little past it, so that it lies in a bin of its own right) or to where weights round to
    // zero units: what falls into the last bin, below the range, weighs nothing
    const float range = fmaxf(fminf((h.top_x - sm_value(low)) * 1.001f, 31.0f * h.T), 1e-30f);
    h.bins = (float)(SM_BINS - 1) / range;
    h.wide = !(range < __builtin_inff());
    return h;
}

template <typename E>
__global__ __launch_bounds__(SM_PT) void sm_top_kernel(SampleArgs a, SmWs w)
{
    const int b = blockIdx.y, s = blockIdx.x, lo = s * w.len, hi = min(a.V, lo + w.len);
    const E* row = static_cast<const E*>(a.logits) + (int64_t)b * a.ld;
    for (int i = s * SM_PT + threadIdx.x; i < SM_BINS; i += w.S * SM_PT)
    {
        w.cnt[(size_t)b * SM_BINS + i] = 0;
        w.mass[(size_t)b * SM_BINS + i] = 0;
    }
    if (s == 0 && threadIdx.x == 0) w.state[b].count = 0;
    SmBatch<E, SM_PT> first;
    first.load(row, lo + threadIdx.x * 4, hi);
    uint32_t top = 0, low = ~0u;
    int arg = 0x7FFFFFFF;
    sm_each<E, SM_PT>(row, lo, hi, first, [&](int i, uint32_t k) {
        if (k > top) top = k, arg = i;
        if (k > SM_MASKED) low = min(low, k);
    });
    __shared__ uint32_t st[SM_PT / 64], sl[SM_PT / 64];
    __shared__ int sa[SM_PT / 64];
#pragma unroll
    for (int o = 32; o; o >>= 1)
    {
        const uint32_t t = (uint32_t)__shfl_xor((int)top, o);
        const int f = __shfl_xor(arg, o);
        if (t > top || (t == top && f < arg)) top = t, arg = f;
        low = min(low, (uint32_t)__shfl_xor((int)low, o));
    }
    if (threadIdx.x % 64 == 0) st[threadIdx.x / 64] = top, sl[threadIdx.x / 64] = low, sa[threadIdx.x / 64] = arg;
    __syncthreads();
    if (threadIdx.x == 0)
    {
        for (int i = 1; i < SM_PT / 64; ++i)
        {
            if (st[i] > top || (st[i] == top && sa[i] < arg)) top = st[i], arg = sa[i];
            low = min(low, sl[i]);
        }
        SmSlice& c = w.slice[(size_t)b * w.S + s];
        c.top = top;
        c.low = low;
        c.arg = arg;
        c.mass = 0;
    }
}

__device__ __forceinline__ int sm_topk(const SampleArgs& a, int b)
{
    const int k = a.top_k ? a.top_k[b] : 0;
    return k > 0 && k < a.V ? k : 0;
}
__device__ __forceinline__ float sm_topp(const SampleArgs& a, int b)
{
    const float p = a.top_p ? a.top_p[b] : 1.0f;
    return p < 1.0f ? p : 1.0f;
}

template <typename E>
__global__ __launch_bounds__(SM_PT) void sm_bins_kernel(SampleArgs a, SmWs w)
{
    __shared__ uint32_t cnt[SM_BINS];
    __shared__ unsigned long long mass[SM_BINS];
    const int b = blockIdx.y, s = blockIdx.x, lo = s * w.len, hi = min(a.V, lo + w.len);
    const E* row = static_cast<const E*>(a.logits) + (int64_t)b * a.ld;
    SmBatch<E, SM_PT> first;
    first.load(row, lo + threadIdx.x * 4, hi);
    const SmHead h = sm_head(a, w, b);
    const int k = sm_topk(a, b);
    const bool p = sm_topp(a, b) < 1.0f;
    if (h.done || h.wide || (!k && !p)) return;
    const bool weigh = p && (!k || k > SM_LISTK);   // a small top-k's list gives its weights itself
    for (int i = threadIdx.x; i < SM_BINS; i += SM_PT) cnt[i] = 0, mass[i] = 0;
    __syncthreads();
    if (weigh)
        sm_each<E, SM_PT>(row, lo, hi, first, [&](int, uint32_t key) {
            if (key <= SM_MASKED) return;
            const int bin = h.bin(key);
            atomicAdd(&cnt[bin], 1u);
            if (bin < SM_BINS - 1) atomicAdd(&mass[bin], (unsigned long long)sm_weight(key, h.top, h.scale));
        });
    else
        sm_each<E, SM_PT>(row, lo, hi, first, [&](int, uint32_t key) {
            if (key > SM_MASKED) atomicAdd(&cnt[h.bin(key)], 1u);
        });
    __syncthreads();
    for (int i = threadIdx.x; i < SM_BINS; i += SM_PT)
    {
        if (cnt[i]) atomicAdd(&w.cnt[(size_t)b * SM_BINS + i], cnt[i]);
        if (mass[i]) atomicAdd(&w.mass[(size_t)b * SM_BINS + i], mass[i]);
    }
}

// exclusive sum over the workgroup's threads in order; `total` gets the sum of all. NT / 64 slots of scratch.
template <int NT>
__device__ __forceinline__ unsigned long long sm_scan(unsigned long long v, unsigned long long* scratch,
                                                      unsigned long long& total)
{
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    unsigned long long c = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
    {
        const unsigned long long t = __shfl_up(c, o);
        if (lane >= o) c += t;
    }
    __syncthreads();
    if (lane == 63) scratch[wave] = c;
    __syncthreads();
    unsigned long long before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i)
    {
        if (i < wave) before += scratch[i];
        total += scratch[i];
    }
    return before + c - v;
}

// the bin in which the kept prefix of a row ends, and the row's mode
struct SmCut
{
    int mode, bin;
    unsigned long long want, above;
};
__device__ SmCut sm_cut(const SampleArgs& a, const SmWs& w, int b, const SmHead& h, unsigned long long* scratch, int* found)
{
    constexpr int PER = SM_BINS / SM_PT;
    const int k = sm_topk(a, b);
    const float p = sm_topp(a, b);
    SmCut c = { SM_ALL, SM_BINS, 0, 0 };
    if (!k && !(p < 1.0f)) return c;
    if (h.wide)
    {
        c.mode = SM_SLOW;
        return c;
    }
    const uint32_t* cnt = w.cnt + (size_t)b * SM_BINS + threadIdx.x * PER;
    const unsigned long long* mass = w.mass + (size_t)b * SM_BINS + threadIdx.x * PER;
    if (threadIdx.x == 0) found[0] = -1, found[1] = 0;
    unsigned long long n = 0, total;
    uint32_t each[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) n += each[i] = cnt[i];
    unsigned long long at = sm_scan<SM_PT>(n, scratch, total);
    bool topk = false;
    if (k && (k <= SM_LISTK || total > (unsigned long long)k))
    {
        // the bin of the k-th logit; all of them where the row has no more
        const unsigned long long want = total < (unsigned long long)k ? total : (unsigned long long)k;
#pragma unroll
        for (int i = 0; i < PER; ++i)
        {
            const int bin = threadIdx.x * PER + i;
            // a prefix that ends in the last bin is the one before it: what lies there weighs nothing
            if (at < want && at + each[i] >= want)
                found[0] = min(bin, SM_BINS - 2), found[1] = (int)(bin == SM_BINS - 1 ? at : at + each[i]);
            at += each[i];
        }
        topk = true;
    }
    else if (p < 1.0f)
    {
        unsigned long long m = 0, eachm[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) m += eachm[i] = mass[i];
        at = sm_scan<SM_PT>(m, scratch, total);
        const double goal = (double)p * (double)total;
        c.want = goal > 1.0 ? (unsigned long long)ceil(goal) : 1ull;
#pragma unroll
        for (int i = 0; i < PER; ++i)
        {
            if (at < c.want && at + eachm[i] >= c.want)
            {
                found[0] = threadIdx.x * PER + i;
                found[1] = (int)each[i];
                scratch[SM_PT / 64] = at;
            }
            at += eachm[i];
        }
    }
    else return c;   // a top-k that keeps every logit
    __syncthreads();
    c.bin = found[0];
    c.mode = found[1] > SM_LIST ? SM_SLOW : topk ? SM_TOPK : SM_BIN;
    if (!topk) c.above = scratch[SM_PT / 64];
    return c;
}

template <typename E>
__global__ __launch_bounds__(SM_PT) void sm_cut_kernel(SampleArgs a, SmWs w)
{
    __shared__ unsigned long long scratch[SM_PT / 64 + 1];
    __shared__ int found[2];
    const int b = blockIdx.y, s = blockIdx.x, lo = s * w.len, hi = min(a.V, lo + w.len);
    const E* row = static_cast<const E*>(a.logits) + (int64_t)b * a.ld;
    SmBatch<E, SM_PT> first;
    first.load(row, lo + threadIdx.x * 4, hi);
    const SmHead h = sm_head(a, w, b);
    if (h.done) return;
    const SmCut c = sm_cut(a, w, b, h, scratch, found);
    if (s == 0 && threadIdx.x == 0)
    {
        w.state[b].mode = c.mode;
        w.state[b].want = c.want;
        w.state[b].above = c.above;
    }
    if (c.mode == SM_SLOW) return;
    unsigned long long* list = w.list + (size_t)b * SM_LIST;
    auto put = [&](int i, uint32_t key) {
        const int at = atomicAdd(&w.state[b].count, 1);
        if (at < SM_LIST) list[at] = (unsigned long long)key << 32 | (uint32_t)~i;
    };
    if (c.mode == SM_TOPK)
    {
        sm_each<E, SM_PT>(row, lo, hi, first, [&](int i, uint32_t key) {
            if (key > SM_MASKED && h.bin(key) <= c.bin) put(i, key);
        });
        return;
    }
    const float mp = a.min_p ? a.min_p[b] : 0.0f;
    const double m = mp > 0.0f ? (double)mp : 0.0;
    unsigned long long mine = 0, total;
    sm_each<E, SM_PT>(row, lo, hi, first, [&](int i, uint32_t key) {
        if (key <= SM_MASKED) return;
        const int bin = c.mode == SM_ALL ? 0 : h.bin(key);
        if (bin > c.bin) return;
        if (bin == c.bin) put(i, key);
        else
        {
            const double e = sm_exp(key, h.top, h.scale);
            if (key == h.top || e >= m) mine += sm_units(e);
        }
    });
    sm_scan<SM_PT>(mine, scratch, total);
    if (threadIdx.x == 0) w.slice[(size_t)b * w.S + s].mass = total;
}

// descending bitonic sort of n (a power of two) entries in LDS. A wave's 64 exchanges over distances up to 64 stay within
// its own 128 entries, so only the longer ones need a barrier.
__device__ __forceinline__ void sm_sort(unsigned long long* v, int n)
{
    __syncthreads();
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j; j >>= 1)
        {
            for (int t = threadIdx.x; t < n / 2; t += SM_T)
            {
                const int i = 2 * t - (t & (j - 1)), l = i + j;
                const unsigned long long x = v[i], y = v[l];
                if ((x < y) == ((i & k) == 0)) v[i] = y, v[l] = x;
            }
            if (j > 64 || (j == 1 && k >= 128)) __syncthreads();
            else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    __syncthreads();
}

template <typename E>
__global__ __launch_bounds__(SM_T) void sm_pick_kernel(SampleArgs a, SmWs w)
{
    __shared__ union
    {
        SmShared slow;
        struct
        {
            unsigned long long list[SM_LIST];
            unsigned long long scratch[SM_W];
            unsigned long long part[SM_MAXS];
            unsigned long long cut, at;
            int n, pick;
        } f;
    } sh;
    const int b = blockIdx.x, V = a.V;
    // loaded ahead of the head: the list's entries of this thread (those past its end are not used) and a slice's weight
    const unsigned long long* list = w.list + (size_t)b * SM_LIST;
    unsigned long long entry[SM_LIST / SM_T], slice_mass = 0;
#pragma unroll
    for (int j = 0; j < SM_LIST / SM_T; ++j) entry[j] = list[threadIdx.x + j * SM_T];
    if ((int)threadIdx.x < w.S) slice_mass = w.slice[(size_t)b * w.S + threadIdx.x].mass;
    const SmState st = w.state[b];
    const SmHead h = sm_head(a, w, b);
    if (h.done)
    {
        if (threadIdx.x == 0)
        {
            const bool none = h.top <= SM_MASKED;
            a.token[b] = none ? -1 : h.arg;
            if (a.prob) a.prob[b] = none ? 0.0f : 1.0f;
        }
        return;
    }
    const E* rowp = static_cast<const E*>(a.logits) + (int64_t)b * a.ld;
    if (st.mode == SM_SLOW)
    {
        SmRow row;
        row.dtype = a.dtype;
        row.p = rowp;
        sm_row_slow(sh.slow, a, b, row, h.top, h.scale);
        return;
    }
    const float mpf = a.min_p ? a.min_p[b] : 0.0f;
    const double mp = mpf > 0.0f ? (double)mpf : 0.0;
    const double u = (double)a.u[b];
    auto& f = sh.f;
    const int n = st.mode == SM_ALL ? 0 : min(st.count, SM_LIST);
    int pow2 = 2;
    while (pow2 < n) pow2 <<= 1;
    constexpr int PER = SM_LIST / SM_T;   // entries of a thread: 4 neighbours
    unsigned long long total = 0;
    if (threadIdx.x == 0) f.n = n, f.pick = -1;
    if (n)
    {
#pragma unroll
        for (int j = 0; j < SM_LIST / SM_T; ++j)
        {
            const int i = threadIdx.x + j * SM_T;
            if (i < pow2) f.list[i] = i < n ? entry[j] : 0;
        }
        sm_sort(f.list, pow2);
    }
    else __syncthreads();
    // weight of a list entry; the masked never enter the list
    auto exp_of = [&](unsigned long long e) { return sm_exp((uint32_t)(e >> 32), h.top, h.scale); };
    const int k = sm_topk(a, b);
    if (n)
    {
        // how many entries of the sorted list are kept
        const int lim = st.mode == SM_TOPK ? min(n, k) : n;
        unsigned long long wt[PER], mine = 0, sum;
        bool drop[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j)
        {
            const int i = threadIdx.x * PER + j;
            const double e = i < lim ? exp_of(f.list[i]) : 0.0;
            drop[j] = i < lim && e < mp && (uint32_t)(f.list[i] >> 32) != h.top;
            wt[j] = sm_units(e);
            mine += wt[j];
        }
        unsigned long long at = sm_scan<SM_T>(mine, f.scratch, sum);
        unsigned long long want = st.want;
        if (st.mode == SM_TOPK)
        {
            const float p = sm_topp(a, b);
            const double goal = p < 1.0f ? (double)p * (double)sum : (double)sum;
            want = p < 1.0f ? (goal > 1.0 ? (unsigned long long)ceil(goal) : 1ull) : ~0ull;
        }
        else at += st.above;
        int keep = lim;
#pragma unroll
        for (int j = 0; j < PER; ++j)
        {
            const int i = threadIdx.x * PER + j;
            if (i < lim && at < want && at + wt[j] >= want) keep = min(keep, i + 1);
            if (drop[j]) keep = min(keep, i);
            at += wt[j];
        }
        if (keep < lim) atomicMin(&f.n, keep);
        else if (threadIdx.x == 0) atomicMin(&f.n, lim);
        __syncthreads();
    }
    const int kept = f.n;
    if (st.mode == SM_TOPK)
    {
        // the kept entries in index order
        __syncthreads();
        int p2 = 2;
        while (p2 < kept) p2 <<= 1;
        unsigned long long mv[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j)
        {
            const int i = threadIdx.x + j * SM_T;
            if (i < p2) mv[j] = i < kept ? f.list[i] << 32 | f.list[i] >> 32 : 0;   // ~index first: descending is by index
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j)
        {
            const int i = threadIdx.x + j * SM_T;
            if (i < p2) f.list[i] = mv[j];
        }
        sm_sort(f.list, p2);
        unsigned long long wt[PER], mine = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j)
        {
            const int i = threadIdx.x * PER + j;
            wt[j] = i < kept ? sm_units(exp_of(f.list[i] << 32)) : 0;
            mine += wt[j];
        }
        unsigned long long at = sm_scan<SM_T>(mine, f.scratch, total);
        const double target = fmax(u * (double)total, 0.0);   // a NaN too becomes 0
#pragma unroll
        for (int j = 0; j < PER; ++j)
        {
            const int i = threadIdx.x * PER + j;
            // the first entry past the target, or the last with weight where none is
            if (wt[j] && !((double)at > target) && ((double)(at + wt[j]) > target || at + wt[j] == total))
            {
                a.token[b] = (int32_t)~(uint32_t)(f.list[i] >> 32);
                if (a.prob) a.prob[b] = (float)((double)wt[j] / (double)total);
            }
            at += wt[j];
        }
        return;
    }
    // from the slices: their weight above the bin and that of the list's kept entries
    if ((int)threadIdx.x < w.S) f.part[threadIdx.x] = slice_mass;
    __syncthreads();
    for (int i = threadIdx.x; i < kept; i += SM_T)
    {
        const uint32_t idx = ~(uint32_t)f.list[i];
        atomicAdd(&f.part[idx / (uint32_t)w.len], (unsigned long long)sm_units(exp_of(f.list[i])));
    }
    if (threadIdx.x == 0) f.cut = st.mode == SM_ALL ? 0 : kept ? f.list[kept - 1] : ~0ull;
    __syncthreads();
    // the last kept entry as key and index; an empty list keeps what lies above the bin, which starts at the list's first
    const unsigned long long none_above = n ? f.list[0] : 0;
    const unsigned long long cut = f.cut;
    unsigned long long at = 0;
    const unsigned long long mine = (int)threadIdx.x < w.S ? f.part[threadIdx.x] : 0;
    at = sm_scan<SM_T>(mine, f.scratch, total);
    const double target = fmax(u * (double)total, 0.0);
    if (mine && !((double)at > target) && ((double)(at + mine) > target || at + mine == total))
        f.pick = (int)threadIdx.x, f.at = at;
    __syncthreads();
    const int s = f.pick, lo = s * w.len, hi = min(V, lo + w.len), per = (hi - lo + SM_T - 1) / SM_T;
    const int i0 = lo + (int)threadIdx.x * per, i1 = min(hi, i0 + per);
    const unsigned long long base = f.at;
    auto weight = [&](int i) -> unsigned long long {
        const uint32_t key = sm_key(static_cast<float>(rowp[i]));
        if (key <= SM_MASKED) return 0;
        const unsigned long long e = (unsigned long long)key << 32 | (uint32_t)~i;
        if (cut == ~0ull ? e <= none_above : e < cut) return 0;
        const double x = sm_exp(key, h.top, h.scale);
        return key == h.top || x >= mp ? sm_units(x) : 0;
    };
    unsigned long long sum = 0, all;
    for (int i = i0; i < i1; ++i) sum += weight(i);
    unsigned long long c = base + sm_scan<SM_T>(sum, f.scratch, all);
    const unsigned long long end = base + all;
    if (sum && !((double)c > target) && ((double)(c + sum) > target || c + sum == end))
        for (int i = i0; i < i1; ++i)
        {
            const unsigned long long x = weight(i);
            if (!x) continue;
            c += x;
            if ((double)c > target || c == end)
            {
                a.token[b] = i;
                if (a.prob) a.prob[b] = (float)((double)x / (double)total);
                break;
            }
        }
}

size_t sample_ws_bytes(int B, int V)
{
    SmWs w;
    return B ? sm_carve(nullptr, B, V, w) : 0;
}

template <typename E>
static void sm_go(const SampleArgs& a, const SmWs& w, hipStream_t st)
{
    const dim3 grid(w.S, a.B);
    hipLaunchKernelGGL(sm_top_kernel<E>, grid, dim3(SM_PT), 0, st, a, w);
    if (a.top_k || a.top_p) hipLaunchKernelGGL(sm_bins_kernel<E>, grid, dim3(SM_PT), 0, st, a, w);
    hipLaunchKernelGGL(sm_cut_kernel<E>, grid, dim3(SM_PT), 0, st, a, w);
    hipLaunchKernelGGL(sm_pick_kernel<E>, dim3(a.B), dim3(SM_T), 0, st, a, w);
}

void launch_sample(const SampleArgs& a, hipStream_t st)
{
    SmWs w;
    sm_carve(a.ws, a.B, a.V, w);
    if (a.dtype == 2) sm_go<float>(a, w, st);
    else if (a.dtype == 1) sm_go<__bf16>(a, w, st);
    else sm_go<_Float16>(a, w, st);
}

}  // namespace gfl
