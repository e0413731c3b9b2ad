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

// exp((x - max) / T) = 2^(n / 64) e^x, n the nearest whole number to 64 times the exponent in base 2: 2^(n / 64) from a table of
// 2^0 .. 2^(63 / 64) and e^x by its Taylor series on |x| <= ln 2 / 128, whose remainder after degree 5 is below 2^-54. (By degree
// 12 on ln 2 / 2 without a table, 256 rows of 131,072 without top-k or top-p took 108 us, 100 with it.) scale = log2(e) / T.
__device__ __forceinline__ double* sm_powers()
{
    __shared__ double t[64];
    return t;
}
// fills the table; a barrier before its first use is the caller's
__device__ __forceinline__ void sm_powers_init()
{
    if (threadIdx.x >= 64) return;
    const double n = threadIdx.x > 32 ? 1.0 : 0.0, x = ((int)threadIdx.x / 64.0 - n) * 0.693147180559945309417;
    double p = 1.0;   // e^x by Horner's rule: remainder below 2^-51 for |x| <= ln 2 / 2
#pragma unroll
    for (int k = 13; k; --k) p = fma(p, x * (1.0 / k), 1.0);
    sm_powers()[threadIdx.x] = n > 0 ? 2.0 * p : p;
}
__device__ __forceinline__ double sm_exp(uint32_t key, uint32_t top, double scale)
{
    // without branches, so that a thread's values run side by side
    const double y0 = ((double)sm_value(key) - (double)sm_value(top)) * (64.0 * scale);
    const bool any = y0 > -64000.0;     // not so for a NaN: finite - inf over an infinite T, inf - inf
    const double y = any ? y0 : 0.0;
    const double n = rint(y), x = (y - n) * (0.693147180559945309417 / 64);
    const int i = (int)n;
    double p = 1.0 / 120;
    p = fma(p, x, 1.0 / 24);
    p = fma(p, x, 1.0 / 6);
    p = fma(p, x, 0.5);
    p = fma(p, x, 1.0);
    p = fma(p, x, 1.0) * sm_powers()[i & 63];
    const double e = __longlong_as_double(__double_as_longlong(p) + ((long long)(i >> 6) << 52));
    return key == top ? 1.0 : any ? e : 0.0;
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

// The weights of 4 keys, those whose exponential lies below `least` or that are masked 0. Every key's exponential is worked out,
// held by the empty asm, so that the four run side by side: behind a branch each (which the compiler makes of the selects) 256
// rows of 131,072 without top-k or top-p took 100 us, 95 now, 1024 rows 740 and 630.
__device__ __forceinline__ void sm_weights(const uint32_t (&key)[4], uint32_t top, double scale, double least,
                                           unsigned long long (&x)[4])
{
    double e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = sm_exp(key[j], top, scale);
    asm volatile("" : "+v"(e[0]), "+v"(e[1]), "+v"(e[2]), "+v"(e[3]));
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (key[j] > SM_MASKED) & (e[j] >= least) ? sm_units(e[j]) : 0;
}

// Wave scans by DPP: shifts by 1, 2, 4, 8 within rows of 16 lanes, then the rows' last lanes to the rows after them. `id` is
// what a lane without a source takes.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t sm_dpp(uint32_t id, uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp((int)id, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long sm_dpp64(unsigned long long v)
{
    return (unsigned long long)sm_dpp<CTRL, ROWS>(0, (uint32_t)(v >> 32)) << 32 | sm_dpp<CTRL, ROWS>(0, (uint32_t)v);
}
__device__ __forceinline__ unsigned long long sm_wave_scan(unsigned long long v)   // inclusive
{
    v += sm_dpp64<0x111, 0xF>(v);
    v += sm_dpp64<0x112, 0xF>(v);
    v += sm_dpp64<0x114, 0xF>(v);
    v += sm_dpp64<0x118, 0xF>(v);
    v += sm_dpp64<0x142, 0xA>(v);
    v += sm_dpp64<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ unsigned long long sm_lane64(unsigned long long v, int lane)
{
    return (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
template <typename V>
__device__ __forceinline__ V sm_wave_sum(V v)
{
    return (V)sm_lane64(sm_wave_scan(v), 63);
}
__device__ __forceinline__ uint32_t sm_wave_max(uint32_t v)
{
    v = max(v, sm_dpp<0x111, 0xF>(0, v));
    v = max(v, sm_dpp<0x112, 0xF>(0, v));
    v = max(v, sm_dpp<0x114, 0xF>(0, v));
    v = max(v, sm_dpp<0x118, 0xF>(0, v));
    v = max(v, sm_dpp<0x142, 0xA>(0, v));
    v = max(v, sm_dpp<0x143, 0xC>(0, v));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t sm_wave_min(uint32_t v) { return ~sm_wave_max(~v); }

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
    auto kept_by_min = [&](uint32_t key) { return !(mp > 0.0f) || sm_exp(key, top, scale) >= (double)mp; };

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
// work in one workgroup took 547 us). Four launches, for up to SM_ROWS rows at a time:
//   top     each slice's largest and smallest logit and the largest's index, and the largest of each of up to 1,024 groups
//           of the row; clears the row's histogram
//   bins    (not for a top-k of up to half the groups: the k-th largest group maximum, rounded down, has at least k logits at
//           or above it and few more, and is the list's floor) 2,047 bins of equal width from the largest logit down to where
//           weights round to zero (or to the smallest), and one for what lies below: logits per bin for a top-k, else the
//           weight per bin (of the row and of each slice)
//   cut     every workgroup finds the bins in which the kept prefix ends from the row's histogram. With a top-k (and few
//           logits down to its bin) all logits down to that bin go into the row's list; else the list takes the bins
//           where the nucleus and min-p end, and each slice sums the weight of its bins above them
//   pick    a workgroup per row finds the last kept logit in the list, and draws: from the list itself (top-k), or
//           from the slice in which the target lies
constexpr int SM_LIST = 4096;         // logits a row's list holds
constexpr int SM_LISTK = 1024;        // top-k up to which the list is expected to hold the whole kept set
constexpr int SM_PT = 256;            // threads of the slice launches
constexpr int SM_MAXS = 256;          // slices of a row
constexpr int SM_GROUPS = 1024;       // group maxima of a row, at most
constexpr int SM_ROWS = 1024;         // rows of one round of launches, which bounds the workspace
constexpr int SM_PER = SM_LIST / SM_T;   // list entries of a thread of the last launch

struct SmSlice
{
    uint32_t top, low;                // largest key, smallest key above -inf (0, ~0 without any)
    int32_t arg;                      // lowest index of the largest
    int32_t pad;
    unsigned long long mass;          // weight above the list's bins (every kept weight: SM_ALL)
};
enum
{
    SM_ALL = 0,                       // every logit kept (but for min-p): draw from the slices
    SM_BIN = 1,                       // the list holds the bins where the nucleus and min-p end
    SM_TOPK = 2,                      // the list holds everything that may be kept
    SM_SLOW = 3,
};
struct SmState                        // of a row
{
    int32_t count;                    // list entries (more than SM_LIST: it overflowed)
    int32_t mode;
    int32_t lo, hi;                   // the list's bins
    unsigned long long want, above;   // SM_BIN: weight at which the nucleus ends, weight above the list's bins
};
struct SmWs
{
    uint32_t* cnt;                    // [B][SM_BINS]
    unsigned long long* mass;         // [B][SM_BINS]
    unsigned long long* part;         // [B][S][SM_BINS] the slices' weights
    unsigned long long* list;         // [B][SM_LIST] key << 32 | ~index
    SmSlice* slice;                   // [B][S]
    SmState* state;                   // [B]
    uint32_t* group;                  // [B][SM_GROUPS] keys
    int S, len;                       // slices of a row, logits of a slice
    int G;                            // groups of a slice: 256 / G neighbouring threads' logits each
};

static void sm_split(int B, int V, int& S, int& len)
{
    const int want = (2048 + B - 1) / B;                     // eight workgroups a CU
    S = V / 2048 < 1 ? 1 : V / 2048;
    if (S > want) S = want;
    if (S > SM_MAXS) S = SM_MAXS;
    len = ((V + S - 1) / S + 3) / 4 * 4;
    S = (V + len - 1) / len;
}

static size_t sm_carve(void* base, int B, int V, SmWs& w)
{
    sm_split(B, V, w.S, w.len);
    size_t at = 0;
    auto take = [&](size_t n) {
        char* r = static_cast<char*>(base) + at;
        at += (n + 255) / 256 * 256;
        return r;
    };
    w.mass = reinterpret_cast<unsigned long long*>(take((size_t)B * SM_BINS * 8));
    w.part = reinterpret_cast<unsigned long long*>(take((size_t)B * w.S * SM_BINS * 8));
    w.list = reinterpret_cast<unsigned long long*>(take((size_t)B * SM_LIST * 8));
    w.slice = reinterpret_cast<SmSlice*>(take((size_t)B * w.S * sizeof(SmSlice)));
    w.state = reinterpret_cast<SmState*>(take((size_t)B * sizeof(SmState)));
    w.cnt = reinterpret_cast<uint32_t*>(take((size_t)B * SM_BINS * 4));
    w.group = reinterpret_cast<uint32_t*>(take((size_t)B * SM_GROUPS * 4));
    w.G = SM_PT;
    while (w.G * w.S > SM_GROUPS) w.G /= 2;
    return at;
}

// use(index, 4 keys) for this thread's logits of [lo, hi): 4 neighbours at a time (key 0: none), 4 loads in flight (`b`: the first 4, loaded
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
        const int next = i + 4 * NT * 4;
        SmBatch<E, NT> n;
        n.load(row, next, hi);   // under this batch's work
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            const int at = i + j * NT * 4;
            // what lies past the slice counts as masked
            uint32_t key[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                key[k] = at + 4 <= hi ? sm_key(static_cast<float>(b.v[j][k]))
                         : at + k < hi ? sm_key(static_cast<float>(row[at + k])) : 0;
            use(at, key);
        }
        i = next;
        b = n;
    }
}

// what every launch after the first knows of a row
struct SmHead
{
    uint32_t top, low;
    int arg;
    bool done;            // the largest logit, or nothing to draw from
    bool wide;            // a range past fp32: no bins
    float T, top_x, bins; // bins per unit of logit
    double scale;
    __device__ __forceinline__ float place(uint32_t key) const { return key == top ? 0.0f : (top_x - sm_value(key)) * bins; }
    __device__ __forceinline__ int bin(uint32_t key) const { return (int)fminf(place(key), (float)(SM_BINS - 1)); }
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
    h.top = sm_wave_max(top);
    h.low = sm_wave_min(low);
    h.arg = (int)sm_wave_min(top == h.top ? (uint32_t)arg : 0x7FFFFFFFu);
    h.T = a.temperature ? a.temperature[b] : 1.0f;
    // a min-p past 1 keeps the largest logit alone
    h.done = h.top <= SM_MASKED || !(h.T > 0.0f) || (a.min_p && a.min_p[b] > 1.0f);
    h.top_x = sm_value(h.top);
    h.scale = 1.4426950408889634074 / (double)h.T;
    // down to the smallest logit (a little past it, so that it lies in a bin of its own right) or to where weights round to
    // zero units: what falls into the last bin, below the range, weighs nothing
    const float range = fmaxf(fminf((h.top_x - sm_value(h.low)) * 1.001f, 31.0f * h.T), 1e-30f);
    h.bins = (float)(SM_BINS - 1) / range;
    h.wide = !(range < __builtin_inff());
    return h;
}

template <typename E>
__global__ __launch_bounds__(SM_PT) void sm_top_kernel(SampleArgs a, SmWs w)
{
    const int b = blockIdx.y, s = blockIdx.x, lo = s * w.len, hi = min(a.V, lo + w.len);
    const E* row = static_cast<const E*>(a.logits) + (int64_t)b * a.ld;
    SmBatch<E, SM_PT> first;
    first.load(row, lo + threadIdx.x * 4, hi);
    for (int i = s * SM_PT + threadIdx.x; i < SM_BINS; i += w.S * SM_PT)
    {
        w.cnt[(size_t)b * SM_BINS + i] = 0;
        w.mass[(size_t)b * SM_BINS + i] = 0;
    }
    if (s == 0 && threadIdx.x == 0) w.state[b].count = 0;
    uint32_t top = 0, low = ~0u;
    int arg = 0x7FFFFFFF;
    sm_each<E, SM_PT>(row, lo, hi, first, [&](int i, const uint32_t (&key)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            if (key[j] > top) top = key[j], arg = i + j;
            if (key[j] > SM_MASKED) low = min(low, key[j]);
        }
    });
    uint32_t group = top;
    const int lanes = SM_PT / w.G;   // 1 to 64
    for (int o = 1; o < lanes; o <<= 1) group = max(group, (uint32_t)__shfl_xor((int)group, o));
    if (threadIdx.x % lanes == 0) w.group[(size_t)b * SM_GROUPS + s * w.G + threadIdx.x / lanes] = group;
    __shared__ uint32_t st[SM_PT / 64], sl[SM_PT / 64];
    __shared__ int sa[SM_PT / 64];
    const uint32_t wt = sm_wave_max(top), wl = sm_wave_min(low);
    const int wa = (int)sm_wave_min(top == wt ? (uint32_t)arg : 0x7FFFFFFFu);
    if (threadIdx.x % 64 == 0) st[threadIdx.x / 64] = wt, sl[threadIdx.x / 64] = wl, sa[threadIdx.x / 64] = wa;
    __syncthreads();
    if (threadIdx.x == 0)
    {
        SmSlice& c = w.slice[(size_t)b * w.S + s];
        c.top = st[0];
        c.low = sl[0];
        c.arg = sa[0];
        c.mass = 0;
        for (int i = 1; i < SM_PT / 64; ++i)
        {
            if (st[i] > c.top || (st[i] == c.top && sa[i] < c.arg)) c.top = st[i], c.arg = sa[i];
            c.low = min(c.low, sl[i]);
        }
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
__device__ __forceinline__ double sm_minp(const SampleArgs& a, int b)
{
    const float m = a.min_p ? a.min_p[b] : 0.0f;
    return m > 0.0f ? (double)m : 0.0;
}

// The list's floor for a top-k from the group maxima: a key that at least k logits reach, the k-th largest maximum with all but
// its leading 14 bits past those common to all cleared. False where the groups do not tell. One wave's work (sm_floor asks the
// first one).
__device__ __forceinline__ bool sm_floor_wave(const SmWs& w, int b, int k, uint32_t top, uint32_t& floor)
{
    const int ng = w.S * w.G, lane = threadIdx.x % 64;
    if (!k || 2 * k > ng) return false;
    uint32_t v[SM_GROUPS / 64], low = ~0u;
    int valid = 0;
#pragma unroll
    for (int i = 0; i < SM_GROUPS / 64; ++i)
        v[i] = i * 64 + lane < ng ? w.group[(size_t)b * SM_GROUPS + i * 64 + lane] : 0;
#pragma unroll
    for (int i = 0; i < SM_GROUPS / 64; ++i)
    {
        const bool in = v[i] > SM_MASKED;
        valid += __popcll(__ballot(in));
        if (in) low = min(low, v[i]);
    }
    if (valid < k) return false;
    low = sm_wave_min(low);
    floor = top;
    if (low == top) return true;
    const int first = 31 - __clz((int)(top ^ low));
    floor = top >> first >> 1 << first << 1;
    for (int bit = first; bit >= 0 && bit > first - 14; --bit)
    {
        const uint32_t c = floor | 1u << bit;
        int n = 0;
#pragma unroll
        for (int i = 0; i < SM_GROUPS / 64; ++i) n += __popcll(__ballot(v[i] >= c));
        if (n >= k) floor = c;
    }
    return true;
}
__device__ __forceinline__ bool sm_floor(const SmWs& w, int b, int k, uint32_t top, uint32_t& floor, int* shared)
{
    if (!k || 2 * k > w.S * w.G) return false;
    if (threadIdx.x < 64)
    {
        uint32_t f = 0;
        const bool ok = sm_floor_wave(w, b, k, top, f);
        if (threadIdx.x == 0) shared[0] = ok, shared[1] = (int)f;
    }
    __syncthreads();
    const bool ok = shared[0];
    floor = (uint32_t)shared[1];
    __syncthreads();
    return ok;
}

// rows whose list a top-k fills take logits per bin; the others with a nucleus their weight
__device__ __forceinline__ bool sm_weighs(int k, float p) { return p < 1.0f && (!k || k > SM_LISTK); }

template <typename E>
__global__ __launch_bounds__(SM_PT) void sm_bins_kernel(SampleArgs a, SmWs w)
{
    __shared__ uint32_t cnt[SM_BINS];
    __shared__ unsigned long long mass[SM_BINS];
    const int b = blockIdx.y, s = blockIdx.x, lo = s * w.len, hi = min(a.V, lo + w.len);
    const E* row = static_cast<const E*>(a.logits) + (int64_t)b * a.ld;
    SmBatch<E, SM_PT> first;
    first.load(row, lo + threadIdx.x * 4, hi);
    sm_powers_init();   // under the loads
    const SmHead h = sm_head(a, w, b);
    const int k = sm_topk(a, b);
    const float p = sm_topp(a, b);
    if (h.done || h.wide || (!k && !(p < 1.0f))) return;
    uint32_t floor;
    __shared__ int shared[2];
    if (sm_floor(w, b, k, h.top, floor, shared)) return;
    const bool weigh = sm_weighs(k, p);
    for (int i = threadIdx.x; i < SM_BINS; i += SM_PT) cnt[i] = 0, mass[i] = 0;
    __syncthreads();
    if (weigh)
        sm_each<E, SM_PT>(row, lo, hi, first, [&](int, const uint32_t (&key)[4]) {
            unsigned long long x[4];
            sm_weights(key, h.top, h.scale, 0.0, x);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (key[j] > SM_MASKED)
                {
                    const int bin = h.bin(key[j]);
                    if (k) atomicAdd(&cnt[bin], 1u);
                    if (bin < SM_BINS - 1) atomicAdd(&mass[bin], x[j]);
                }
        });
    else
        sm_each<E, SM_PT>(row, lo, hi, first, [&](int, const uint32_t (&key)[4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (key[j] > SM_MASKED) atomicAdd(&cnt[h.bin(key[j])], 1u);
        });
    __syncthreads();
    unsigned long long* part = w.part + ((size_t)b * w.S + s) * SM_BINS;
    for (int i = threadIdx.x; i < SM_BINS; i += SM_PT)
    {
        if (cnt[i]) atomicAdd(&w.cnt[(size_t)b * SM_BINS + i], cnt[i]);
        if (weigh)
        {
            part[i] = mass[i];
            if (mass[i]) atomicAdd(&w.mass[(size_t)b * SM_BINS + i], mass[i]);
        }
    }
}

// exclusive sum over the workgroup's threads in order; `total` gets the sum of all. NT / 64 slots of scratch.
template <int NT>
__device__ __forceinline__ unsigned long long sm_scan(unsigned long long v, unsigned long long* scratch,
                                                      unsigned long long& total)
{
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const unsigned long long c = sm_wave_scan(v);
    __syncthreads();
    if (lane == 63) scratch[wave] = c;
    __syncthreads();
    // every wave scans the waves' sums in its first lanes
    const unsigned long long all = sm_wave_scan(lane < NT / 64 ? scratch[lane] : 0);
    total = sm_lane64(all, NT / 64 - 1);
    return (wave ? sm_lane64(all, __builtin_amdgcn_readfirstlane(wave) - 1) : 0) + c - v;
}

// the bins in which the kept prefix of a row ends, and the row's mode
struct SmCut
{
    int mode, lo, hi;
    unsigned long long want, above;
    uint32_t floor;      // smallest key of the list (where it is not given by the bins: 0)
};
__device__ SmCut sm_cut(const SampleArgs& a, const SmWs& w, int b, const SmHead& h, unsigned long long* scratch, int* found)
{
    constexpr int PER = SM_BINS / SM_PT;
    const int k = sm_topk(a, b);
    const float p = sm_topp(a, b);
    SmCut c = { SM_ALL, 0, SM_BINS - 1, 0, 0, 0 };
    if (!k && !(p < 1.0f)) return c;
    if (sm_floor(w, b, k, h.top, c.floor, found))
    {
        c.mode = SM_TOPK;
        c.hi = h.bin(c.floor);
        return c;
    }
    c.floor = 0;
    if (h.wide)
    {
        c.mode = SM_SLOW;
        return c;
    }
    const uint32_t* cnt = w.cnt + (size_t)b * SM_BINS + threadIdx.x * PER;
    const unsigned long long* mass = w.mass + (size_t)b * SM_BINS + threadIdx.x * PER;
    unsigned long long total = 0;
    if (threadIdx.x == 0) found[0] = -1, found[1] = 0;
    if (k)
    {
        uint32_t each[PER];
        unsigned long long n = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) n += each[i] = cnt[i];
        unsigned long long at = sm_scan<SM_PT>(n, scratch, total);
        if (k <= SM_LISTK || total > (unsigned long long)k)
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
            __syncthreads();
            c.hi = found[0];
            c.mode = found[1] > SM_LIST ? SM_SLOW : SM_TOPK;
            return c;
        }
        if (!(p < 1.0f)) return c;   // a top-k that keeps every logit
        __syncthreads();
    }
    unsigned long long each[PER], m = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) m += each[i] = mass[i];
    const unsigned long long before = sm_scan<SM_PT>(m, scratch, total);
    unsigned long long at = before;
    const double goal = (double)p * (double)total;
    c.want = goal > 1.0 ? (unsigned long long)ceil(goal) : 1ull;
#pragma unroll
    for (int i = 0; i < PER; ++i)
    {
        if (at < c.want && at + each[i] >= c.want) found[0] = threadIdx.x * PER + i;
        at += each[i];
    }
    __syncthreads();
    c.mode = SM_BIN;
    c.lo = c.hi = found[0];
    const double mp = sm_minp(a, b);
    if (mp > 0.0)
    {
        // min-p ends where exp(-d / T) = m: the bins beside that place, too, where they are not past the nucleus. The place
        // in d / T is known to fp64's roundings of 1 (2^-48 holds those of the exponential and of the logarithm): at an infinite T, or
        // one of 2^48 bins, all weights reach m = 1, not the bin at d = 0 alone.
        const double end = -log(mp), low = end - 0x1p-48, high = end + 0x1p-48;
        auto bin = [&](double x) { return (int)fminf((float)(x * (double)h.T) * h.bins, (float)(SM_BINS - 1)); };
        c.lo = min(c.lo, max((low > 0.0 ? bin(low) : 0) - 1, 0));
        c.hi = min(c.hi, bin(high) + 1);
    }
    // weight above the list's bins
    at = before;
#pragma unroll
    for (int i = 0; i < PER; ++i)
    {
        if (threadIdx.x * PER + i == c.lo) scratch[SM_PT / 64] = at;
        at += each[i];
    }
    __syncthreads();
    c.above = scratch[SM_PT / 64];
    return c;
}

template <typename E>
__global__ __launch_bounds__(SM_PT) void sm_cut_kernel(SampleArgs a, SmWs w)
{
    __shared__ unsigned long long scratch[SM_PT / 64 + 1];
    __shared__ int found[2];
    const int b = blockIdx.y, s = blockIdx.x, lo = s * w.len, hi = min(a.V, lo + w.len);
    const E* row = static_cast<const E*>(a.logits) + (int64_t)b * a.ld;
    // short slices are loaded ahead; of long ones many rows read only some groups
    const bool ahead = w.len <= SM_PT * 16;
    SmBatch<E, SM_PT> first;
    if (ahead) first.load(row, lo + threadIdx.x * 4, hi);
    sm_powers_init();   // under the loads
    const SmHead h = sm_head(a, w, b);
    if (h.done) return;
    const SmCut c = sm_cut(a, w, b, h, scratch, found);
    if (s == 0 && threadIdx.x == 0)
    {
        SmState& st = w.state[b];
        st.mode = c.mode;
        st.lo = c.lo;
        st.hi = c.hi;
        st.want = c.want;
        st.above = c.above;
    }
    if (c.mode == SM_SLOW) return;
    if (!ahead && !(c.floor && w.group[(size_t)b * SM_GROUPS + s * w.G + threadIdx.x / (SM_PT / w.G)] < c.floor))
        first.load(row, lo + threadIdx.x * 4, hi);
    unsigned long long mine = 0, total;
    if (c.mode == SM_ALL)
    {
        const double m = sm_minp(a, b);
        __syncthreads();   // the table of powers
        sm_each<E, SM_PT>(row, lo, hi, first, [&](int, const uint32_t (&key)[4]) {
            unsigned long long x[4];
            sm_weights(key, h.top, h.scale, m, x);
            mine += x[0] + x[1] + (x[2] + x[3]);
        });
    }
    else
    {
        unsigned long long* list = w.list + (size_t)b * SM_LIST;
        auto put = [&](int i, uint32_t key) {
            const int at = atomicAdd(&w.state[b].count, 1);
            if (at < SM_LIST) list[at] = (unsigned long long)key << 32 | (uint32_t)~i;
        };
        if (c.floor)
        {
            // only the groups that reach the floor are read
            if (w.group[(size_t)b * SM_GROUPS + s * w.G + threadIdx.x / (SM_PT / w.G)] >= c.floor)
                sm_each<E, SM_PT>(row, lo, hi, first, [&](int i, const uint32_t (&key)[4]) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (key[j] >= c.floor && key[j] > SM_MASKED) put(i + j, key[j]);
                });
        }
        else
            sm_each<E, SM_PT>(row, lo, hi, first, [&](int i, const uint32_t (&key)[4]) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    const int bin = h.bin(key[j]);
                    if (key[j] > SM_MASKED && bin >= c.lo && bin <= c.hi) put(i + j, key[j]);
                }
            });
        if (c.mode == SM_TOPK) return;
        const unsigned long long* part = w.part + ((size_t)b * w.S + s) * SM_BINS;
        for (int i = threadIdx.x; i < c.lo; i += SM_PT) mine += part[i];
    }
    sm_scan<SM_PT>(mine, scratch, total);
    if (threadIdx.x == 0) w.slice[(size_t)b * w.S + s].mass = total;
}

struct SmPick
{
    unsigned long long hist[SM_T], comp[SM_T], wt[SM_T];
    unsigned long long scratch[SM_W];
    unsigned long long part[SM_MAXS];
    unsigned long long at, cut, cut_wt;
    int bin, m, pick;
};

// Of the list's entries (SM_PER a thread; wt 0: not one) the one at which the weights summed in order reach `want`, the sum
// starting at `before`: order is by place (0 .. SM_T - 1) and within a place by comp, largest first. s.cut = its comp and
// s.cut_wt = its weight. Returns 0 = found, 1 = the sum stays below, 2 = too many entries share the place.
__device__ int sm_cross(SmPick& s, const int (&place)[SM_PER], const unsigned long long (&comp)[SM_PER],
                        const unsigned long long (&wt)[SM_PER], unsigned long long before, unsigned long long want)
{
    __syncthreads();
    s.hist[threadIdx.x] = 0;
    if (threadIdx.x == 0) s.bin = -1, s.m = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SM_PER; ++j)
        if (wt[j]) atomicAdd(&s.hist[place[j]], wt[j]);
    __syncthreads();
    const unsigned long long mine = s.hist[threadIdx.x];
    unsigned long long total;
    const unsigned long long at = before + sm_scan<SM_T>(mine, s.scratch, total);
    if (at < want && at + mine >= want) s.bin = (int)threadIdx.x, s.at = at;
    __syncthreads();
    const int bin = s.bin;
    if (bin < 0) return 1;
#pragma unroll
    for (int j = 0; j < SM_PER; ++j)
        if (wt[j] && place[j] == bin)
        {
            const int i = atomicAdd(&s.m, 1);
            if (i < SM_T) s.comp[i] = comp[j], s.wt[i] = wt[j];
        }
    __syncthreads();
    const int m = s.m;
    if (m > SM_T) return 2;
    if ((int)threadIdx.x < m)
    {
        const unsigned long long c = s.comp[threadIdx.x], x = s.wt[threadIdx.x];
        unsigned long long sum = s.at;
        for (int i = 0; i < m; ++i)
            if (s.comp[i] > c) sum += s.wt[i];
        if (sum < want && sum + x >= want) s.cut = c, s.cut_wt = x;
    }
    __syncthreads();
    return 0;
}

// the sum at which the draw stops: the smallest whole number past u * total
__device__ __forceinline__ unsigned long long sm_target(float u, unsigned long long total)
{
    const double t = fmax((double)u * (double)total, 0.0);   // a NaN too becomes 0
    return t < (double)total ? min((unsigned long long)t + 1, total) : total;
}

template <typename E>
__global__ __launch_bounds__(SM_T) void sm_pick_kernel(SampleArgs a, SmWs w)
{
    __shared__ union
    {
        SmShared slow;
        SmPick f;
    } sh;
    const int b = blockIdx.x, V = a.V;
    SmPick& f = sh.f;
    // loaded ahead of the head: this thread's list entries (those past its end are not used) and a slice's weight
    const unsigned long long* list = w.list + (size_t)b * SM_LIST;
    unsigned long long comp[SM_PER], slice_mass = 0;
#pragma unroll
    for (int j = 0; j < SM_PER; ++j) comp[j] = list[threadIdx.x + j * SM_T];
    if ((int)threadIdx.x < w.S) slice_mass = w.slice[(size_t)b * w.S + threadIdx.x].mass;
    sm_powers_init();   // under the loads
    const SmState st = w.state[b];
    const SmHead h = sm_head(a, w, b);
    auto answer = [&](int token, unsigned long long x, unsigned long long total) {
        a.token[b] = token;
        if (a.prob) a.prob[b] = (float)((double)x / (double)total);
    };
    if (h.done)
    {
        if (threadIdx.x == 0)
        {
            const bool none = h.top <= SM_MASKED;
            answer(none ? -1 : h.arg, none ? 0 : 1, 1);
        }
        return;
    }
    const E* row = static_cast<const E*>(a.logits) + (int64_t)b * a.ld;
    auto slow = [&]() {
        SmRow r;
        r.dtype = a.dtype;
        r.p = row;
        __syncthreads();
        sm_row_slow(sh.slow, a, b, r, h.top, h.scale);
    };
    __syncthreads();   // the table of powers
    if (st.mode == SM_SLOW || (st.mode != SM_ALL && st.count > SM_LIST)) return slow();
    const double mp = sm_minp(a, b);
    const int n = st.mode == SM_ALL ? 0 : st.count;
    unsigned long long wt[SM_PER], total = 0, cut = 0;
    int place[SM_PER];
    const float per_bin = (float)SM_T / (float)(st.hi - st.lo + 1);
#pragma unroll
    for (int j = 0; j < SM_PER; ++j)
    {
        const bool in = (int)threadIdx.x + j * SM_T < n;
        const uint32_t key = (uint32_t)(comp[j] >> 32);
        wt[j] = 0;
        place[j] = 0;
        if (in)
        {
            const double e = sm_exp(key, h.top, h.scale);
            wt[j] = sm_units(e);
            place[j] = (int)fminf(fmaxf((fminf(h.place(key), (float)SM_BINS) - (float)st.lo) * per_bin, 0.0f), (float)(SM_T - 1));
        }
    }
    auto kept_by_min = [&](uint32_t key) { return mp == 0.0 || sm_exp(key, h.top, h.scale) >= mp; };

    if (st.mode == SM_TOPK)
    {
        const int k = sm_topk(a, b);
        const float p = sm_topp(a, b);
        if (n > k)
        {
            unsigned long long one[SM_PER];
#pragma unroll
            for (int j = 0; j < SM_PER; ++j) one[j] = (int)threadIdx.x + j * SM_T < n;
            if (sm_cross(f, place, comp, one, 0, (unsigned long long)k)) return slow();
            cut = f.cut;
#pragma unroll
            for (int j = 0; j < SM_PER; ++j)
                if (comp[j] < cut) wt[j] = 0;
        }
        unsigned long long mine = 0;
        if (p < 1.0f)
        {
#pragma unroll
            for (int j = 0; j < SM_PER; ++j) mine += wt[j];
            sm_scan<SM_T>(mine, f.scratch, total);
            const double goal = (double)p * (double)total;
            if (sm_cross(f, place, comp, wt, 0, goal > 1.0 ? (unsigned long long)ceil(goal) : 1ull)) return slow();
            cut = f.cut;
#pragma unroll
            for (int j = 0; j < SM_PER; ++j)
                if (comp[j] < cut) wt[j] = 0;
        }
        mine = 0;
        unsigned long long by_index[SM_PER];
        const float per_index = (float)SM_T / (float)V;
#pragma unroll
        for (int j = 0; j < SM_PER; ++j)
        {
            if (wt[j] && !kept_by_min((uint32_t)(comp[j] >> 32))) wt[j] = 0;
            mine += wt[j];
            by_index[j] = (uint32_t)comp[j];   // ~index: the lowest index is the largest
            place[j] = min((int)((float)~(uint32_t)comp[j] * per_index), SM_T - 1);
        }
        sm_scan<SM_T>(mine, f.scratch, total);
        if (sm_cross(f, place, by_index, wt, 0, sm_target(a.u[b], total))) return slow();
        if (threadIdx.x == 0) answer((int)~(uint32_t)f.cut, f.cut_wt, total);
        return;
    }
    // from the slices: their weight above the list's bins and that of the list's kept entries
    if (st.mode == SM_BIN)
    {
        const int r = sm_cross(f, place, comp, wt, st.above, st.want);
        if (r == 2) return slow();
        cut = r ? 0 : f.cut;   // not reached: min-p ends first
    }
    __syncthreads();
    if ((int)threadIdx.x < w.S) f.part[threadIdx.x] = slice_mass;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SM_PER; ++j)
        if (wt[j] && comp[j] >= cut && kept_by_min((uint32_t)(comp[j] >> 32)))
            atomicAdd(&f.part[~(uint32_t)comp[j] / (uint32_t)w.len], wt[j]);
    __syncthreads();
    const unsigned long long mine = (int)threadIdx.x < w.S ? f.part[threadIdx.x] : 0;
    unsigned long long at = sm_scan<SM_T>(mine, f.scratch, total);
    const unsigned long long target = sm_target(a.u[b], total);
    if (at < target && at + mine >= target) f.pick = (int)threadIdx.x, f.at = at;
    __syncthreads();
    const int s = f.pick, lo = s * w.len, hi = min(V, lo + w.len), per = (hi - lo + SM_T - 1) / SM_T;
    const int i0 = lo + (int)threadIdx.x * per, i1 = min(hi, i0 + per);
    const unsigned long long base = f.at;
    auto weight = [&](int i) -> unsigned long long {
        const uint32_t key = sm_key(static_cast<float>(row[i]));
        if (key <= SM_MASKED || ((unsigned long long)key << 32 | (uint32_t)~i) < cut) return 0;
        const double x = sm_exp(key, h.top, h.scale);
        return x >= mp ? sm_units(x) : 0;
    };
    unsigned long long sum = 0, all;
    for (int i = i0; i < i1; i += 4)   // 4 at a time, their exponentials side by side
    {
        uint32_t key[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) key[j] = i + j < i1 ? sm_key(static_cast<float>(row[i + j])) : 0;
        unsigned long long x[4];
        sm_weights(key, h.top, h.scale, mp, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += ((unsigned long long)key[j] << 32 | (uint32_t)~(i + j)) < cut ? 0 : x[j];
    }
    unsigned long long c = base + sm_scan<SM_T>(sum, f.scratch, all);
    if (c < target && c + sum >= target)
        for (int i = i0; i < i1; ++i)
        {
            const unsigned long long x = weight(i);
            if (c < target && c + x >= target) answer(i, x, total);
            c += x;
        }
}

size_t sample_ws_bytes(int B, int V)
{
    SmWs w;
    return B ? sm_carve(nullptr, B < SM_ROWS ? B : SM_ROWS, V, w) : 0;
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

void launch_sample(const SampleArgs& all, hipStream_t st)
{
    SmWs w;
    sm_carve(all.ws, all.B < SM_ROWS ? all.B : SM_ROWS, all.V, w);
    for (int b = 0; b < all.B; b += SM_ROWS)
    {
        SampleArgs a = all;
        a.B = all.B - b < SM_ROWS ? all.B - b : SM_ROWS;
        a.logits = static_cast<const char*>(all.logits) + (int64_t)b * all.ld * (all.dtype == 2 ? 4 : 2);
        if (a.temperature) a.temperature += b;
        if (a.top_k) a.top_k += b;
        if (a.top_p) a.top_p += b;
        if (a.min_p) a.min_p += b;
        a.u += b;
        a.token += b;
        if (a.prob) a.prob += b;
        if (a.dtype == 2) sm_go<float>(a, w, st);
        else if (a.dtype == 1) sm_go<__bf16>(a, w, st);
        else sm_go<_Float16>(a, w, st);
    }
}

}  // namespace gfl
