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

// weight of a key in units of 2^-43 of the largest logit's
__device__ __forceinline__ uint64_t sm_weight(uint32_t key, uint32_t top, double inv_t)
{
    if (key == top) return 1ull << 43;
    if (key <= SM_MASKED) return 0;
    const double d = ((double)sm_value(key) - (double)sm_value(top)) * inv_t;
    return d > -31.0 ? (uint64_t)(exp(d) * 0x1p43 + 0.5) : 0;   // also when the largest is +inf
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
__device__ uint32_t sm_select(SmShared& s, const SmRow& row, int V, uint32_t top, double inv_t, int mode,
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
                const uint64_t w = sm_weight(k, top, inv_t);
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

__global__ __launch_bounds__(SM_T) void sample_kernel(SampleArgs a)
{
    __shared__ SmShared s;
    __shared__ int result;
    const int b = blockIdx.x, V = a.V, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    SmRow row;
    row.dtype = a.dtype;
    row.p = static_cast<const char*>(a.logits) + (int64_t)b * a.ld * (a.dtype == 2 ? 4 : 2);
    const float T = a.temperature ? a.temperature[b] : 1.0f;
    const bool greedy = !(T > 0.0f);

    // the largest key and its lowest index
    uint32_t top = 0;
    int first = V;
    for (int i = threadIdx.x; i < V; i += SM_T)
    {
        const uint32_t k = row.key(i);
        if (k > top) top = k, first = i;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1)
    {
        const uint32_t k = (uint32_t)__shfl_xor((int)top, o);
        const int f = __shfl_xor(first, o);
        if (k > top || (k == top && f < first)) top = k, first = f;
    }
    if (lane == 0) s.wcnt[wave] = top, s.cnt[wave] = (uint32_t)first;
    __syncthreads();
    top = s.wcnt[0];
    first = (int)s.cnt[0];
    for (int w = 1; w < SM_W; ++w)
        if (s.wcnt[w] > top || (s.wcnt[w] == top && (int)s.cnt[w] < first)) top = s.wcnt[w], first = (int)s.cnt[w];
    __syncthreads();
    if (top <= SM_MASKED || greedy)
    {
        if (threadIdx.x == 0)
        {
            a.token[b] = top <= SM_MASKED ? -1 : first;
            if (a.prob) a.prob[b] = top <= SM_MASKED ? 0.0f : 1.0f;
        }
        return;
    }
    const double inv_t = 1.0 / (double)T;

    // the kept prefix: keys above `cut`, and the first `ties` of those equal to it
    uint32_t cut = 0;
    unsigned long long ties = ~0ull;
    unsigned long long total = 0;   // weight of the top-k
    const int k = a.top_k ? a.top_k[b] : 0;
    if (k > 0 && k < V)
    {
        cut = sm_select(s, row, V, top, inv_t, 0, (unsigned long long)k);
        ties = (unsigned long long)k - s.above;
        total = s.above_mass + ties * sm_weight(cut, top, inv_t);
        __syncthreads();
    }
    const float p = a.top_p ? a.top_p[b] : 1.0f;
    if (p < 1.0f)
    {
        if (cut == 0)
        {
            unsigned long long m = 0;
            for (int i = threadIdx.x; i < V; i += SM_T) m += sm_weight(row.key(i), top, inv_t);
            m = sm_wave_sum(m);
            if (lane == 0) s.wmass[wave] = m;
            __syncthreads();
            for (int w = 0; w < SM_W; ++w) total += s.wmass[w];
            __syncthreads();
        }
        const double goal = (double)p * (double)total;
        const unsigned long long want = goal > 1.0 ? (unsigned long long)ceil(goal) : 1ull;
        const uint32_t pc = sm_select(s, row, V, top, inv_t, 1, want);
        const unsigned long long w = sm_weight(pc, top, inv_t);
        unsigned long long t = w ? (want - s.above + w - 1) / w : 1;
        if (pc > cut || (pc == cut && t < ties)) cut = pc, ties = t;
        __syncthreads();
    }
    const float mp = a.min_p ? a.min_p[b] : 0.0f;
    // by fp64, as the filter's definition has it; the largest stays
    auto kept_by_min = [&](uint32_t key) {
        if (!(mp > 0.0f) || key == top) return true;
        if (key <= SM_MASKED || top == 0xFF800000u) return false;
        return exp(((double)sm_value(key) - (double)sm_value(top)) * inv_t) >= (double)mp;
    };

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
            if (use(i, keep ? (unsigned long long)sm_weight(key, top, inv_t) : 0ull)) break;
        }
    };
    unsigned long long mine = 0;
    walk([&](int, unsigned long long w) {
        mine += w;
        return false;
    });
    mine = sm_wave_sum(mine);
    if (lane == 0) s.wmass[wave] = mine;
    if (threadIdx.x == 0) result = -1;
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

size_t sample_ws_bytes(int, int) { return 0; }

void launch_sample(const SampleArgs& a, hipStream_t st)
{
    hipLaunchKernelGGL(sample_kernel, dim3(a.B), dim3(SM_T), 0, st, a);
}

}  // namespace gfl
