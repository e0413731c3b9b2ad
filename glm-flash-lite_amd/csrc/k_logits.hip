// Logits as a request's settings change them before a token is drawn: penalties for tokens that were there before, biases, a mask.
//
// A workgroup takes a slice of a row. What the row's history says of each of the slice's tokens is gathered in LDS by integer
// atomics (the same in any order), then the slice is read, changed and written once.
//
// Large batches are bound by the logits' way through memory and by what cannot overlap it, a slice's search of its row's history: 256
// rows of 131,072 with 30,000 tokens each 84 us (in place without a mask 78), 52 without lists (a copy 50), 57 without histories (bytes
// 60 us). Small ones by latency: a row of 131,072 5.0 us, 24 of 100,003 10.7 (5 without lists: a launch, two trips to memory).
#include "gfl_internal.hpp"
#include "gfl_open.hpp"

#include <algorithm>

namespace gfl {

constexpr int LG_T = 512, LG_UNIT = 4 * LG_T;   // a slice is whole units: 4 neighbouring tokens a thread
constexpr int LG_BIAS = (MAX_BIASES + LG_T - 1) / LG_T;   // biases a thread takes

// v0 .. v0 + n - 1 of a row's elements as fp32, n <= 4; rows start anywhere
template <typename E>
__device__ __forceinline__ void lg_load(const E* p, int n, float (&v)[4])
{
    E e[4] = {};
    if (n >= 4) __builtin_memcpy(e, p, sizeof e);
    else
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < n) e[i] = p[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(e[i]);
}
template <typename E>
__device__ __forceinline__ void lg_store(E* p, int n, const float (&v)[4])
{
    E e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = static_cast<E>(v[i]);
    if (n >= 4) __builtin_memcpy(p, e, sizeof e);
    else
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < n) p[i] = e[i];
}

// What the history says of a token: whether it is in the prompt, and how often it comes after. Histories of up to 32,767 tokens take
// 16 bits a token, so that a slice of 32,768 fits twice into a CU's LDS: every slice reads the whole history.
template <bool HALF>
struct LgWord
{
    static constexpr uint32_t SEEN = HALF ? 0x8000u : 0x80000000u;
    static constexpr int PER = HALF ? 2 : 1;   // tokens of a 32-bit word
    static __device__ __forceinline__ void seen(uint32_t* w, uint32_t v)
    {
        if constexpr (HALF) atomicOr(&w[v / 2], SEEN << (v % 2 * 16));
        else atomicOr(&w[v], SEEN);
    }
    static __device__ __forceinline__ void count(uint32_t* w, uint32_t v)
    {
        if constexpr (HALF) atomicAdd(&w[v / 2], 1u << (v % 2 * 16));
        else atomicAdd(&w[v], 1u);
    }
    static __device__ __forceinline__ bool four(const uint32_t* w, int i, uint32_t (&out)[4])   // of 4 tokens from i on; any?
    {
        if constexpr (HALF)
        {
            const uint2 p = *reinterpret_cast<const uint2*>(w + i / 2);
            out[0] = p.x & 0xFFFF, out[1] = p.x >> 16, out[2] = p.y & 0xFFFF, out[3] = p.y >> 16;
            return (p.x | p.y) != 0;
        }
        else
        {
            const uint4 p = *reinterpret_cast<const uint4*>(w + i);
            out[0] = p.x, out[1] = p.y, out[2] = p.z, out[3] = p.w;
            return (p.x | p.y | p.z | p.w) != 0;
        }
    }
};

template <typename E, bool HALF>
__global__ __launch_bounds__(LG_T, 4) void logits_kernel(LogitsArgs a)
{
    typedef LgWord<HALF> W;
    extern __shared__ __align__(16) uint32_t word[];   // the slice's words; with biases, see below
    const int tid = threadIdx.x, slice = a.slice;
    uint32_t* marked = word + (a.L ? slice / W::PER : 0);
    uint32_t* before = marked + slice / 32;
    uint32_t* total = before + slice / 32;
    uint32_t* last = total + LG_T / 64;
    float* bval = reinterpret_cast<float*>(last + a.n_bias);
    uint32_t* open = a.n_bias ? reinterpret_cast<uint32_t*>(bval + a.n_bias) : marked;   // the slice's words of the mask

    int64_t b = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
    if (a.by_xcd)
    {
        const int64_t k = blockIdx.x / 8;
        b = k / a.slices * 8 + blockIdx.x % 8, s = k % a.slices;
        if (b >= a.B) return;
    }
    s = (s + b) % a.slices;
    const int v0 = (int)s * slice, nv = min(slice, a.V - v0);
    const E* x = static_cast<const E*>(a.logits) + b * a.ld + v0;
    E* out = static_cast<E*>(a.out) + b * a.ldo + v0;
    const int32_t* allowed = a.allowed ? a.allowed + b * a.lda : nullptr;
    // The mask goes to LDS with the first loads. Read a word a thread beside the logits, it costs 256 rows of 131,072 98 us instead of 87.
    const bool lazy = a.lazy;   // only what the lists name is read and written

    constexpr int U = 4, NB = 2;   // loads of 4 ids, of 4 logits under way
    const int32_t* h = a.L ? a.history + b * a.ldh : nullptr;
    int32_t id[U][4];
    auto ids_at = [&](int at) {
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(id[u], h + min(at + u * LG_UNIT, a.L - 4), 16);
    };
    uint32_t m[2] = {};   // (a slice has at most 1024)
    if (allowed)
#pragma unroll
        for (int k = 0; k < 2; ++k) m[k] = (uint32_t)allowed[v0 / 32 + min(tid + k * LG_T, (nv - 1) / 32)];
    if (a.L >= 4) ids_at(tid * 4);   // as many as the row has room for; which of them count is seen later
    // Four logits from i on, or where fewer are left the slice's last four, without a branch around the load, which would wait for the
    // loads before it (256 rows of 131,072 87 us instead of 80); the thread at the end loads its own one by one when it comes to them.
    E y[NB][4] = {};
    auto read = [&](int at) {
#pragma unroll
        for (int j = 0; j < NB; ++j) __builtin_memcpy(y[j], x + min(at + j * LG_UNIT, nv - 4), sizeof y[j]);
    };
    const bool four = a.V >= 4;   // (a slice of fewer has others before it)
    if (!lazy && four) read(tid * 4);

    float rep = a.repetition ? a.repetition[b] : 1.0f;
    if (!(rep > 0.0f)) rep = 1.0f;   // off
    const float freq = a.frequency ? a.frequency[b] : 0.0f, pres = a.presence ? a.presence[b] : 0.0f;
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.L) : a.L, prompt = a.prompt ? min(max(a.prompt[b], 0), len) : 0;
    const bool penal = len > 0 && (rep != 1.0f || freq != 0.0f || pres != 0.0f);
    auto place = [&](int32_t t) { return (uint32_t)t - (uint32_t)v0; };   // (an id below v0 wraps to a large number)
    if (penal)
        for (int i = tid * 4; i < slice / W::PER; i += LG_UNIT) *reinterpret_cast<uint4*>(&word[i]) = uint4{ 0, 0, 0, 0 };
    if (allowed)
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (tid + k * LG_T < slice / 32) open[tid + k * LG_T] = m[k];
    // Biases: a bit for each of the slice's tokens that has one (marked), how many have one before each 32 tokens (before), and by
    // a token's number among them the last entry that names it: what a token's bias costs does not depend on how many there are.
    int32_t mine[LG_BIAS] = {};
    if (a.n_bias)
    {
        for (int i = tid; i < slice / 32; i += LG_T) marked[i] = 0;
#pragma unroll
        for (int k = 0; k < LG_BIAS; ++k)
        {
            const int i = tid + k * LG_T;
            if (i >= a.n_bias) continue;
            mine[k] = a.bias_ids[b * a.ldb + i];
            bval[i] = a.bias[b * a.ldv + i];
            last[i] = 0;
        }
    }
    if (penal || a.n_bias) __syncthreads();
    if (a.n_bias)
    {
#pragma unroll
        for (int k = 0; k < LG_BIAS; ++k)
            if (tid + k * LG_T < a.n_bias && place(mine[k]) < (uint32_t)nv)
                atomicOr(&marked[place(mine[k]) / 32], 1u << (place(mine[k]) % 32));
        __syncthreads();
        // two words a thread (a slice has at most 1024)
        const int w = tid * 2, n = slice / 32;
        const uint32_t c0 = w < n ? __popc(marked[w]) : 0, c1 = w + 1 < n ? __popc(marked[w + 1]) : 0;
        uint32_t sum = c0 + c1;
#pragma unroll
        for (int o = 1; o < 64; o *= 2)
        {
            const uint32_t up = __shfl_up(sum, o);
            if (tid % 64 >= o) sum += up;
        }
        if (tid % 64 == 63) total[tid / 64] = sum;
        __syncthreads();
        for (int k = 0; k < tid / 64; ++k) sum += total[k];
        if (w < n) before[w] = sum - c0 - c1;
        if (w + 1 < n) before[w + 1] = sum - c1;
        __syncthreads();
    }
    auto number = [&](uint32_t v) { return before[v / 32] + __popc(marked[v / 32] & ((1u << (v % 32)) - 1)); };
#pragma unroll
    for (int k = 0; k < LG_BIAS; ++k)
        if (tid + k * LG_T < a.n_bias && place(mine[k]) < (uint32_t)nv)
            atomicMax(&last[number(place(mine[k]))], (uint32_t)(tid + k * LG_T + 1));
    if (penal)
    {
        auto edge = [&](int i) {
            const uint32_t v = place(h[i]);
            if (v >= (uint32_t)nv) return;
            if (i < prompt) W::seen(word, v);
            else W::count(word, v);
        };
        // four ids that all count, on one side of the prompt's end: an id costs a subtraction, a comparison and, where it is in the
        // slice, an atomic
        for (int at = tid * 4; at < len; at += U * LG_UNIT)
        {
            if (a.L >= 4 && at != tid * 4) ids_at(at);
#pragma unroll
            for (int u = 0; u < U; ++u)
            {
                const int from = at + u * LG_UNIT;
                if (from + 4 <= prompt)
                {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (place(id[u][i]) < (uint32_t)nv) W::seen(word, place(id[u][i]));
                }
                else if (from >= prompt && from + 4 <= len)
                {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (place(id[u][i]) < (uint32_t)nv) W::count(word, place(id[u][i]));
                }
                else
                    for (int i = from; i < min(from + 4, len); ++i) edge(i);
            }
        }
    }
    if (penal || a.n_bias || allowed) __syncthreads();

    auto change = [&](int i, float (&v)[4]) {   // tokens i .. i + 3 of the slice
        uint32_t w[4] = {};
        const bool any = penal && W::four(word, i, w);
        if (any)
#pragma unroll
            for (int k = 0; k < 4; ++k)
            {
                if (w[k]) v[k] = v[k] > 0.0f ? v[k] / rep : v[k] * rep;
                const uint32_t n = w[k] & (W::SEEN - 1);
                if (n)
                {
                    v[k] -= freq * (float)n;
                    v[k] -= pres;
                }
            }
        const uint32_t mark = a.n_bias ? marked[i / 32] >> (i % 32) & 15 : 0;
        if (mark)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (mark >> k & 1) v[k] += bval[last[number(i + k)] - 1];
        if (!allowed) return;
        const uint32_t ok = open[i / 32] >> (i % 32);   // (4 tokens from a multiple of 4 on: one word)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = ok >> k & 1 ? v[k] : -INFINITY;
    };
    if (lazy)
    {
        for (int i = tid * 4; i < nv; i += LG_UNIT)
        {
            uint32_t w[4];
            if (!(penal && W::four(word, i, w)) && !(a.n_bias && (marked[i / 32] >> (i % 32) & 15))) continue;
            float v[4];
            lg_load(x + i, nv - i, v);
            change(i, v);
            lg_store(out + i, nv - i, v);
        }
        return;
    }
    for (int at = tid * 4; at < nv; at += NB * LG_UNIT)
    {
        float v[NB][4];
#pragma unroll
        for (int j = 0; j < NB; ++j)
        {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[j][k] = static_cast<float>(y[j][k]);
        }
        if (four) read(at + NB * LG_UNIT);   // the next ones, before this step's stores
#pragma unroll
        for (int j = 0; j < NB; ++j)
        {
            const int i = at + j * LG_UNIT;
            if (i >= nv) continue;
            if (i + 4 > nv) lg_load(x + i, nv - i, v[j]);
            change(i, v[j]);
            lg_store(out + i, nv - i, v[j]);
        }
    }
}

template <typename E, bool HALF>
static void logits_go(LogitsArgs a, hipStream_t st)
{
    // Bytes of words: twice in a CU. Smaller slices overlap better and each read the whole history: us by slices of 32,768, 16,384 and 8,192
    // tokens, 256 rows, 80, 84 and 88.
    constexpr int most = 65536;
    auto* kern = &logits_kernel<E, HALF>;
    static std::atomic<uint64_t> opened{ 0 };
    gm_open(reinterpret_cast<const void*>(kern), LDS_LIMIT, opened);
    const int64_t units = (int64_t)a.B * ((a.V + LG_UNIT - 1) / LG_UNIT);
    // as many slices as fill the card, no smaller than they must be: 24 rows of 100,003 by 2,048 tokens 14.8 us, 4,096 11.6, 8,192 13.8
    const int largest = a.L ? most / 4 * LgWord<HALF>::PER : a.B < 32768 ? 4 * LG_UNIT : 8 * LG_UNIT;   // (a launch has fewer than 2^32 threads)
    a.slice = (int)std::min<int64_t>(std::max<int64_t>((units + 1023) / 1024, 1) * LG_UNIT, largest);
    a.slices = (a.V + a.slice - 1) / a.slice;
    // A row's slices on one XCD read its history once from memory: us with and without, 256 rows of 30,000 81 and 84, 128 52 and 57, 64 26.5 and
    // 27.1; 16 rows, of which an XCD then has two, 18.1 and 17.8.
    a.by_xcd = a.B >= 64;
    // In place without a mask, short lists leave most logits unread; what longer ones name lies in most lines, and is slower one by one than
    // the whole row in order. us, lists alone and the whole row, 256 rows of 131,072 fp32 with 100, 2,000, 4,000, 8,000 and 30,000 ids 30 and
    // 69, 52 and 71, 57 and 72, 76 and 73, 95 and 81; bf16 with 100, 500, 2,000, 30,000 28 and 34, 39 and 38, 44 and 41, 63 and 58; 24 rows
    // of 100,003 fp32 with 100 and 4,000 9.0 and 10.8, 10.9 and 11.8.
    a.lazy = a.out == a.logits && !a.allowed && ((int64_t)a.L + a.n_bias) * 128 <= (int64_t)a.V * (int)sizeof(E);

    const unsigned grid = (unsigned)(a.by_xcd ? (a.B + 7) / 8 * 8 : a.B) * a.slices;
    const size_t lds = (a.L ? a.slice / LgWord<HALF>::PER : 0) * 4 + (a.n_bias ? a.slice / 4 + LG_T / 16 + a.n_bias * 8 : 0) + (a.allowed ? a.slice / 8 : 0);
    hipLaunchKernelGGL(kern, dim3(grid), dim3(LG_T), lds, st, a);
}

template <typename E>
static void logits_of(const LogitsArgs& a, hipStream_t st)
{
    (a.L <= 32767 ? &logits_go<E, true> : &logits_go<E, false>)(a, st);
}

void launch_logits(const LogitsArgs& a, hipStream_t st)
{
    (a.dtype == 2 ? &logits_of<float> : a.dtype == 1 ? &logits_of<__bf16> : &logits_of<_Float16>)(a, st);
}

}  // namespace gfl
