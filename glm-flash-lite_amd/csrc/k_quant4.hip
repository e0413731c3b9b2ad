// Weights of 4 bits: rounding, packing and unpacking.
//
// A row of K values lies in blocks of 128, 64 bytes each: the 32-bit word j of the 16-byte piece g holds the inputs 32 j + 8 g + 0, 2, 4,
// 6, 1, 3, 5, 7, four bits each from the lowest on. A lane that loads a piece so has, in word j, the 8 values of lane group g of the
// j-th MFMA of 32 inputs, and a shift and a mask put two neighbours into the halves of a register.
#include "gfl_quant.hpp"

namespace gfl {

constexpr int Q4_T = 256;

// A thread per word: the row, the block and the first of its 8 inputs, in the inputs' order (so that a group's threads are neighbours),
// and where the word lies. N * blocks * 16 is at most 2^29.
struct Q4Place
{
    uint32_t n;
    int k;
    int64_t at;   // bytes
    __device__ __forceinline__ Q4Place(uint32_t id, uint32_t words)
    {
        n = id / words;
        const int in = (int)(id - n * words), t = in % 16;
        k = in * 8;
        at = (int64_t)n * words * 4 + in / 16 * 64 + t % 4 * 16 + t / 4 * 4;
    }
};
// values 0, 2, 4, 6, 1, 3, 5, 7 from the lowest bits on
__device__ __forceinline__ uint32_t q4_word(const uint32_t (&u)[8])
{
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= u[i] << (i / 2 * 4 + i % 2 * 16);
    return w;
}

// Symmetric: scale = max |w| / 7, value = w / scale rounded + 8. With zero points: scale = (max - min) / 15 with 0 in the range, zero =
// -min / scale rounded, value = w / scale rounded + zero. The scale is rounded to w's type first. A group that is all zeros, or
// whose scale rounds to zero, has scale 0; one that holds an infinity or a NaN a scale of NaN: both have values of 8. Past K there are zeros,
// which are in every range.
// 12288 x 5120 bf16 68 us, bound by eight divisions a thread (bytes 31; a wave a block, two inputs a lane and words joined by shuffles,
// took 190); pack_i4 20 (bytes 19; 72).
template <typename E>
__global__ __launch_bounds__(Q4_T) void quant_i4_kernel(const E* w, int64_t ld, int N, int K, int group, int blocks, uint8_t* q,
                                                        E* scale, uint8_t* zero)
{
    const uint32_t words = blocks * 16, id = blockIdx.x * Q4_T + threadIdx.x;
    if (id >= N * words) return;   // (16 threads together)
    const Q4Place p(id, words);
    const E* row = w + p.n * ld;
    E e[8] = {};
    if (p.k + 8 <= K) __builtin_memcpy(e, row + p.k, sizeof e);
    else
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (p.k + i < K) e[i] = row[p.k + i];
    float v[8], lo = 0.0f, hi = 0.0f;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        v[i] = static_cast<float>(e[i]);
        bad |= !(fabsf(v[i]) < INFINITY);
        lo = fminf(lo, v[i]);
        hi = fmaxf(hi, v[i]);
    }
    for (int o = 1; o < group / 8; o *= 2)
    {
        lo = fminf(lo, __shfl_xor(lo, o));
        hi = fmaxf(hi, __shfl_xor(hi, o));
        bad |= (uint32_t)__shfl_xor((int)bad, o);
    }
    // (a range past the largest number is halved first, which is exact there)
    const float half = fmaxf(-lo, hi) > 0x1p126f ? 0.5f : 1.0f;
    const float wide = zero ? (hi * half - lo * half) / (15.0f * half) : fmaxf(-lo, hi) / 7.0f;
    const E se = bad ? static_cast<E>(NAN) : static_cast<E>(wide);
    const float s = static_cast<float>(se);
    const bool some = s > 0.0f && !bad;
    const float z = zero && some ? fminf(rintf(-lo / s), 15.0f) : 8.0f;
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = p.k + i >= K ? 0 : some ? (uint32_t)fminf(fmaxf(rintf(v[i] / s) + z, 0.0f), 15.0f) : 8;
    *reinterpret_cast<uint32_t*>(q + p.at) = q4_word(u);
    if (p.k % group == 0 && p.k < K)
    {
        const int64_t g = (int64_t)(p.k / group) * N + p.n;
        scale[g] = se;
        if (zero) zero[g] = (uint8_t)z;
    }
}

__global__ __launch_bounds__(Q4_T) void pack_i4_kernel(const uint8_t* v, int64_t ld, int N, int K, int blocks, uint8_t* q)
{
    const uint32_t words = blocks * 16, id = blockIdx.x * Q4_T + threadIdx.x;
    if (id >= N * words) return;
    const Q4Place p(id, words);
    const uint8_t* row = v + p.n * ld;
    uint8_t e[8] = {};
    if (p.k + 8 <= K) __builtin_memcpy(e, row + p.k, sizeof e);
    else
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (p.k + i < K) e[i] = row[p.k + i];
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = e[i] & 15;
    *reinterpret_cast<uint32_t*>(q + p.at) = q4_word(u);
}

// (value - zero) * scale, rounded to E once, as rows of ldw elements (K up to a multiple of 8): what the
// large products read as their weights. A thread per word: 12288 x 5120 35 us, 4.5 TB/s.
template <typename E>
__global__ __launch_bounds__(Q4_T) void dequant_i4_kernel(Q4Args a, E* w, int64_t ldw)
{
    const uint32_t words = a.blocks * 16, at = blockIdx.x * Q4_T + threadIdx.x;   // (at most 2^29)
    if (at >= a.N * words) return;
    const int64_t n = at / words;
    const int in = (int)(at % words), k = in / 16 * 128 + in % 4 * 32 + in / 4 % 4 * 8;
    if (k >= a.K) return;
    const uint32_t u = reinterpret_cast<const uint32_t*>(a.q)[at];
    const int64_t g = (int64_t)(k / a.group) * a.N + n;
    const float s = q4_scale(a, g), z = a.zero ? (float)a.zero[g] : 8.0f;
    typedef E e8 __attribute__((ext_vector_type(8)));
    e8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        const int v = u >> (i / 2 * 4 + i % 2 * 16) & 15;
        o[i] = static_cast<E>(((float)v - z) * s);
    }
    *reinterpret_cast<e8*>(w + n * ldw + k) = o;
}

static unsigned q4_grid(int64_t n, int per) { return (unsigned)((n + per - 1) / per); }

void launch_quant_i4(const void* w, int64_t ld, int bf16, int N, int K, int group, uint8_t* q, void* scale, uint8_t* zero,
                     hipStream_t st)
{
    const int blocks = (K + 127) / 128;
    const dim3 grid(q4_grid((int64_t)N * blocks * 16, Q4_T)), block(Q4_T);
    if (bf16)
        hipLaunchKernelGGL(quant_i4_kernel<__bf16>, grid, block, 0, st, static_cast<const __bf16*>(w), ld, N, K, group, blocks, q,
                           static_cast<__bf16*>(scale), zero);
    else
        hipLaunchKernelGGL(quant_i4_kernel<_Float16>, grid, block, 0, st, static_cast<const _Float16*>(w), ld, N, K, group, blocks, q,
                           static_cast<_Float16*>(scale), zero);
}

void launch_pack_i4(const uint8_t* v, int64_t ld, int N, int K, uint8_t* q, hipStream_t st)
{
    const int blocks = (K + 127) / 128;
    hipLaunchKernelGGL(pack_i4_kernel, dim3(q4_grid((int64_t)N * blocks * 16, Q4_T)), dim3(Q4_T), 0, st, v, ld, N, K, blocks, q);
}

void launch_dequant_i4(const Q4Args& a, int bf16, void* w, int64_t ldw, hipStream_t st)
{
    const dim3 grid(q4_grid((int64_t)a.N * a.blocks * 16, Q4_T));
    if (bf16) hipLaunchKernelGGL(dequant_i4_kernel<__bf16>, grid, dim3(Q4_T), 0, st, a, static_cast<__bf16*>(w), ldw);
    else hipLaunchKernelGGL(dequant_i4_kernel<_Float16>, grid, dim3(Q4_T), 0, st, a, static_cast<_Float16*>(w), ldw);
}

}  // namespace gfl
