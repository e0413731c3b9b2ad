// Logits as a request's settings change them before a token is drawn: penalties for tokens that were there before, biases, a mask.
//
// A workgroup takes a slice of a row. What the row's history and biases say of each of the slice's tokens is gathered in a word of
// LDS a token by integer atomics (sums and maxima: the same in any order), then the slice is read, changed and written once.
#include "gfl_internal.hpp"

#include <algorithm>

namespace gfl {

constexpr int LG_T = 512;
constexpr uint32_t LG_SEEN = 1u << 20, LG_COUNT = LG_SEEN - 1;   // a token's word: bias entry + 1 | seen | count
constexpr int LG_BIAS = 21;

template <typename E>
__global__ __launch_bounds__(LG_T) void logits_kernel(LogitsArgs a, int slice)
{
    extern __shared__ uint32_t word[];
    const int64_t b = blockIdx.y;
    const int v0 = blockIdx.x * slice, nv = min(slice, a.V - v0);
    const E* x = static_cast<const E*>(a.logits) + b * a.ld + v0;
    E* out = static_cast<E*>(a.out) + b * a.ldo + v0;

    float rep = a.repetition ? a.repetition[b] : 1.0f;
    if (!(rep > 0.0f)) rep = 1.0f;   // off
    const float freq = a.frequency ? a.frequency[b] : 0.0f, pres = a.presence ? a.presence[b] : 0.0f;
    const bool penal = a.L > 0 && (rep != 1.0f || freq != 0.0f || pres != 0.0f);
    const bool words = penal || a.n_bias > 0;
    if (words)
    {
        for (int i = threadIdx.x; i < nv; i += LG_T) word[i] = 0;
        __syncthreads();
        const int32_t* ids = a.n_bias ? a.bias_ids + b * a.ldb : nullptr;
        for (int i = threadIdx.x; i < a.n_bias; i += LG_T)
        {
            const uint32_t v = (uint32_t)(ids[i] - v0);
            if (ids[i] >= v0 && v < (uint32_t)nv) atomicMax(&word[v], (uint32_t)(i + 1) << LG_BIAS);   // the last entry counts
        }
        __syncthreads();
        if (penal)
        {
            const int32_t* h = a.history + b * a.ldh;
            const int len = a.lengths ? min(max(a.lengths[b], 0), a.L) : a.L;
            const int prompt = a.prompt ? min(max(a.prompt[b], 0), len) : 0;
            for (int i = threadIdx.x; i < len; i += LG_T)
            {
                const int id = h[i];
                const uint32_t v = (uint32_t)(id - v0);
                if (id < v0 || v >= (uint32_t)nv) continue;
                if (i < prompt) atomicOr(&word[v], LG_SEEN);
                else atomicAdd(&word[v], 1u);
            }
        }
        __syncthreads();
    }
    const float* by = a.n_bias ? a.bias + b * a.ldv : nullptr;
    const int32_t* allowed = a.allowed ? a.allowed + b * a.lda : nullptr;
    for (int i = threadIdx.x; i < nv; i += LG_T)
    {
        float y = static_cast<float>(x[i]);
        const uint32_t w = words ? word[i] : 0;
        if (w)
        {
            if (w & (LG_SEEN | LG_COUNT)) y = y > 0.0f ? y / rep : y * rep;
            if (w & LG_COUNT)
            {
                y -= freq * (float)(w & LG_COUNT);
                y -= pres;
            }
            if (w >> LG_BIAS) y += by[(w >> LG_BIAS) - 1];
        }
        const int v = v0 + i;
        if (allowed && !(allowed[v / 32] >> (v % 32) & 1)) y = -INFINITY;
        out[i] = static_cast<E>(y);
    }
}

void launch_logits(const LogitsArgs& a, hipStream_t st)
{
    const int slice = 8192;
    const dim3 grid((a.V + slice - 1) / slice, a.B);
    auto* kern = a.dtype == 2 ? &logits_kernel<float> : a.dtype == 1 ? &logits_kernel<__bf16> : &logits_kernel<_Float16>;
    hipLaunchKernelGGL(kern, grid, dim3(LG_T), slice * sizeof(uint32_t), st, a, slice);
}

}  // namespace gfl
