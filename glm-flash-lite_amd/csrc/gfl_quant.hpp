// A row's scale and its elements to 8 bits, for the launches that quantise tokens.
#pragma once
#include "gfl_internal.hpp"

namespace gfl {

template <bool BF>
__device__ __forceinline__ float q_val(uint16_t b)
{
    return BF ? __uint_as_float((uint32_t)b << 16) : static_cast<float>(__builtin_bit_cast(_Float16, b));
}

// max |x| is the integer maximum of the magnitudes' bits (`top`), which puts NaN above infinity above every number, so a row
// that is not finite is seen as such. q = x * 127 / max: the product is exact in fp32 (at most 18 significant bits), so the
// correctly rounded quotient lies on the true side of every half and q is the exact rounding. Values past 2^100 are scaled
// down first so that the product stays finite.
template <bool BF>
struct QRow
{
    float scale, pre, amax;
    uint16_t mask;   // of the elements: none for a row of zeros or one that is not finite
    __device__ __forceinline__ explicit QRow(uint32_t top)
    {
        amax = q_val<BF>((uint16_t)top);
        scale = amax / 127.0f;
        const bool ok = top != 0 && top < (BF ? 0x7F80u : 0x7C00u);
        mask = ok ? 0xFFFF : 0;
        pre = amax > 0x1p100f ? 0x1p-64f : 1.0f;
        amax = ok ? amax * pre : 1.0f;
    }
    __device__ __forceinline__ int8_t one(uint16_t b) const
    {
        return (int8_t)(int)rintf(q_val<BF>(b & mask) * pre * 127.0f / amax);
    }
    __device__ __forceinline__ uint64_t eight(const uint16_t (&v)[8]) const
    {
        uint64_t o = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) o |= (uint64_t)(uint8_t)one(v[i]) << (8 * i);
        return o;
    }
};

// scale at place `at` ([groups][N]) of a 4-bit weight
__device__ __forceinline__ float q4_scale(const Q4Args& a, int64_t at)
{
    const uint16_t b = static_cast<const uint16_t*>(a.scale)[at];
    return a.scale_bf ? q_val<true>(b) : q_val<false>(b);
}

}  // namespace gfl
