// Rows of 16-bit activations to 8 bits with a scale each.
#include "gfl_internal.hpp"

namespace gfl {

// A workgroup per row. max |x| is the integer maximum of the magnitudes' bits, which puts NaN above infinity above every
// number, so a row that is not finite is seen as such. q = x * 127 / max: the product is exact in fp32 (at most 18
// significant bits), so the correctly rounded quotient lies on the true side of every half and q is the exact rounding.
// Values past 2^100 are scaled down first so that the product stays finite. Bound by memory: K is read once (16 values a
// thread stay in registers; longer rows are read again, from cache).
constexpr int QT = 256;

template <bool BF>
__device__ __forceinline__ float q_val(uint16_t b)
{
    return BF ? __uint_as_float((uint32_t)b << 16) : static_cast<float>(__builtin_bit_cast(_Float16, b));
}

template <bool BF>
__global__ __launch_bounds__(QT) void quant_i8_kernel(const uint16_t* x, int64_t ldx, int K, int8_t* q, int64_t ldq,
                                                      float* scale)
{
    __shared__ uint32_t red[QT / 64];
    const int64_t m = blockIdx.x;
    const uint16_t* row = x + m * ldx;
    int8_t* out = q + m * ldq;
    const bool vec = (reinterpret_cast<uintptr_t>(row) & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0;
    const int nv = vec ? K / 8 : 0;   // whole chunks of 8
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    u16x8 keep[2];
    uint32_t top = 0;
    for (int c = threadIdx.x, s = 0; c < nv; c += QT, ++s)
    {
        const u16x8 v = *reinterpret_cast<const u16x8*>(row + 8 * c);
        if (s == 0) keep[0] = v;
        if (s == 1) keep[1] = v;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, (uint32_t)(v[i] & 0x7FFF));
    }
    for (int k = 8 * nv + threadIdx.x; k < K; k += QT) top = max(top, (uint32_t)(row[k] & 0x7FFF));
#pragma unroll
    for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = top;
    __syncthreads();
    top = max(max(red[0], red[1]), max(red[2], red[3]));
    float amax = q_val<BF>((uint16_t)top);
    if (threadIdx.x == 0) scale[m] = amax / 127.0f;
    const bool ok = top != 0 && top < (BF ? 0x7F80u : 0x7C00u);
    const float pre = amax > 0x1p100f ? 0x1p-64f : 1.0f;
    amax *= pre;
    auto one = [&](uint16_t b) { return ok ? (int8_t)(int)rintf(q_val<BF>(b) * pre * 127.0f / amax) : (int8_t)0; };
    for (int c = threadIdx.x, s = 0; c < nv; c += QT, ++s)
    {
        u16x8 v;
        if (s == 0) v = keep[0];
        else if (s == 1) v = keep[1];
        else v = *reinterpret_cast<const u16x8*>(row + 8 * c);
        uint64_t o = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) o |= (uint64_t)(uint8_t)one(v[i]) << (8 * i);
        *reinterpret_cast<uint64_t*>(out + 8 * c) = o;
    }
    for (int k = 8 * nv + threadIdx.x; k < K; k += QT) out[k] = one(row[k]);
}

void launch_quant_i8(const void* x, int64_t ldx, int bf16, int M, int K, int8_t* q, int64_t ldq, float* scale, hipStream_t st)
{
    const uint16_t* p = static_cast<const uint16_t*>(x);
    if (bf16) hipLaunchKernelGGL(quant_i8_kernel<true>, dim3(M), dim3(QT), 0, st, p, ldx, K, q, ldq, scale);
    else hipLaunchKernelGGL(quant_i8_kernel<false>, dim3(M), dim3(QT), 0, st, p, ldx, K, q, ldq, scale);
}

}  // namespace gfl
