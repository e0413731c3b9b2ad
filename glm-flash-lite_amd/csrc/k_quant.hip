// Rows of 16-bit activations to 8 bits with a scale each.
#include "gfl_quant.hpp"

namespace gfl {

// A workgroup per row. Bound by memory: K is read once (16 values a thread stay in registers; longer rows are read again, from
// cache). bf16 16384 x 8192 99 us (4.05 TB/s; a large copy reaches 4.8), 4096 x 5120 22 (2.9), 9 x 4096 4.0, the launch; rows that
// start at no multiple of 16 bytes go value by value: 4096 x 5123 43.
constexpr int QT = 256;

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
    const QRow<BF> r(top);
    if (threadIdx.x == 0) scale[m] = r.scale;
    for (int c = threadIdx.x, s = 0; c < nv; c += QT, ++s)
    {
        u16x8 v;
        if (s == 0) v = keep[0];
        else if (s == 1) v = keep[1];
        else v = *reinterpret_cast<const u16x8*>(row + 8 * c);
        uint16_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = v[i];
        *reinterpret_cast<uint64_t*>(out + 8 * c) = r.eight(e);
    }
    for (int k = 8 * nv + threadIdx.x; k < K; k += QT) out[k] = r.one(row[k]);
}

void launch_quant_i8(const void* x, int64_t ldx, int bf16, int M, int K, int8_t* q, int64_t ldq, float* scale, hipStream_t st)
{
    const uint16_t* p = static_cast<const uint16_t*>(x);
    if (bf16) hipLaunchKernelGGL(quant_i8_kernel<true>, dim3(M), dim3(QT), 0, st, p, ldx, K, q, ldq, scale);
    else hipLaunchKernelGGL(quant_i8_kernel<false>, dim3(M), dim3(QT), 0, st, p, ldx, K, q, ldq, scale);
}

}  // namespace gfl
