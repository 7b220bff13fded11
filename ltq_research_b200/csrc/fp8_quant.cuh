// Scales and values of e4m3 blocks of 128 (shared by the quantization kernels and the product for few rows).
#pragma once
#include <cuda_fp8.h>
#include <string.h>
#include "vec_types.cuh"

namespace {

constexpr int QB = 128;  // width of a block of K under one scale
constexpr float E4M3_MAX = 448.f, S_MIN = 1.17549435e-38f;

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ float block_scale(uint32_t amax_bits)  // the largest |x| by its bits: NaN above infinity
{
    const float s = __fdiv_rn(__uint_as_float(amax_bits), E4M3_MAX);
    return s < S_MIN ? S_MIN : s;
}
// x / s rounded correctly without a division each: with r = 1 / s correctly rounded, q = x r and then q + (x - q s) r is the
// correctly rounded quotient (Markstein's correction, IBM J. Res. Dev. 34, 1990) while the remainder stays above the smallest
// normal number, which 2^-80 <= s guarantees for every quotient that e4m3 does not round to 0
__device__ __forceinline__ float quotient(float x, float s, float r)
{
    const float q = __fmul_rn(x, r);
    return __fmaf_rn(__fmaf_rn(-q, s, x), r, q);
}
// eight values under one scale, as eight bytes
__device__ __forceinline__ uint2 quant8(float (&v)[8], float scale)
{
    if (!(scale >= 0x1p-80f)) {  // a tiny scale, or NaN
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __fdiv_rn(v[i], scale);
    } else {
        const float r = __frcp_rn(scale);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = quotient(v[i], scale, r);
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        w[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}
// the largest |v| of a block whose eight-value pieces lie on half a warp
__device__ __forceinline__ uint32_t half_warp_amax(const float (&v)[8])
{
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) a = max(a, abs_bits(v[i]));
#pragma unroll
    for (int o = 8; o; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
    return a;
}

// eight elements of a row from column c on (zeros beyond K), as they are
template <typename T>
struct Raw8 {
    uint4 u[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ void load8(const T* row, int c, int K, bool aligned, Raw8<T>& x)
{
    if (aligned && c + 8 <= K) {
#pragma unroll
        for (int h = 0; h < (int)sizeof(T) / 2; h++) x.u[h] = __ldg(reinterpret_cast<const uint4*>(row + c) + h);
    } else {
        T t[8];
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = c + i < K ? row[c + i] : from_f<T>(0.f);
        memcpy(&x, t, sizeof(x));
    }
}
__device__ __forceinline__ void unpack8(const Raw8<float>& x, float (&f)[8])
{
    f[0] = __uint_as_float(x.u[0].x), f[1] = __uint_as_float(x.u[0].y), f[2] = __uint_as_float(x.u[0].z), f[3] = __uint_as_float(x.u[0].w);
    f[4] = __uint_as_float(x.u[1].x), f[5] = __uint_as_float(x.u[1].y), f[6] = __uint_as_float(x.u[1].z), f[7] = __uint_as_float(x.u[1].w);
}
__device__ __forceinline__ void unpack8(const Raw8<__nv_bfloat16>& x, float (&f)[8]) { unpack16(x.u[0], f, __nv_bfloat16()); }
__device__ __forceinline__ void unpack8(const Raw8<__half>& x, float (&f)[8]) { unpack16(x.u[0], f, __half()); }

}  // namespace
