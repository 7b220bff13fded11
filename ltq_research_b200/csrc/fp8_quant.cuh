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
// eight values under one scale s (r: its reciprocal, rounded correctly), as eight bytes.  The quotients x / s are rounded correctly
// without a division each: q = x r and then q + (x - q s) r is the correctly rounded quotient (Markstein's correction, IBM J.
// Res. Dev. 34, 1990) while the remainder stays above the smallest normal number, which 2^-80 <= s guarantees for every quotient
// that e4m3 does not round to 0; below, x and s are taken 2^64 times as large, which is exact
__device__ __forceinline__ uint2 quant8(float (&v)[8], float s, float r)
{
    if (!(s >= 0x1p-80f)) {  // a tiny scale, or NaN
        s *= 0x1p64f, r *= 0x1p-64f;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= 0x1p64f;
    }
    const uint64_t rr = pair(r, r), ns = pair(-s, -s);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint64_t x = pair(v[i], v[i + 1]), q = mul2(x, rr);
        const float2 y = unpair(fma2(fma2(q, ns, x), rr, q));
        v[i] = y.x, v[i + 1] = y.y;
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        w[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
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

// the largest |x| of eight elements, by its fp32 bits (16-bit types: two at a time, as unsigned integers, NaN above infinity)
__device__ __forceinline__ uint32_t amax8(const Raw8<float>& x)
{
    float f[8];
    unpack8(x, f);
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) a = max(a, abs_bits(f[i]));
    return a;
}
__device__ __forceinline__ uint32_t amax16_bits(const uint4& u)
{
    const uint32_t m = 0x7fff7fffu;
    const uint32_t a = __vmaxu2(__vmaxu2(u.x & m, u.y & m), __vmaxu2(u.z & m, u.w & m));
    return max(a >> 16, a & 0xffffu);
}
__device__ __forceinline__ uint32_t amax8(const Raw8<__nv_bfloat16>& x) { return amax16_bits(x.u[0]) << 16; }
__device__ __forceinline__ uint32_t amax8(const Raw8<__half>& x)
{
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)amax16_bits(x.u[0]))));
}
// over the half warp that holds a block
__device__ __forceinline__ uint32_t half_warp_max(uint32_t a)
{
#pragma unroll
    for (int o = 8; o; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
    return a;
}
// The scales and reciprocals of four pairs of blocks, a half warp's load each.  The maxima are exchanged so that a lane ends with that
// of one of the four and divides for it alone; the others take the results from there.
template <typename T>
__device__ __forceinline__ void scales4(const Raw8<T> (&x)[4], int lane, float (&s)[4], float (&r)[4])
{
    uint32_t a[4];
#pragma unroll
    for (int j = 0; j < 4; j++) a[j] = amax8(x[j]);
    const bool b0 = lane & 1, b1 = lane & 2;
    const uint32_t k0 = max(b0 ? a[1] : a[0], __shfl_xor_sync(0xffffffffu, b0 ? a[0] : a[1], 1));
    const uint32_t k1 = max(b0 ? a[3] : a[2], __shfl_xor_sync(0xffffffffu, b0 ? a[2] : a[3], 1));
    uint32_t mine = max(b1 ? k1 : k0, __shfl_xor_sync(0xffffffffu, b1 ? k0 : k1, 2));
    mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 4));
    mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 8));
    const float sc = block_scale(mine), rc = __frcp_rn(sc);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        s[j] = __shfl_sync(0xffffffffu, sc, (lane & 16) | j);
        r[j] = __shfl_sync(0xffffffffu, rc, (lane & 16) | j);
    }
}

}  // namespace
