// Element types of the token, logit and 8-bit operators: codes of the C ABI, 16-byte vectors, conversions through fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace {

constexpr int DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2;  // `dtype` arguments of include/ltq_b200.h

inline int dt_bytes(int dt) { return dt == DT_F32 ? 4 : (dt == DT_BF16 || dt == DT_F16) ? 2 : 0; }

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// y[i] = v in the type of the code
__device__ __forceinline__ void store_as(void* y, int dt, long long i, float v)
{
    if (dt == DT_F32) ((float*)y)[i] = v;
    else if (dt == DT_BF16) ((__nv_bfloat16*)y)[i] = from_f<__nv_bfloat16>(v);
    else ((__half*)y)[i] = from_f<__half>(v);
}

// V elements of T moved as one access of V * sizeof(T) bytes (2, 4, 8, 16 or 32: two of 16)
template <typename T, int V>
struct alignas(V * sizeof(T) > 16 ? 16 : V * sizeof(T)) Vec {
    T v[V];
};
// the fp32 values of 16 bytes of T
__device__ __forceinline__ void unpack16(const uint4& u, float (&f)[4], float)
{
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack16(const uint4& u, float (&f)[8], __nv_bfloat16)
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ __forceinline__ void unpack16(const uint4& u, float (&f)[8], __half)
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
}
// two fp32 values in a 64-bit register pair, and products and sums of both in one instruction
__device__ __forceinline__ uint64_t pair(float x, float y)
{
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ float2 unpair(uint64_t v)
{
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// the largest element of 16 bytes of T (NaN only where all are)
__device__ __forceinline__ float max16(const uint4& u, float)
{
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
}
__device__ __forceinline__ float max16(const uint4& u, __nv_bfloat16)
{
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float max16(const uint4& u, __half)
{
    const __half2* h = reinterpret_cast<const __half2*>(&u);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
}
// 16 bytes of T with the elements of `mask` (bit i: element i) replaced by -infinity
__device__ __forceinline__ uint4 mask16(uint4 u, uint32_t mask, float)
{
    uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (mask >> i & 1u) w[i] = 0xff800000u;
    return u;
}
__device__ __forceinline__ uint4 mask16_16(uint4 u, uint32_t mask, uint32_t inf)
{
    uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (mask >> (2 * i) & 1u) w[i] = (w[i] & 0xffff0000u) | inf;
        if (mask >> (2 * i + 1) & 1u) w[i] = (w[i] & 0xffffu) | inf << 16;
    }
    return u;
}
__device__ __forceinline__ uint4 mask16(uint4 u, uint32_t mask, __nv_bfloat16) { return mask16_16(u, mask, 0xff80u); }
__device__ __forceinline__ uint4 mask16(uint4 u, uint32_t mask, __half) { return mask16_16(u, mask, 0xfc00u); }
__device__ __forceinline__ uint4 pack16(const float (&f)[4], float)
{
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 pack16(const float (&f)[8], __nv_bfloat16)
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack16(const float (&f)[8], __half)
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// barrier of the cluster's CTAs: shared and global writes before it are seen by all of them after it (those of a thread that
// arrives relaxed need not be)
__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
// writes a 32-bit word at `p` of this CTA's shared memory into the same place of CTA `rank`
__device__ __forceinline__ void st_cluster_u32(const void* p, uint32_t rank, uint32_t v)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(a), "r"(v) : "memory");
}

}  // namespace
