// Quantization to 8-bit floating point (e4m3) with a scale for each block of 128 (B200, sm_100a); the products are in
// ltq_fp8_gemm.cu.
//
// 128 values: s = max |x| / 448 (at least 2^-126), q = e4m3(x / s), an fp32 quotient rounded to nearest even; a block with a
// NaN or an infinity becomes NaN.  Activations: one scale per row and 128 columns; weights: one per 128 x 128 block.
#include <cuda_fp8.h>
#include "ltq_b200.h"
#include "vec_types.cuh"

namespace {

constexpr int QB = 128;
constexpr float E4M3_MAX = 448.f, S_MIN = 1.17549435e-38f;

__device__ __forceinline__ float block_scale(uint32_t amax_bits)  // the largest |x| by its bits: NaN above infinity
{
    const float s = __fdiv_rn(__uint_as_float(amax_bits), E4M3_MAX);
    return s < S_MIN ? S_MIN : s;
}
__device__ __forceinline__ uint32_t quant4(const float (&x)[4], float s)
{
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x[0], s), __fdiv_rn(x[1], s)), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x[2], s), __fdiv_rn(x[3], s)), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// four elements of a row from column c on (zeros beyond K)
template <typename T>
__device__ __forceinline__ void load4(const T* row, int c, int K, bool aligned, float (&x)[4])
{
    if (aligned && c + 4 <= K) {
        const Vec<T, 4> v = *reinterpret_cast<const Vec<T, 4>*>(row + c);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = to_f(v.v[i]);
    } else
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = c + i < K ? to_f(row[c + i]) : 0.f;
}
__device__ __forceinline__ void store4(uint8_t* row, int c, int K, uint32_t q)
{
    if (c + 4 <= K) *reinterpret_cast<uint32_t*>(row + c) = q;
    else
        for (int i = 0; c + i < K; i++) row[c + i] = (uint8_t)(q >> (8 * i));
}

// a warp per row and 128 columns
template <typename T>
__global__ void __launch_bounds__(256) quant_rows_kernel(const T* __restrict__ x, long long ld, int M, int K,
                                                         uint8_t* __restrict__ q, long long ld_q, float* __restrict__ s,
                                                         long long ld_s, int aligned)
{
    const int kb = (K + QB - 1) / QB, lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= (long long)M * kb) return;
    const int m = (int)(unit / kb), b = (int)(unit - (long long)m * kb), c = b * QB + 4 * lane;
    float v[4];
    load4(x + m * ld, c, K, aligned, v);
    uint32_t a = max(max(abs_bits(v[0]), abs_bits(v[1])), max(abs_bits(v[2]), abs_bits(v[3])));
    a = __reduce_max_sync(0xffffffffu, a);
    const float sc = block_scale(a);
    store4(q + m * ld_q, c, K, quant4(v, sc));
    if (lane == 0) s[b * ld_s + m] = sc;
}

// a CTA per 128 x 128 block
template <typename T>
__global__ void __launch_bounds__(256) quant_blocks_kernel(const T* __restrict__ w, long long ld, int N, int K,
                                                           uint8_t* __restrict__ q, long long ld_q, float* __restrict__ s,
                                                           long long ld_s, int aligned)
{
    __shared__ uint32_t red[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n0 = blockIdx.y * QB, c = blockIdx.x * QB + 4 * lane;
    uint32_t a = 0;
    float v[4];
    for (int r = warp; r < QB && n0 + r < N; r += 8) {
        load4(w + (n0 + r) * ld, c, K, aligned, v);
        a = max(a, max(max(abs_bits(v[0]), abs_bits(v[1])), max(abs_bits(v[2]), abs_bits(v[3]))));
    }
    a = __reduce_max_sync(0xffffffffu, a);
    if (lane == 0) red[warp] = a;
    __syncthreads();
    for (int i = 0; i < 8; i++) a = max(a, red[i]);
    const float sc = block_scale(a);
    for (int r = warp; r < QB && n0 + r < N; r += 8) {
        load4(w + (n0 + r) * ld, c, K, aligned, v);
        store4(q + (n0 + r) * ld_q, c, K, quant4(v, sc));
    }
    if (threadIdx.x == 0) s[blockIdx.y * ld_s + blockIdx.x] = sc;
}

template <typename T>
int quant_rows(const void* x, long long ld, int M, int K, uint8_t* q, long long ld_q, float* s, long long ld_s, cudaStream_t st)
{
    const long long units = (long long)M * ((K + QB - 1) / QB);
    const int aligned = (uintptr_t)x % (4 * sizeof(T)) == 0 && ld % 4 == 0;
    quant_rows_kernel<T><<<(unsigned)((units + 7) / 8), 256, 0, st>>>((const T*)x, ld, M, K, q, ld_q, s, ld_s, aligned);
    return (int)cudaGetLastError();
}
template <typename T>
int quant_blocks(const void* w, long long ld, int N, int K, uint8_t* q, long long ld_q, float* s, long long ld_s, cudaStream_t st)
{
    const int aligned = (uintptr_t)w % (4 * sizeof(T)) == 0 && ld % 4 == 0;
    const dim3 grid((K + QB - 1) / QB, (N + QB - 1) / QB);
    quant_blocks_kernel<T><<<grid, 256, 0, st>>>((const T*)w, ld, N, K, q, ld_q, s, ld_s, aligned);
    return (int)cudaGetLastError();
}

}  // namespace

extern "C" int ltq_fp8_quant_rows(const void* x, int dtype, long long ld, int M, int K, uint8_t* q, long long ld_q, float* s,
                                  long long ld_s, void* stream)
{
    const int es = dt_bytes(dtype);
    if (!es || M < 0 || K < 1 || ld < K || ld_s < M || ld_q % 16 || ld_q < K) return -1;
    if (M == 0) return 0;
    if (!x || (uintptr_t)x % es || !q || (uintptr_t)q % 16 || !s || (uintptr_t)s % 4) return -1;
    if ((long long)M * ((K + QB - 1) / QB) > (1LL << 33)) return -1;
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F32) return quant_rows<float>(x, ld, M, K, q, ld_q, s, ld_s, st);
    if (dtype == DT_BF16) return quant_rows<__nv_bfloat16>(x, ld, M, K, q, ld_q, s, ld_s, st);
    return quant_rows<__half>(x, ld, M, K, q, ld_q, s, ld_s, st);
}

extern "C" int ltq_fp8_quant_blocks(const void* w, int dtype, long long ld, int N, int K, uint8_t* q, long long ld_q, float* s,
                                    long long ld_s, void* stream)
{
    const int es = dt_bytes(dtype);
    if (!es || N < 0 || N > 65535 * QB || K < 1 || ld < K || ld_s < (K + QB - 1) / QB || ld_q % 16 || ld_q < K) return -1;
    if (N == 0) return 0;
    if (!w || (uintptr_t)w % es || !q || (uintptr_t)q % 16 || !s || (uintptr_t)s % 4) return -1;
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F32) return quant_blocks<float>(w, ld, N, K, q, ld_q, s, ld_s, st);
    if (dtype == DT_BF16) return quant_blocks<__nv_bfloat16>(w, ld, N, K, q, ld_q, s, ld_s, st);
    return quant_blocks<__half>(w, ld, N, K, q, ld_q, s, ld_s, st);
}
