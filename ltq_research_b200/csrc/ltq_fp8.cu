// Quantization to 8-bit floating point (e4m3) with a scale for each block of 128 (B200, sm_100a); the products are in
// ltq_fp8_gemm.cu.
//
// 128 values: s = max |x| / 448 (at least 2^-126), q = e4m3(x / s), an fp32 quotient rounded to nearest even; a block with a
// NaN or an infinity becomes NaN.  Activations: one scale per row and 128 columns; weights: one per 128 x 128 block.
#include "launch_next.cuh"
#include "ltq_b200.h"
#include "fp8_quant.cuh"

namespace {

__device__ __forceinline__ uint32_t quant4(const float (&x)[4], float s)
{
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x[0], s), __fdiv_rn(x[1], s)), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x[2], s), __fdiv_rn(x[3], s)), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

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

// Activations.  A warp takes 1024 columns of ROWS rows, eight columns a lane and load (16 bytes of a 16-bit type), so a block of
// 128 is half a warp's load; four blocks' maxima are exchanged together; a row's loads are in flight while the row before it is
// worked on.  The scales of a CTA's rows are gathered in shared memory and leave as one run of rows per block, the layout the products
// read.  Bound by memory: 8192 x 4096 bf16 (67 MB in, 35 MB out) 18 us, 5.6 TB/s; 1003 x 128256 61 us, 6.4 TB/s (75 with the maxima
// exchanged one by one and a slow path that divides; 180 with a division a value and a warp a block).
template <typename T, int ROWS>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 3) quant_rows_kernel(const T* __restrict__ x, long long ld, int M, int K,
                                                         uint8_t* __restrict__ q, long long ld_q, float* __restrict__ s,
                                                         long long ld_s, int aligned)
{
    __shared__ float sc[8][8 * ROWS];
    next_may_start();  // the product
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, groups = (K + 1023) / 1024;
    const int group = blockIdx.x % groups, c0 = group * 1024, mb = blockIdx.x / groups * (8 * ROWS);
    const int m0 = mb + warp * ROWS, m1 = min(M, m0 + ROWS);
    Raw8<T> next[4];
    if (m0 < m1)
#pragma unroll
        for (int j = 0; j < 4; j++) load8(x + (long long)m0 * ld, c0 + 256 * j + 8 * lane, K, aligned, next[j]);
    for (int m = m0; m < m1; m++) {
        Raw8<T> cur[4];
#pragma unroll
        for (int j = 0; j < 4; j++) cur[j] = next[j];
        if (m + 1 < m1)  // the next row's loads are on their way while this one is worked on
#pragma unroll
            for (int j = 0; j < 4; j++) load8(x + (m + 1) * ld, c0 + 256 * j + 8 * lane, K, aligned, next[j]);
        float scale[4], rec[4];
        scales4(cur, lane, scale, rec);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float v[8];
            unpack8(cur[j], v);
            const uint2 w = quant8(v, scale[j], rec[j]);
            const int c = c0 + 256 * j + 8 * lane;
            uint8_t* o = q + m * ld_q + c;
            if (c + 8 <= K) *reinterpret_cast<uint2*>(o) = w;
            else
                for (int i = 0; c + i < K; i++) o[i] = (uint8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
            if ((lane & 15) == 0) sc[2 * j + (lane >> 4)][m - mb] = scale[j];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * 8 * ROWS; i += 256) {
        const int b = group * 8 + i / (8 * ROWS), m = mb + i % (8 * ROWS);
        if (b * QB < K && m < M) s[b * ld_s + m] = sc[i / (8 * ROWS)][i % (8 * ROWS)];
    }
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

// 8-bit transpose, 64 x 64 bytes through shared memory
__global__ void __launch_bounds__(256) transpose8_kernel(const uint8_t* __restrict__ q, long long ld, int R, int C,
                                                         uint8_t* __restrict__ out, long long ld_out)
{
    __shared__ uint8_t t[64][68];
    const long long r0 = blockIdx.y * 64LL, c0 = blockIdx.x * 64LL;
    const int x = (threadIdx.x & 15) * 4, y = threadIdx.x >> 4;
#pragma unroll
    for (int i = y; i < 64; i += 16) {
        if (r0 + i >= R) break;
        const uint8_t* p = q + (r0 + i) * ld + c0 + x;
        if (c0 + x + 4 <= C) *reinterpret_cast<uint32_t*>(&t[i][x]) = *reinterpret_cast<const uint32_t*>(p);
        else
            for (int e = 0; c0 + x + e < C; e++) t[i][x + e] = p[e];
    }
    __syncthreads();
#pragma unroll
    for (int i = y; i < 64; i += 16) {
        if (c0 + i >= C) break;
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) w |= (uint32_t)(r0 + x + e < R ? t[x + e][i] : 0) << (8 * e);
        // a row's padding up to ld_out is written too, as zeros
        if (r0 + x < ld_out) *reinterpret_cast<uint32_t*>(out + (c0 + i) * ld_out + r0 + x) = w;
    }
}

template <typename T, int ROWS>
int quant_rows(const void* x, long long ld, int M, int K, uint8_t* q, long long ld_q, float* s, long long ld_s, cudaStream_t st)
{
    const int aligned = (uintptr_t)x % 16 == 0 && ld * sizeof(T) % 16 == 0;
    const long long grid = (K + 1023LL) / 1024 * ((M + 8LL * ROWS - 1) / (8 * ROWS));
    if (grid > 0x7fffffff) return -1;
    quant_rows_kernel<T, ROWS><<<(unsigned)grid, 256, 0, st>>>((const T*)x, ld, M, K, q, ld_q, s, ld_s, aligned);
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
    if (M > 0x7fffffff - 32 || K > 0x7fffffff - 2048) return -1;
    const cudaStream_t st = (cudaStream_t)stream;
    // one row a warp while that fills the GPU no more than a few times over, else four
    const bool few = (long long)M * ((K + 1023) / 1024) < 8192;
#define QUANT(T) return few ? quant_rows<T, 1>(x, ld, M, K, q, ld_q, s, ld_s, st) : quant_rows<T, 4>(x, ld, M, K, q, ld_q, s, ld_s, st)
    if (dtype == DT_F32) QUANT(float);
    if (dtype == DT_BF16) QUANT(__nv_bfloat16);
    QUANT(__half);
#undef QUANT
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

extern "C" int ltq_fp8_transpose(const uint8_t* q, long long ld, int R, int C, uint8_t* out, long long ld_out, void* stream)
{
    if (R < 1 || C < 1 || ld < C || ld % 4 || ld_out < R || ld_out % 16 || !q || (uintptr_t)q % 4 || !out || (uintptr_t)out % 16 ||
        R > 65535 * 64 || ld_out > ((long long)R + 63) / 64 * 64)
        return -1;
    transpose8_kernel<<<dim3((C + 63) / 64, (R + 63) / 64), 256, 0, (cudaStream_t)stream>>>(q, ld, R, C, out, ld_out);
    return (int)cudaGetLastError();
}
