// Token table lookup with scaling, and the table's gradient by sorted tokens (B200, sm_100a).
//
//     lookup    y_i = s E[t_i]                       one rounding, to the table's type
//     gradient  dE[v] = s sum_{i : t_i = v} dy_i     fp32 sums in the order of i, one rounding to the output's type
//
// A token outside [0, V) reads as a row of zeros and takes no gradient; neither does the padding token.
//
// The gradient runs in three launches.  (1) One cluster of 8 CTAs sorts the positions by token (stable, least digit
// first, 10 bits a pass); the other CTAs meanwhile write zeros to the table rows that no token names.  (2) The sorted
// list is cut into chunks of equal length; a warp sums one chunk's rows over 32 vectors of the width and writes the rows
// whose positions all lie in the chunk, and the sums of the rows that reach over its ends to a workspace.  (3) Those
// sums are joined from the row's first chunk to its last.  Nothing depends on the order in which CTAs run.
#include "ltq_b200.h"
#include "stride_grid.cuh"
#include "vec_types.cuh"

namespace {

__device__ __forceinline__ long long load_token(const void* t, int t64, long long i)
{
    return t64 ? ((const long long*)t)[i] : ((const int*)t)[i];
}

// ---------------------------------------------------------------------------------------------------------- lookup

template <typename T, int VEC>
__global__ void __launch_bounds__(256) lookup_kernel(const T* __restrict__ E, long long ld, const void* __restrict__ tok,
                                                     int t64, long long n, int V, int nv, float scale, T* __restrict__ out,
                                                     long long ld_out)
{
    const long long total = n * nv;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
        const long long r = i / nv;
        const int v = (int)(i - r * nv);
        const long long t = load_token(tok, t64, r);
        Vec<T, VEC> x;
        if (t >= 0 && t < V) {
            x = *reinterpret_cast<const Vec<T, VEC>*>(E + t * ld + (long long)v * VEC);
#pragma unroll
            for (int q = 0; q < VEC; q++) x.v[q] = from_f<T>(to_f(x.v[q]) * scale);
        } else
#pragma unroll
            for (int q = 0; q < VEC; q++) x.v[q] = from_f<T>(0.f);
        *reinterpret_cast<Vec<T, VEC>*>(out + r * ld_out + (long long)v * VEC) = x;
    }
}

// the widest access (in elements of es bytes) that rows of D elements at these addresses and strides allow
int access_width(int es, int D, const void* a, long long lda, const void* b, long long ldb)
{
    for (int w = 16 / es; w > 1; w /= 2)
        if (D % w == 0 && lda % w == 0 && ldb % w == 0 && ((uintptr_t)a % (w * es)) == 0 && ((uintptr_t)b % (w * es)) == 0)
            return w;
    return 1;
}

template <typename T, int VEC>
int lookup_launch(const void* E, long long ld, const void* tok, int t64, long long n, int V, int D, float scale, void* out,
                  long long ld_out, cudaStream_t st)
{
    const int nv = D / VEC;
    const long long need = (n * nv + 255) / 256;
    lookup_kernel<T, VEC><<<stride_grid(need, 8), 256, 0, st>>>((const T*)E, ld, tok, t64, n, V, nv, scale, (T*)out, ld_out);
    return (int)cudaGetLastError();
}

// -------------------------------------------------------------------------------------------------------- gradient

constexpr int S_THREADS = 1024, S_WARPS = 32, S_CL = 8;
constexpr int DIGIT = 10, BINS = 1 << DIGIT;
constexpr int FILL_ROWS = 1 << 17;  // rows of a fill CTA's bitmap at a time
constexpr int SORT_SMEM = (S_WARPS * BINS + S_CL * BINS + 64) * 4;
static_assert(BINS == S_THREADS, "one thread per bin");
static_assert(FILL_ROWS / 32 <= S_WARPS * BINS, "the fill's bitmap fits the histograms' memory");

struct SortParams {
    const void* tok;
    int t64;
    int n, V, passes;
    long long pad;  // padding token, or -1
    uint32_t* key[2];
    uint32_t* pos[2];  // pass p reads buffer 1 - (p & 1) (the first: the tokens) and writes buffer p & 1
    // fill
    uint8_t* out;
    long long ld_bytes, row_bytes;
    int fill_ctas;
};

// buffer of the sorted list
inline int sorted_buffer(int passes) { return (passes - 1) & 1; }

__device__ __forceinline__ uint32_t sort_key(const SortParams& p, long long i)
{
    const long long t = load_token(p.tok, p.t64, i);
    return t >= 0 && t < p.V && t != p.pad ? (uint32_t)t : (uint32_t)p.V;  // what takes no gradient sorts to the end
}

__device__ void sort_cluster(const SortParams& p, uint32_t* sm)
{
    uint32_t* hist = sm;                        // [warp][bin]
    uint32_t* all = sm + S_WARPS * BINS;        // [CTA of the cluster][bin]
    uint32_t* wsum = all + S_CL * BINS;         // 32 warp sums
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = (int)cluster_rank();
    const int gw = rank * S_WARPS + warp;
    const int per = (p.n + S_CL * S_WARPS * 32 - 1) / (S_CL * S_WARPS * 32) * 32;  // positions of a warp
    const long long a = (long long)gw * per;
    const int i0 = (int)(a < p.n ? a : p.n), i1 = (int)(a + per < p.n ? a + per : p.n);
    uint32_t* mine = hist + warp * BINS;
    for (int pass = 0; pass < p.passes; pass++) {
        const int shift = pass * DIGIT;
        const uint32_t* ik = p.key[(pass & 1) ^ 1];
        const uint32_t* ip = p.pos[(pass & 1) ^ 1];
        uint32_t *ok = p.key[pass & 1], *op = p.pos[pass & 1];
        for (int w = 0; w < S_WARPS; w++) hist[w * BINS + tid] = 0;
        __syncthreads();
        for (int i = i0 + lane; i < i1; i += 32) {
            const uint32_t k = pass == 0 ? sort_key(p, i) : ik[i];
            atomicAdd(&mine[(k >> shift) & (BINS - 1)], 1u);
        }
        __syncthreads();
        uint32_t run = 0;  // thread = bin: the warps' counts become offsets within the CTA
        for (int w = 0; w < S_WARPS; w++) {
            const uint32_t c = hist[w * BINS + tid];
            hist[w * BINS + tid] = run;
            run += c;
        }
        for (int q = 0; q < S_CL; q++) st_cluster_u32(&all[rank * BINS + tid], q, run);
        cluster_arrive();
        cluster_wait();
        uint32_t tot = 0, before = 0;
        for (int q = 0; q < S_CL; q++) {
            const uint32_t c = all[q * BINS + tid];
            before += q < rank ? c : 0;
            tot += c;
        }
        uint32_t inc = tot;  // exclusive scan of the totals over the bins
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
        }
        if (lane == 31) wsum[warp] = inc;
        __syncthreads();
        uint32_t base = 0;
        for (int w = 0; w < warp; w++) base += wsum[w];
        base += inc - tot + before;
        for (int w = 0; w < S_WARPS; w++) hist[w * BINS + tid] += base;
        __syncthreads();
        for (int g = i0; g < i1; g += 32) {  // in the order of the list: stable
            const int i = g + lane;
            const bool on = i < i1;
            const uint32_t k = on ? (pass == 0 ? sort_key(p, i) : ik[i]) : 0;
            const uint32_t ps = on ? (pass == 0 ? (uint32_t)i : ip[i]) : 0;
            const uint32_t d = on ? (k >> shift) & (BINS - 1) : BINS;
            const uint32_t peers = __match_any_sync(0xffffffffu, d);
            const int leader = __ffs(peers) - 1;
            uint32_t at = 0;
            if (on && lane == leader) {
                at = mine[d];
                mine[d] = at + __popc(peers);
            }
            at = __shfl_sync(0xffffffffu, at, leader) + __popc(peers & ((1u << lane) - 1));
            if (on) ok[at] = k, op[at] = ps;
            __syncwarp();
        }
        cluster_arrive();  // the pass's list is written, and `all` is free again
        cluster_wait();
    }
}

template <int B>  // bytes of a store
__device__ void zero_row(uint8_t* row, long long bytes, int lane)
{
    for (long long o = lane * B; o < bytes; o += 32 * B) {
        if (B == 16) *reinterpret_cast<uint4*>(row + o) = make_uint4(0, 0, 0, 0);
        else if (B == 4) *reinterpret_cast<uint32_t*>(row + o) = 0;
        else *reinterpret_cast<uint16_t*>(row + o) = 0;
    }
}

__device__ void fill_rows(const SortParams& p, uint32_t* bits, int f)
{
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const long long per = (p.V + p.fill_ctas - 1) / p.fill_ctas;
    const long long b0 = f * per, b1 = b0 + per < p.V ? b0 + per : p.V;
    const int width = !((uintptr_t)p.out % 16 || p.ld_bytes % 16 || p.row_bytes % 16)  ? 16
                      : !((uintptr_t)p.out % 4 || p.ld_bytes % 4 || p.row_bytes % 4) ? 4
                                                                                     : 2;
    for (long long r0 = b0; r0 < b1; r0 += FILL_ROWS) {
        const int nr = (int)(b1 - r0 < FILL_ROWS ? b1 - r0 : FILL_ROWS);
        for (int i = tid; i < (nr + 31) / 32; i += S_THREADS) bits[i] = 0;
        __syncthreads();
        for (int i = tid; i < p.n; i += S_THREADS) {
            const long long t = load_token(p.tok, p.t64, i);
            if (t >= r0 && t < r0 + nr && t != p.pad) atomicOr(&bits[(t - r0) >> 5], 1u << ((t - r0) & 31));
        }
        __syncthreads();
        for (int r = warp; r < nr; r += S_WARPS) {
            if (bits[r >> 5] >> (r & 31) & 1u) continue;
            uint8_t* row = p.out + (r0 + r) * p.ld_bytes;
            if (width == 16) zero_row<16>(row, p.row_bytes, lane);
            else if (width == 4) zero_row<4>(row, p.row_bytes, lane);
            else zero_row<2>(row, p.row_bytes, lane);
        }
        __syncthreads();
    }
}

__global__ void __cluster_dims__(S_CL, 1, 1) __launch_bounds__(S_THREADS, 1) sort_fill_kernel(const SortParams p)
{
    extern __shared__ uint32_t sm[];
    const int cluster = blockIdx.x / S_CL;
    if (cluster == 0) sort_cluster(p, sm);
    else fill_rows(p, sm, blockIdx.x - S_CL);
}

struct SumParams {
    const uint32_t* key;
    const uint32_t* pos;
    const void* d;
    long long ld_d;
    void* out;
    long long ld_out;
    float* part;  // [chunk][2][D]: the sum of a row begun in an earlier chunk; of one that a later chunk goes on with
    int n, V, D, chunk, nchunks, accumulate;
    float scale;
};

template <typename TO, int VEC>
__device__ __forceinline__ void write_row(const SumParams& p, uint32_t row, int v, const float (&a)[VEC])
{
    TO* o = (TO*)p.out + (long long)row * p.ld_out + (long long)v * VEC;
    Vec<TO, VEC> x;
    if (p.accumulate) {
        x = *reinterpret_cast<const Vec<TO, VEC>*>(o);
#pragma unroll
        for (int q = 0; q < VEC; q++) x.v[q] = from_f<TO>(fmaf(p.scale, a[q], to_f(x.v[q])));
    } else
#pragma unroll
        for (int q = 0; q < VEC; q++) x.v[q] = from_f<TO>(p.scale * a[q]);
    *reinterpret_cast<Vec<TO, VEC>*>(o) = x;
}

template <int VEC>
__device__ __forceinline__ void store_part(float* part, const float (&a)[VEC])
{
    Vec<float, VEC> x;
#pragma unroll
    for (int q = 0; q < VEC; q++) x.v[q] = a[q];
    *reinterpret_cast<Vec<float, VEC>*>(part) = x;
}

template <typename TI, typename TO, int VEC>
__global__ void __launch_bounds__(128) sum_chunks_kernel(const SumParams p)
{
    const int lane = threadIdx.x, ch = blockIdx.x * 4 + threadIdx.y, v = blockIdx.y * 32 + lane, nv = p.D / VEC;
    if (ch >= p.nchunks) return;
    const int c0 = ch * p.chunk, c1 = min(p.n, c0 + p.chunk);
    uint32_t cur = p.key[c0];
    if (cur >= (uint32_t)p.V) return;  // from here on nothing takes a gradient
    const bool on = v < nv;
    const bool open = c0 > 0 && p.key[c0 - 1] == cur;  // the first row was begun in an earlier chunk
    bool first = true;
    float a[VEC];
#pragma unroll
    for (int q = 0; q < VEC; q++) a[q] = 0.f;
    float* part = p.part + (long long)ch * 2 * p.D + (long long)v * VEC;
    for (int i = c0; i < c1; i++) {
        const uint32_t k = p.key[i];
        if (k != cur) {
            if (on) {
                if (first && open) store_part<VEC>(part, a);
                else write_row<TO, VEC>(p, cur, v, a);
            }
            first = false;
            cur = k;
#pragma unroll
            for (int q = 0; q < VEC; q++) a[q] = 0.f;
            if (cur >= (uint32_t)p.V) return;
        }
        if (on) {
            const Vec<TI, VEC> x =
                *reinterpret_cast<const Vec<TI, VEC>*>((const TI*)p.d + (long long)p.pos[i] * p.ld_d + (long long)v * VEC);
#pragma unroll
            for (int q = 0; q < VEC; q++) a[q] += to_f(x.v[q]);
        }
    }
    if (!on) return;
    if (first && open) store_part<VEC>(part, a);  // the chunk is the middle or the end of a row begun earlier
    else if (c1 < p.n && p.key[c1] == cur) store_part<VEC>(part + p.D, a);
    else write_row<TO, VEC>(p, cur, v, a);
}

template <typename TO, int VEC>
__global__ void __launch_bounds__(128) join_chunks_kernel(const SumParams p)
{
    const int ch = blockIdx.x * 4 + threadIdx.y, v = blockIdx.y * 32 + threadIdx.x;
    if (ch >= p.nchunks - 1 || v >= p.D / VEC) return;
    const int c0 = ch * p.chunk, c1 = c0 + p.chunk;
    const uint32_t k = p.key[c1 - 1];
    if (k >= (uint32_t)p.V || p.key[c1] != k) return;               // no row goes on into the next chunk
    if (c0 > 0 && p.key[c0] == k && p.key[c0 - 1] == k) return;     // it was begun earlier: joined from there
    float a[VEC];
    const float* part = p.part + (long long)ch * 2 * p.D + (long long)v * VEC;
#pragma unroll
    for (int q = 0; q < VEC; q++) a[q] = part[p.D + q];
    for (int c = ch + 1; c < p.nchunks && p.key[c * p.chunk] == k; c++) {
        part += 2 * p.D;
#pragma unroll
        for (int q = 0; q < VEC; q++) a[q] += part[q];
    }
    write_row<TO, VEC>(p, k, v, a);
}

constexpr long long N_MAX = 1LL << 30;  // positions of a gradient call
constexpr int D_MAX = 1 << 20;

// positions of a chunk: about a thousand chunks, 8 positions at least
int chunk_of(long long n) { return (int)(n <= 8192 ? 8 : (n + 1023) / 1024); }
size_t align256(size_t b) { return (b + 255) / 256 * 256; }

template <typename TI, typename TO, int VEC>
int sum_launch(const SumParams& p, cudaStream_t st)
{
    const dim3 grid((p.nchunks + 3) / 4, (p.D / VEC + 31) / 32), block(32, 4);
    sum_chunks_kernel<TI, TO, VEC><<<grid, block, 0, st>>>(p);
    if (p.nchunks > 1) join_chunks_kernel<TO, VEC><<<grid, block, 0, st>>>(p);
    return (int)cudaGetLastError();
}
template <typename TI, typename TO>
int sum_dispatch(const SumParams& p, cudaStream_t st)
{
    constexpr int W = 16 / sizeof(TI);
    if (p.D % W == 0 && p.ld_d % W == 0 && p.ld_out % W == 0 && (uintptr_t)p.d % 16 == 0 && (uintptr_t)p.out % 16 == 0)
        return sum_launch<TI, TO, W>(p, st);
    return sum_launch<TI, TO, 1>(p, st);
}
template <typename TI>
int sum_type(const SumParams& p, int odt, cudaStream_t st)
{
    if (odt == DT_F32) return sum_dispatch<TI, float>(p, st);
    if (odt == DT_BF16) return sum_dispatch<TI, __nv_bfloat16>(p, st);
    return sum_dispatch<TI, __half>(p, st);
}

}  // namespace

extern "C" int ltq_embed_lookup(const void* table, int dtype, long long ld, const void* tokens, int tok64, long long n,
                                int V, int D, float scale, void* out, long long ld_out, void* stream)
{
    const int es = dt_bytes(dtype);
    if (!es || n < 0 || V < 1 || D < 1 || ld < D || ld_out < D) return -1;
    if (n == 0) return 0;
    if (!table || !tokens || !out || (uintptr_t)table % es || (uintptr_t)out % es || (uintptr_t)tokens % (tok64 ? 8 : 4)) return -1;
    const cudaStream_t st = (cudaStream_t)stream;
    const int w = access_width(es, D, table, ld, out, ld_out);
#define LOOKUP(T, VEC) return lookup_launch<T, VEC>(table, ld, tokens, tok64, n, V, D, scale, out, ld_out, st)
    if (dtype == DT_F32) {
        if (w == 4) LOOKUP(float, 4);
        if (w == 2) LOOKUP(float, 2);
        LOOKUP(float, 1);
    }
    if (dtype == DT_BF16) {
        if (w == 8) LOOKUP(__nv_bfloat16, 8);
        if (w >= 2) LOOKUP(__nv_bfloat16, 2);
        LOOKUP(__nv_bfloat16, 1);
    }
    if (w == 8) LOOKUP(__half, 8);
    if (w >= 2) LOOKUP(__half, 2);
    LOOKUP(__half, 1);
#undef LOOKUP
}

extern "C" size_t ltq_embed_grad_workspace_bytes(long long n, int D)
{
    if (n <= 0 || n > N_MAX || D < 1 || D > D_MAX) return 0;
    const int c = chunk_of(n);
    return 4 * align256(4 * (size_t)n) + align256(8 * (size_t)((n + c - 1) / c) * D);
}

extern "C" int ltq_embed_grad(const void* tokens, int tok64, long long n, int V, long long padding, const void* dout,
                              int dtype, long long ld_d, int D, float scale, void* out, int out_dtype, long long ld_out,
                              int accumulate, void* workspace, size_t workspace_bytes, void* stream)
{
    const int es = dt_bytes(dtype), eo = dt_bytes(out_dtype);
    if (!es || !eo || n < 0 || n > N_MAX || V < 1 || V > (1 << 30) || D < 1 || D > D_MAX || ld_d < D || ld_out < D) return -1;
    if (!out || (uintptr_t)out % eo) return -1;
    if (n == 0 && accumulate) return 0;
    if (n > 0 && (!tokens || !dout || (uintptr_t)dout % es || (uintptr_t)tokens % (tok64 ? 8 : 4) || !workspace ||
                  ((uintptr_t)workspace & 255) || workspace_bytes < ltq_embed_grad_workspace_bytes(n, D)))
        return -1;
    const cudaStream_t st = (cudaStream_t)stream;
    SortParams s{};
    s.tok = tokens, s.t64 = tok64 != 0, s.n = (int)n, s.V = V, s.pad = padding;
    s.passes = 1;
    while (s.passes * DIGIT < 31 && ((unsigned)V >> (s.passes * DIGIT))) s.passes++;
    uint8_t* ws = (uint8_t*)workspace;
    const size_t a = align256(4 * (size_t)n);
    for (int i = 0; i < 2; i++) s.key[i] = (uint32_t*)(ws + 2 * i * a), s.pos[i] = (uint32_t*)(ws + (2 * i + 1) * a);
    s.out = (uint8_t*)out, s.ld_bytes = ld_out * eo, s.row_bytes = (long long)D * eo;
    static std::atomic<int> clusters[64];  // clusters of the sort kernel that a device holds at once
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
    int nc = clusters[dev].load(std::memory_order_acquire);
    if (nc == 0) {
        cudaError_t e = cudaFuncSetAttribute(sort_fill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SORT_SMEM);
        if (e != cudaSuccess) return (int)e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(S_CL), cfg.blockDim = dim3(S_THREADS), cfg.dynamicSmemBytes = SORT_SMEM;
        if ((e = cudaOccupancyMaxActiveClusters(&nc, sort_fill_kernel, &cfg)) != cudaSuccess) return (int)e;
        if (nc < 2) nc = 2;
        clusters[dev].store(nc, std::memory_order_release);
    }
    s.fill_ctas = accumulate ? 0 : (nc - 1) * S_CL;
    sort_fill_kernel<<<S_CL + s.fill_ctas, S_THREADS, SORT_SMEM, st>>>(s);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || n == 0) return (int)e;
    SumParams p{};
    const int b = sorted_buffer(s.passes);
    p.key = s.key[b], p.pos = s.pos[b], p.d = dout, p.ld_d = ld_d, p.out = out, p.ld_out = ld_out;
    p.part = (float*)(ws + 4 * a);
    p.n = (int)n, p.V = V, p.D = D, p.chunk = chunk_of(n), p.accumulate = accumulate != 0, p.scale = scale;
    p.nchunks = (int)((n + p.chunk - 1) / p.chunk);
    if (dtype == DT_F32) return sum_type<float>(p, out_dtype, st);
    if (dtype == DT_BF16) return sum_type<__nv_bfloat16>(p, out_dtype, st);
    return sum_type<__half>(p, out_dtype, st);
}
