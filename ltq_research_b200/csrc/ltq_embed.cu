// Token table lookup with scaling, and the table's gradient by sorted tokens (B200, sm_100a).
//
//     lookup    y_i = s E[t_i]                       one rounding, to the table's type
//     gradient  dE[v] = s sum_{i : t_i = v} dy_i     fp32 sums, one rounding to the output's type
//
// A token outside [0, V) reads as a row of zeros and takes no gradient; neither does the padding token.
//
// The gradient runs in three launches.  (1) The positions are sorted by token (stable) and zeros written to some of the table
// rows that no token names.  Up to 8192 positions every CTA counts the ranks of a few positions; beyond, one cluster of 8 CTAs
// sorts (least digit first, 10 bits a pass) while the other CTAs write the zeros.  (2) The sorted list is cut into chunks of
// equal length; a warp sums one chunk's rows over 32 vectors of the width and writes the rows whose positions all lie in the
// chunk, and the sums of the rows that reach over its ends to a workspace; the last CTAs write the zeros that are left.
// (3) The sums are joined from the row's first chunk to its last.  Nothing depends on the order in which CTAs run.
//
// So a row's sum is grouped by the places of its positions in the sorted list: in the order of i within a chunk, the chunks' sums
// added in order; of nine chunks or more, in eight stretches of equally many chunks, these added in order.  The grouping follows from
// the tokens and from n and D (chunk_of): the same bits at every call, but not those of one sum over all i.
//
// Both directions are bound by memory.  Lookup of 16384 rows of 2560 bf16: 27 us, 6.2 TB/s.  Gradient of 16384 positions (bf16)
// into 128256 x 2048 fp32, 1.1 GB of it written: 193 us, 5.8 TB/s; 33 us sort and the zeros beside it, 143 us sums and the other
// zeros, 10 us joins.
#include <algorithm>

#include "launch_next.cuh"
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

constexpr int S_THREADS = 512, S_WARPS = 16, S_CL = 8;  // two CTAs an SM, so that the fill uses all of them
constexpr int DIGIT = 10, BINS = 1 << DIGIT;
constexpr int FILL_ROWS = 1 << 15;  // rows of a fill CTA's bitmap at a time
constexpr int RANK_BITS = FILL_ROWS / 32;
constexpr int SORT_SMEM = (S_WARPS * BINS + S_CL * BINS + BINS + 64) * 4;
constexpr int KEPT = 4;  // groups of 32 positions that a warp keeps in registers between counting and scattering
static_assert(BINS == 2 * S_THREADS, "two bins a thread");
static_assert(FILL_ROWS / 32 <= S_WARPS * BINS, "the fill's bitmap fits the histograms' memory");

// Zeros to the rows that no token names, in equal shares: the first `early` rows of each share beside the sort, the others beside
// the sums, so that neither leaves the memory idle.
struct Fill {
    uint8_t* out;
    long long ld_bytes, row_bytes;
    int V, shares, parts;  // CTAs of a share's later rows
    long long early;
    int* start;  // [shares]: sorted keys below the share's later rows; NULL without positions, when no row is late
    __device__ void share(int f, long long& b0, long long& b1, long long& e) const
    {
        const long long per = (V + shares - 1) / shares;
        b0 = f * per < V ? f * per : V;
        b1 = b0 + per < V ? b0 + per : V;
        e = b0 + early < b1 ? b0 + early : b1;
    }
};

struct SortParams {
    const void* tok;
    int t64;
    int n, V, passes;
    long long pad;  // padding token, or -1
    uint32_t* key[2];
    uint32_t* pos[2];  // pass p reads buffer 1 - (p & 1) (the first: the tokens) and writes buffer p & 1
    Fill fill;
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
    uint32_t* base = all + S_CL * BINS;         // first place of this CTA's keys of a bin
    uint32_t* wsum = base + BINS;               // warp sums
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = (int)cluster_rank();
    const int gw = rank * S_WARPS + warp;
    const int per = (p.n + S_CL * S_WARPS * 32 - 1) / (S_CL * S_WARPS * 32) * 32;  // positions of a warp
    const long long a = (long long)gw * per;
    const int i0 = (int)(a < p.n ? a : p.n), i1 = (int)(a + per < p.n ? a + per : p.n);
    const bool kept = per <= 32 * KEPT;
    uint32_t* mine = hist + warp * BINS;
    cluster_arrive_relaxed();  // paired with the first pass's wait: the others' shared memory is written once they have started
    for (int pass = 0; pass < p.passes; pass++) {
        const int shift = pass * DIGIT;
        const uint32_t* ik = p.key[(pass & 1) ^ 1];
        const uint32_t* ip = p.pos[(pass & 1) ^ 1];
        uint32_t *ok = p.key[pass & 1], *op = p.pos[pass & 1];
        uint32_t kr[KEPT], pr[KEPT];
        if (kept) {
#pragma unroll
            for (int q = 0; q < KEPT; q++) {
                const int i = i0 + 32 * q + lane;
                kr[q] = i < i1 ? (pass == 0 ? sort_key(p, i) : ik[i]) : 0;
                pr[q] = i < i1 ? (pass == 0 ? (uint32_t)i : ip[i]) : 0;
            }
        }
        for (int i = tid; i < S_WARPS * BINS / 4; i += S_THREADS) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        if (kept) {
#pragma unroll
            for (int q = 0; q < KEPT; q++)
                if (i0 + 32 * q + lane < i1) atomicAdd(&mine[(kr[q] >> shift) & (BINS - 1)], 1u);
        } else
            for (int i = i0 + lane; i < i1; i += 32) {
                const uint32_t k = pass == 0 ? sort_key(p, i) : ik[i];
                atomicAdd(&mine[(k >> shift) & (BINS - 1)], 1u);
            }
        __syncthreads();
        // a thread's two bins (adjacent): the warps' counts become offsets within the CTA
        uint2 run = make_uint2(0, 0), c[S_WARPS];
#pragma unroll
        for (int w = 0; w < S_WARPS; w++) c[w] = reinterpret_cast<const uint2*>(hist + w * BINS)[tid];
#pragma unroll
        for (int w = 0; w < S_WARPS; w++) {
            reinterpret_cast<uint2*>(hist + w * BINS)[tid] = run;
            run.x += c[w].x, run.y += c[w].y;
        }
        if (pass == 0) cluster_wait();  // the later passes have the barrier at the end of the one before
        for (int q = 0; q < S_CL; q++) {
            st_cluster_u32(&all[rank * BINS + 2 * tid], q, run.x);
            st_cluster_u32(&all[rank * BINS + 2 * tid + 1], q, run.y);
        }
        cluster_arrive();
        cluster_wait();
        uint2 tot = make_uint2(0, 0), before = make_uint2(0, 0);
#pragma unroll
        for (int q = 0; q < S_CL; q++) {
            const uint2 v = reinterpret_cast<const uint2*>(all + q * BINS)[tid];
            if (q < rank) before.x += v.x, before.y += v.y;
            tot.x += v.x, tot.y += v.y;
        }
        uint32_t inc = tot.x + tot.y;  // exclusive scan of the totals over the bins
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
        }
        if (lane == 31) wsum[warp] = inc;
        __syncthreads();
        uint32_t first = inc - tot.x - tot.y;
        for (int w = 0; w < warp; w++) first += wsum[w];
        base[2 * tid] = first + before.x;
        base[2 * tid + 1] = first + tot.x + before.y;
        __syncthreads();
        auto scatter = [&](bool on, uint32_t k, uint32_t ps) {  // 32 positions in the order of the list: stable
            const uint32_t d = on ? (k >> shift) & (BINS - 1) : BINS;
            const uint32_t peers = __match_any_sync(0xffffffffu, d);
            const int leader = __ffs(peers) - 1;
            uint32_t at = 0;
            if (on && lane == leader) {
                const uint32_t o = mine[d];
                at = o + base[d];
                mine[d] = o + __popc(peers);
            }
            at = __shfl_sync(0xffffffffu, at, leader) + __popc(peers & ((1u << lane) - 1));
            if (on) ok[at] = k, op[at] = ps;
            __syncwarp();
        };
        if (kept) {
#pragma unroll
            for (int q = 0; q < KEPT; q++) scatter(i0 + 32 * q + lane < i1, kr[q], pr[q]);
        } else
            for (int g = i0; g < i1; g += 32) {
                const int i = g + lane;
                const bool on = i < i1;
                scatter(on, on ? (pass == 0 ? sort_key(p, i) : ik[i]) : 0, on ? (pass == 0 ? (uint32_t)i : ip[i]) : 0);
            }
        cluster_arrive();  // the pass's list is written, and `all` is free again
        cluster_wait();
    }
}

template <int B>  // bytes of a store
__device__ void zero_row(uint8_t* row, long long bytes, int lane)
{
    for (long long o = lane * B; o < bytes; o += 32 * B) {
        if (B == 16) __stcs(reinterpret_cast<uint4*>(row + o), make_uint4(0, 0, 0, 0));
        else if (B == 4) *reinterpret_cast<uint32_t*>(row + o) = 0;
        else *reinterpret_cast<uint16_t*>(row + o) = 0;
    }
}

// zeros to rows r0 .. r0 + nr - 1 whose bit is not set, a warp a row
__device__ void zero_rows(const Fill& p, const uint32_t* bits, long long r0, int nr, int warp, int warps, int lane)
{
    const int width = !((uintptr_t)p.out % 16 || p.ld_bytes % 16 || p.row_bytes % 16)  ? 16
                      : !((uintptr_t)p.out % 4 || p.ld_bytes % 4 || p.row_bytes % 4) ? 4
                                                                                     : 2;
    for (int r = warp; r < nr; r += warps) {
        if (bits[r >> 5] >> (r & 31) & 1u) continue;
        uint8_t* row = p.out + (r0 + r) * p.ld_bytes;
        if (width == 16) zero_row<16>(row, p.row_bytes, lane);
        else if (width == 4) zero_row<4>(row, p.row_bytes, lane);
        else zero_row<2>(row, p.row_bytes, lane);
    }
}

// The early rows of share f, and where its later rows' keys will begin; keys: all sort keys in shared memory, or NULL to read the
// tokens.
__device__ void fill_early(const SortParams& p, uint32_t* bits, int f, const uint32_t* keys)
{
    __shared__ int below;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    long long b0, b1, e;
    p.fill.share(f, b0, b1, e);
    if (tid == 0) below = 0;
    long long r0 = b0;
    do {  // once at least, for the count
        const int nr = (int)(e - r0 < FILL_ROWS ? e - r0 : FILL_ROWS);
        for (int i = tid; i < (nr + 31) / 32; i += S_THREADS) bits[i] = 0;
        __syncthreads();
        int c = 0;
        for (int i = tid; i < p.n; i += S_THREADS) {
            const long long t = keys ? (long long)keys[i] : (long long)sort_key(p, i);
            c += t < e;
            if (t >= r0 && t < r0 + nr) atomicOr(&bits[(t - r0) >> 5], 1u << ((t - r0) & 31));
        }
        if (r0 == b0) {
            c = __reduce_add_sync(0xffffffffu, c);
            if (lane == 0) atomicAdd(&below, c);
        }
        __syncthreads();
        zero_rows(p.fill, bits, r0, nr, warp, S_WARPS, lane);
        __syncthreads();
        r0 += FILL_ROWS;
    } while (r0 < e);
    if (tid == 0 && p.fill.start) p.fill.start[f] = below;
}

// A part of share f's later rows, by a CTA of 128 threads; the sorted keys are there now.
constexpr int LATE_BYTES = 49152, LATE_ROWS = 4096;
__device__ void fill_late(const Fill& p, const uint32_t* key, int n, int f, int part)
{
    __shared__ uint32_t bits[LATE_ROWS / 32];
    const int tid = threadIdx.y * 32 + threadIdx.x;
    long long b0, b1, e;
    p.share(f, b0, b1, e);
    const long long step = (b1 - e + p.parts - 1) / p.parts, p0 = e + part * step, p1 = p0 + step < b1 ? p0 + step : b1;
    for (long long r0 = p0; r0 < p1; r0 += LATE_ROWS) {
        const int nr = (int)(p1 - r0 < LATE_ROWS ? p1 - r0 : LATE_ROWS);
        for (int i = tid; i < LATE_ROWS / 32; i += 128) bits[i] = 0;
        __syncthreads();
        for (int i = p.start[f] + tid; i < n; i += 128 * 8) {
            uint32_t k[8];
#pragma unroll
            for (int q = 0; q < 8; q++) k[q] = i + 128 * q < n ? key[i + 128 * q] : 0xffffffffu;
#pragma unroll
            for (int q = 0; q < 8; q++)
                if (k[q] >= r0 && k[q] < r0 + nr) atomicOr(&bits[(k[q] - r0) >> 5], 1u << ((k[q] - r0) & 31));
            if (k[7] >= r0 + nr) break;
        }
        __syncthreads();
        zero_rows(p, bits, r0, nr, tid >> 5, 4, tid & 31);
        __syncthreads();
    }
}

// Few positions: a position's place in the sorted list is the number of smaller keys and of equal keys before it, counted by a
// warp over all keys in shared memory.  4099 positions: 9 us, where the digit passes of one cluster take 21.
constexpr int RANK_MAX = 8192;
__global__ void __launch_bounds__(S_THREADS, 2) rank_fill_kernel(const SortParams p)
{
    __shared__ __align__(16) uint32_t key[RANK_MAX];
    __shared__ uint32_t bits[RANK_BITS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n4 = (p.n + 3) / 4;
    next_may_start();
    for (int i = tid; i < 4 * n4; i += S_THREADS) key[i] = i < p.n ? sort_key(p, i) : 0xffffffffu;
    __syncthreads();
    for (int i = blockIdx.x * S_WARPS + warp; i < p.n; i += gridDim.x * S_WARPS) {
        const uint32_t k = key[i];
        int below = 0;
        for (int j = lane; j < n4; j += 32) {
            const uint4 q = reinterpret_cast<const uint4*>(key)[j];
            const int e = 4 * j;
            below += (q.x < k || (q.x == k && e < i)) + (q.y < k || (q.y == k && e + 1 < i)) + (q.z < k || (q.z == k && e + 2 < i)) +
                     (q.w < k || (q.w == k && e + 3 < i));
        }
        below = __reduce_add_sync(0xffffffffu, below);
        if (lane == 0) p.key[0][below] = k, p.pos[0][below] = i;
    }
    if (p.fill.shares) {
        __syncthreads();
        fill_early(p, bits, blockIdx.x, key);
    }
}

__global__ void __cluster_dims__(S_CL, 1, 1) __launch_bounds__(S_THREADS, 2) sort_fill_kernel(const SortParams p)
{
    extern __shared__ uint32_t sm[];
    const int cluster = blockIdx.x / S_CL;
    next_may_start();
    if (cluster == 0) sort_cluster(p, sm);
    else fill_early(p, sm, blockIdx.x - S_CL, nullptr);
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
    int sum_ctas, slices;
    Fill fill;
};

template <typename TO, int VEC>
__device__ __forceinline__ Vec<TO, VEC>* out_vec(const SumParams& p, uint32_t row, int v)
{
    return reinterpret_cast<Vec<TO, VEC>*>((TO*)p.out + (long long)row * p.ld_out + (long long)v * VEC);
}
// x: with ACC, what the row holds
template <typename TO, int VEC, bool ACC>
__device__ __forceinline__ void write_row(const SumParams& p, uint32_t row, int v, const float (&a)[VEC], Vec<TO, VEC> x)
{
    if (ACC) {
#pragma unroll
        for (int q = 0; q < VEC; q++) x.v[q] = from_f<TO>(fmaf(p.scale, a[q], to_f(x.v[q])));
    } else
#pragma unroll
        for (int q = 0; q < VEC; q++) x.v[q] = from_f<TO>(p.scale * a[q]);
    *out_vec<TO, VEC>(p, row, v) = x;
}

template <int VEC>
__device__ __forceinline__ void store_part(float* part, const float (&a)[VEC])
{
    Vec<float, VEC> x;
#pragma unroll
    for (int q = 0; q < VEC; q++) x.v[q] = a[q];
    *reinterpret_cast<Vec<float, VEC>*>(part) = x;
}

// a warp per chunk and 32 vectors of the width; four rows' loads in flight
template <typename TI, typename TO, int VEC, bool ACC>
__global__ void __launch_bounds__(128) sum_chunks_kernel(const SumParams p)
{
    wait_for_previous();
    next_may_start();
    if (!ACC && blockIdx.x >= p.sum_ctas) {
        const int f = blockIdx.x - p.sum_ctas;
        fill_late(p.fill, p.key, p.n, f / p.fill.parts, f % p.fill.parts);
        return;
    }
    const int lane = threadIdx.x, ch = blockIdx.x / p.slices * 4 + threadIdx.y, v = blockIdx.x % p.slices * 32 + lane, nv = p.D / VEC;
    if (ch >= p.nchunks) return;
    const int c0 = ch * p.chunk, c1 = min(p.n, c0 + p.chunk);
    // keys and positions of up to 32 places, a lane each, and the keys beside the chunk: one round of loads
    uint32_t kk = c0 + lane < c1 ? p.key[c0 + lane] : (uint32_t)p.V, pp = c0 + lane < c1 ? p.pos[c0 + lane] : 0;
    const uint32_t before = c0 > 0 ? p.key[c0 - 1] : (uint32_t)p.V, after = c1 < p.n ? p.key[c1] : (uint32_t)p.V;
    uint32_t cur = __shfl_sync(0xffffffffu, kk, 0);
    if (cur >= (uint32_t)p.V) return;  // from here on nothing takes a gradient
    const bool on = v < nv;
    const bool open = before == cur;  // the first row was begun in an earlier chunk
    bool first = true;
    float a[VEC];
#pragma unroll
    for (int q = 0; q < VEC; q++) a[q] = 0.f;
    float* part = p.part + (long long)ch * 2 * p.D + (long long)v * VEC;
    const TI* d = (const TI*)p.d + (long long)v * VEC;
    for (int g = c0; g < c1; g += 32) {
        if (g > c0) kk = g + lane < c1 ? p.key[g + lane] : (uint32_t)p.V, pp = g + lane < c1 ? p.pos[g + lane] : 0;
        const int m = min(32, c1 - g);
        for (int i = 0; i < m; i += 4) {
            Vec<TI, VEC> x[4];
            Vec<TO, VEC> old[4];  // ACC: the row that ends at this place, if one does
            uint32_t k[4];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                k[q] = __shfl_sync(0xffffffffu, kk, i + q);
                const uint32_t row = __shfl_sync(0xffffffffu, pp, i + q);
                if (on && k[q] < (uint32_t)p.V) x[q] = *reinterpret_cast<const Vec<TI, VEC>*>(d + (long long)row * p.ld_d);
            }
            if (ACC) {
                uint32_t k0 = cur;  // the row before each place: written when the place's key differs
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    if (on && k[q] != k0) old[q] = *out_vec<TO, VEC>(p, k0, v);
                    k0 = k[q];
                    if (k0 >= (uint32_t)p.V) break;
                }
            }
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (i + q >= m) break;
                if (k[q] != cur) {
                    if (on) {
                        if (first && open) store_part<VEC>(part, a);
                        else write_row<TO, VEC, ACC>(p, cur, v, a, old[q]);
                    }
                    first = false;
                    cur = k[q];
                    if (cur >= (uint32_t)p.V) return;
#pragma unroll
                    for (int e = 0; e < VEC; e++) a[e] = 0.f;
                }
#pragma unroll
                for (int e = 0; e < VEC; e++) a[e] += to_f(x[q].v[e]);
            }
        }
    }
    if (!on) return;
    if (first && open) store_part<VEC>(part, a);  // the chunk is the middle or the end of a row begun earlier
    else if (after == cur) store_part<VEC>(part + p.D, a);
    else {
        Vec<TO, VEC> x;
        if (ACC) x = *out_vec<TO, VEC>(p, cur, v);
        write_row<TO, VEC, ACC>(p, cur, v, a, x);
    }
}

// sum of chunks q0 .. q1 - 1 of a row whose first chunk is `part`'s: that chunk's sum lies in its second place, the others' in their first
template <int VEC>
__device__ __forceinline__ void add_parts(float (&a)[VEC], const float* part, int q0, int q1, int D)
{
#pragma unroll 4
    for (int q = q0; q < q1; q++) {
        const Vec<float, VEC> x = *reinterpret_cast<const Vec<float, VEC>*>(part + (long long)q * 2 * D + (q == 0 ? D : 0));
#pragma unroll
        for (int i = 0; i < VEC; i++) a[i] += x.v[i];
    }
}

// Rows that go on over chunks.  A CTA looks at 32 chunks; a warp joins a row of up to SHORT chunks, the whole CTA (eight stretches,
// added in order) a longer one.
template <typename TO, int VEC, bool ACC>
__global__ void __launch_bounds__(256) join_chunks_kernel(const SumParams p)
{
    constexpr int SHORT = 8;
    __shared__ float stretch[8][32][VEC + 1];
    __shared__ int ends[32];  // the last chunk of a long row that begins in chunk i, or -1
    const int lane = threadIdx.x, warp = threadIdx.y, v = blockIdx.y * 32 + lane, nv = p.D / VEC, base = blockIdx.x * 32;
    wait_for_previous();
    // those whose last row goes on into the next chunk and was not begun in an earlier one
    const int mine = base + lane, c0 = mine * p.chunk, c1 = c0 + p.chunk;
    uint32_t k1 = (uint32_t)p.V;
    bool b = mine < p.nchunks - 1;
    if (b) {
        const uint32_t at = p.key[c0], before = c0 > 0 ? p.key[c0 - 1] : (uint32_t)p.V, after = p.key[c1];
        k1 = p.key[c1 - 1];
        b = k1 < (uint32_t)p.V && after == k1 && !(at == k1 && before == k1);
    }
    const uint32_t begins = __ballot_sync(0xffffffffu, b);
    if (warp == 0) ends[lane] = -1;
    __syncthreads();
    int nth = 0;
    for (uint32_t rest = begins; rest; rest &= rest - 1, nth++) {
        if ((nth & 7) != warp) continue;
        const int i = __ffs(rest) - 1, ch = base + i;
        const uint32_t k = __shfl_sync(0xffffffffu, k1, i);
        int last = ch + 1;  // the last chunk that begins with it
        while (true) {
            const bool same = last + lane < p.nchunks && p.key[(long long)(last + lane) * p.chunk] == k;
            const uint32_t no = ~__ballot_sync(0xffffffffu, same);
            if (no) {
                last += __ffs(no) - 2;
                break;
            }
            last += 32;
        }
        if (last - ch >= SHORT) {
            if (lane == 0) ends[i] = last;
        } else if (v < nv) {
            float a[VEC];
#pragma unroll
            for (int q = 0; q < VEC; q++) a[q] = 0.f;
            add_parts<VEC>(a, p.part + (long long)ch * 2 * p.D + (long long)v * VEC, 0, last - ch + 1, p.D);
            Vec<TO, VEC> x;
            if (ACC) x = *out_vec<TO, VEC>(p, k, v);
            write_row<TO, VEC, ACC>(p, k, v, a, x);
        }
    }
    __syncthreads();
    for (uint32_t rest = begins; rest; rest &= rest - 1) {
        const int i = __ffs(rest) - 1, ch = base + i, last = ends[i];
        if (last < 0) continue;  // uniform
        const int count = last - ch + 1, each = (count + 7) / 8, q0 = min(count, warp * each);
        float a[VEC];
#pragma unroll
        for (int q = 0; q < VEC; q++) a[q] = 0.f;
        if (v < nv) add_parts<VEC>(a, p.part + (long long)ch * 2 * p.D + (long long)v * VEC, q0, min(count, q0 + each), p.D);
#pragma unroll
        for (int q = 0; q < VEC; q++) stretch[warp][lane][q] = a[q];
        __syncthreads();
        if (warp == 0 && v < nv) {
#pragma unroll
            for (int w = 1; w < 8; w++)
#pragma unroll
                for (int q = 0; q < VEC; q++) a[q] += stretch[w][lane][q];
            const uint32_t k = p.key[(long long)(ch + 1) * p.chunk];
            Vec<TO, VEC> x;
            if (ACC) x = *out_vec<TO, VEC>(p, k, v);
            write_row<TO, VEC, ACC>(p, k, v, a, x);
        }
        __syncthreads();
    }
}

constexpr long long N_MAX = 1LL << 30;  // positions of a gradient call
constexpr int D_MAX = 1 << 20;

// Positions of a chunk, a multiple of 4: 8 at least, and so many that about 8192 warps (a chunk times 32 vectors of the width,
// eight elements each) share the sums, 1024 chunks at least.
int chunk_of(long long n, int D)
{
    const int slices = (D + 255) / 256, target = slices >= 8 ? 1024 : 8192 / slices;
    return n <= 8LL * target ? 8 : (int)(((n + target - 1) / target + 3) / 4 * 4);
}
size_t align256(size_t b) { return (b + 255) / 256 * 256; }
size_t part_bytes(long long n, int D)
{
    const int c = chunk_of(n, D);
    return align256(8 * (size_t)((n + c - 1) / c) * D);
}
constexpr int MAX_SHARES = 512;

template <typename TI, typename TO, int VEC, bool ACC>
int sum_launch(SumParams p, cudaStream_t st)
{
    const unsigned slices = (p.D / VEC + 31) / 32;
    p.slices = (int)slices;
    p.sum_ctas = (p.nchunks + 3) / 4 * p.slices;
    const cudaError_t e = launch_next(sum_chunks_kernel<TI, TO, VEC, ACC>, p.sum_ctas + p.fill.shares * p.fill.parts, dim3(32, 4), 0, st, p);
    if (e != cudaSuccess || p.nchunks == 1) return (int)e;
    return (int)launch_next(join_chunks_kernel<TO, VEC, ACC>, dim3((p.nchunks + 30) / 32, slices), dim3(32, 8), 0, st, p);
}
template <typename TI, typename TO>
int sum_dispatch(const SumParams& p, cudaStream_t st)
{
    constexpr int W = 16 / sizeof(TI);
    if (p.D % W == 0 && p.ld_d % W == 0 && p.ld_out % W == 0 && (uintptr_t)p.d % 16 == 0 && (uintptr_t)p.out % 16 == 0)
        return p.accumulate ? sum_launch<TI, TO, W, true>(p, st) : sum_launch<TI, TO, W, false>(p, st);
    return p.accumulate ? sum_launch<TI, TO, 1, true>(p, st) : sum_launch<TI, TO, 1, false>(p, st);
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
    return 4 * align256(4 * (size_t)n) + part_bytes(n, D) + 4 * MAX_SHARES;
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
    const size_t a = align256(4 * (size_t)n), parts = n > 0 ? part_bytes(n, D) : 0;
    for (int i = 0; i < 2; i++) s.key[i] = (uint32_t*)(ws + 2 * i * a), s.pos[i] = (uint32_t*)(ws + (2 * i + 1) * a);
    static std::atomic<int> clusters[64], sms[64];  // clusters of the sort kernel that a device holds at once
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
    int nc = clusters[dev].load(std::memory_order_acquire);
    cudaError_t e;
    if (nc == 0) {
        e = cudaFuncSetAttribute(sort_fill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SORT_SMEM);
        if (e != cudaSuccess) return (int)e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(S_CL), cfg.blockDim = dim3(S_THREADS), cfg.dynamicSmemBytes = SORT_SMEM;
        if ((e = cudaOccupancyMaxActiveClusters(&nc, sort_fill_kernel, &cfg)) != cudaSuccess) return (int)e;
        int m = 0;
        if ((e = cudaDeviceGetAttribute(&m, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return (int)e;
        sms[dev].store(m, std::memory_order_relaxed);
        if (nc < 2) nc = 2;
        clusters[dev].store(nc, std::memory_order_release);
    }
    const bool rank = n <= RANK_MAX;
    const int m = sms[dev].load(std::memory_order_relaxed);
    Fill& fl = s.fill;
    fl.out = (uint8_t*)out, fl.ld_bytes = ld_out * eo, fl.row_bytes = (long long)D * eo, fl.V = V;
    fl.shares = accumulate ? 0 : rank ? 2 * m : (nc - 1) * S_CL;
    if (fl.shares > MAX_SHARES) fl.shares = MAX_SHARES;
    fl.start = n > 0 ? (int*)(ws + 4 * a + parts) : nullptr;
    // Early: what can be written while the digits are sorted, 15 us and 0.5 us a thousand positions, at 6 TB/s.  Beside ranks nothing,
    // those are counted by all CTAs first; without positions everything, there are no sums to hide the rest behind.  Late: about 48 KB
    // a CTA.  To 128256 x 4096 bf16: 220 us from 16384 positions, 253 with all rows early; 177 and 204 from 4096.
    const double early = (15.0 + n / 2000.0) * 6e6 / (double)fl.row_bytes;
    fl.early = n == 0 ? V : rank || !fl.shares ? 0 : (long long)(early / fl.shares) + 1;
    const long long late = fl.shares ? (V + (long long)fl.shares - 1) / fl.shares - fl.early : 0;
    fl.parts = late > 0 ? (int)std::min(((double)late * fl.row_bytes + LATE_BYTES - 1) / LATE_BYTES, 1024.0) : 0;
    if (rank) {
        s.passes = 1;
        const int need = (int)((n + S_WARPS - 1) / S_WARPS);
        rank_fill_kernel<<<accumulate ? (need < 2 * m ? need : 2 * m) : fl.shares, S_THREADS, 0, st>>>(s);
    } else
        sort_fill_kernel<<<S_CL + fl.shares, S_THREADS, SORT_SMEM, st>>>(s);
    e = cudaGetLastError();
    if (e != cudaSuccess || n == 0) return (int)e;
    SumParams p{};
    const int b = sorted_buffer(s.passes);
    p.key = s.key[b], p.pos = s.pos[b], p.d = dout, p.ld_d = ld_d, p.out = out, p.ld_out = ld_out;
    p.part = (float*)(ws + 4 * a);
    p.n = (int)n, p.V = V, p.D = D, p.chunk = chunk_of(n, D), p.accumulate = accumulate != 0, p.scale = scale, p.fill = s.fill;
    p.nchunks = (int)((n + p.chunk - 1) / p.chunk);
    if (dtype == DT_F32) return sum_type<float>(p, out_dtype, st);
    if (dtype == DT_BF16) return sum_type<__nv_bfloat16>(p, out_dtype, st);
    return sum_type<__half>(p, out_dtype, st);
}
