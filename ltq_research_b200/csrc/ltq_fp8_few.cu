// y = x W^T for few rows x (at most 32) and a block-scaled e4m3 weight, in one launch (B200, sm_100a).
//
// The weight is read once and is all of the traffic, so the kernel is a stream of weight blocks with everything else kept out
// of its way.  The roles of the operands are exchanged: 128 rows of the weight are the M side of tcgen05.mma and the rows of x,
// padded to 16 or 32, its N side, so a block of 128 x 128 weights costs a fraction of its load's time.  A CTA quantizes its
// share of x once, into shared memory in the layout the MMAs read, while the first weight blocks are on their way.
//
//   warp 0        TMA producer: weight blocks [128 rows][128 of K] into a ring
//   warp 1        MMA issuer: four tcgen05.mma a block into tensor-memory buffers of two blocks
//   warps 2 .. 5  epilogue: lane = weight row; each block's sums times sw sx added to fp32 registers
//   warps 1 ..    first quantize x
//
// Bound by the weight's bytes where it is large: 1 x 128256 x 2048 48 us, 5.5 TB/s; 24 rows 51 us, 5.2 TB/s: all CTAs read x
// from L2 at the start, and the first MMAs wait for it longer than the ring of weight blocks lasts.  A small
// weight is bound by the chain launch, first loads, MMAs, epilogue: 1 x 8192 x 2048 12 us, where the bytes alone would take 3.
//
// Narrow weights are cut along K over a cluster of 2, 4 or 8 CTAs; each hands the others their columns of its sums through
// distributed shared memory and adds its own in the order of K.  Wide ones: one CTA an SM walks the row tiles.
// Every mbarrier wait is bounded, as in ltq_fp8_gemm.cu.
#include "ltq_b200.h"
#include "fp8_tc.cuh"

namespace {

constexpr int F_ROWS = 32;
constexpr int F_THREADS = 384, F_WARPS = F_THREADS / 32;
constexpr int F_STAGES = 12, F_MIN_STAGES = 4, F_STAGE = 128 * QB;  // weight blocks of 16 KB on their way
constexpr int F_SMEM = 226 * 1024;
constexpr uint32_t F_WAIT = 1u << 24;

struct FewArgs {
    const void* x;
    long long ldx;
    const float* sb;
    long long ld_sb;
    void* y;
    long long ldy;
    int* err;
    int M, N, K, nkb, tiles, splits, cap, stages, out_dt, aligned;
};

template <int BN>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t acc)
{
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc_f8(128, BN)), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void arrive(uint64_t* b)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(b)) : "memory");
}

// where `p` of this CTA's shared memory lies in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t map_other(const void* p, uint32_t rank)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}

template <typename T, int BN>
__global__ void __launch_bounds__(F_THREADS, BN == 16 ? 2 : 1) gemm_few_kernel(const __grid_constant__ CUtensorMap tmW, const FewArgs g)
{
    constexpr bool DUO = BN > 16;             // pairs of CTAs, each of which quantizes half of x for both (K is never cut then)
    constexpr int PER = 2;                    // blocks whose sums are handed over together
    constexpr int F_BUFS = BN == 16 ? 8 : 4;  // tensor-memory buffers
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* ring = smem;
    uint8_t* xq = ring + g.stages * F_STAGE;                            // [block][BN rows][128], 128-byte swizzle
    float* xs = reinterpret_cast<float*>(xq + g.cap * BN * QB);         // [block][BN]
    float* joined = xs + g.cap * BN;                                    // [split][column of this CTA][128]
    uint64_t* full = reinterpret_cast<uint64_t*>(joined + (g.splits > 1 ? BN * 128 : 0));
    uint64_t* empty = full + F_STAGES;
    uint64_t* accfull = empty + F_STAGES;
    uint64_t* accempty = accfull + F_BUFS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accempty + F_BUFS);
    constexpr int COLS = F_BUFS * PER * BN;  // 256 columns

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = g.splits > 1 ? (int)cluster_rank() : 0;
    const int worker = blockIdx.x / g.splits, workers = gridDim.x / g.splits;
    const int kb0 = (int)((long long)g.nkb * split / g.splits), kb1 = (int)((long long)g.nkb * (split + 1) / g.splits);
    const int nb = kb1 - kb0;

    // Four rows of x in two blocks of K, for one warp: eight columns a lane and row
    constexpr int STEP = F_WARPS - 1;
    const int quads = (g.M + 3) / 4;
    Raw8<T> next[4] = {};
    auto load_quad = [&](int u) {
        const int pair = u / quads, m0 = 4 * (u - pair * quads), c = (kb0 + 2 * pair) * QB + 8 * lane;
        const T* row = (const T*)g.x + m0 * g.ldx;
#pragma unroll
        for (int q = 0; q < 4; q++, row += g.ldx)
            if (m0 + q < g.M) load8(row, c, g.K, g.aligned, next[q]);
    };
    const int duo_rank = DUO ? (int)cluster_rank() : 0, first = 2 * (warp - 1) + duo_rank;
    if (DUO && warp >= 1 && first < (nb + 1) / 2 * quads) load_quad(first);
    if (tid == 0) {
        for (int i = 0; i < F_STAGES; i++) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        for (int i = 0; i < F_BUFS; i++) mbar_init(&accfull[i], 1), mbar_init(&accempty[i], 4);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)), "r"(COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    if (g.splits > 1) cluster_arrive_relaxed();  // paired with the wait before the columns are handed over
    if (DUO) cluster_arrive_relaxed();           // paired with the wait before x is written to both CTAs
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool waited = false;  // for the cluster's start

    if (warp == 0) {
        if (DUO) cluster_wait(), cluster_arrive_relaxed();  // for the barrier behind x, to which this warp adds nothing
        int st = 0;
        uint32_t parity = 1;  // the first wait for each buffer passes at once
        int issued = 0;
        bool ok = true;
        for (int tile = worker; tile < g.tiles && ok; tile += workers)
            for (int k = kb0; k < kb1; k++) {
                ok = mbar_wait_warp(&empty[st], parity, g.err, F_WAIT);
                if (!ok) break;
                if (elect_one()) {
                    mbar_expect_tx(&full[st], F_STAGE);
                    tma_load_2d(ring + st * F_STAGE, &tmW, k * QB, tile * 128, &full[st]);
                }
                __syncwarp();
                issued++;
                if (++st == g.stages) st = 0, parity ^= 1;
            }
        // none of this CTA's copies is in flight when it leaves: a buffer is free again once they have landed and been read
        for (int j = issued > g.stages ? issued - g.stages : 0; j < issued; j++)
            mbar_wait_warp(&empty[j % g.stages], (j / g.stages) & 1, g.err, F_WAIT);
        __syncwarp();
        if (DUO) cluster_wait();
    } else {
        const int pairs = (nb + 1) / 2, piece = lane & 15;
        // rows M .. BN - 1 are zeros
        for (int i = tid - 32; i < nb * BN * (QB / 16); i += F_THREADS - 32)
            if (i / (QB / 16) % BN >= g.M) reinterpret_cast<uint4*>(xq)[i] = make_uint4(0, 0, 0, 0);
        for (int i = tid - 32; i < nb * BN; i += F_THREADS - 32)
            if (i % BN >= g.M) xs[i] = 0.f;
        if constexpr (!DUO) {
            // a row at a time, four in flight: little else fits the registers of two CTAs an SM
            constexpr int AHEAD = 4;
            const T* x = (const T*)g.x;
            for (int u0 = warp - 1; u0 < pairs * g.M; u0 += AHEAD * STEP) {
                Raw8<T> raw[AHEAD];
#pragma unroll
                for (int q = 0; q < AHEAD; q++) {
                    const int u = u0 + q * STEP, m = u % g.M, c = (kb0 + 2 * (u / g.M)) * QB + 8 * lane;
                    if (u < pairs * g.M) load8(x + m * g.ldx, c, g.K, g.aligned, raw[q]);
                }
#pragma unroll
                for (int q = 0; q < AHEAD; q++) {
                    const int u = u0 + q * STEP, m = u % g.M, b = 2 * (u / g.M) + (lane >> 4);
                    if (u >= pairs * g.M) break;
                    float v[8];
                    unpack8(raw[q], v);
                    const float scale = block_scale(half_warp_max(amax8(raw[q])));
                    const uint2 w = quant8(v, scale, __frcp_rn(scale));
                    if (b < nb) {  // eight bytes; 16-byte chunks are swizzled by the row
                        *reinterpret_cast<uint2*>(xq + b * BN * QB + m * QB + (((piece >> 1) ^ (m & 7)) << 4) + (piece & 1) * 8) = w;
                        if (piece == 0) xs[b * BN + m] = scale;
                    }
                }
            }
        } else {
            // four rows at a time, the next four in flight, half of them each CTA of a pair: 32 x 128256 x 4096 100 us, 106 if each does
            // all, 117 also in the form above; two or three groups in flight are no faster
            cluster_wait();
            const uint32_t xq_other = map_other(xq, duo_rank ^ 1), xs_other = map_other(xs, duo_rank ^ 1);
            for (int u = first; u < pairs * quads; u += 2 * STEP) {
                const int pair = u / quads, m0 = 4 * (u - pair * quads), b = 2 * pair + (lane >> 4);
                Raw8<T> raw[4];
                float scale[4], rec[4];
#pragma unroll
                for (int q = 0; q < 4; q++) raw[q] = next[q];
                if (u + 2 * STEP < pairs * quads) load_quad(u + 2 * STEP);
                scales4(raw, lane, scale, rec);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int m = m0 + q;
                    float v[8];
                    unpack8(raw[q], v);
                    const uint2 w = quant8(v, scale[q], rec[q]);
                    if (m < g.M && b < nb) {
                        const int at = b * BN * QB + m * QB + (((piece >> 1) ^ (m & 7)) << 4) + (piece & 1) * 8;
                        *reinterpret_cast<uint2*>(xq + at) = w;
                        asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};\n" ::"r"(xq_other + at), "r"(w.x), "r"(w.y) : "memory");
                        if (piece == 0) {
                            xs[b * BN + m] = scale[q];
                            asm volatile("st.shared::cluster.f32 [%0], %1;\n" ::"r"(xs_other + 4 * (b * BN + m)), "f"(scale[q]) : "memory");
                        }
                    }
                }
            }
        }
        asm volatile("fence.proxy.async;\n" ::: "memory");  // written here, read by the MMAs
        __syncwarp();
        if (DUO) {
            cluster_arrive();
            cluster_wait();
            asm volatile("fence.proxy.async;\n" ::: "memory");
        } else
            asm volatile("bar.sync 1, %0;\n" ::"n"(F_THREADS - 32) : "memory");

        if (warp == 1) {
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint64_t wdesc = sw128_kmajor_desc(smem_u32(ring)), xdesc = sw128_kmajor_desc(smem_u32(xq));
            int st = 0, buf = 0;
            uint32_t full_parity = 0, free_parity = 1;
            bool ok = true;
            for (int tile = worker; tile < g.tiles && ok; tile += workers)
                for (int k = 0; k < nb; k++) {
                    ok = mbar_wait_warp(&full[st], full_parity, g.err, F_WAIT) &&
                         (k % PER || mbar_wait_warp(&accempty[buf], free_parity, g.err, F_WAIT));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t a = wdesc + (uint32_t)(st * (F_STAGE >> 4)), b = xdesc + (uint32_t)(k * (BN * QB >> 4));
                    const bool last = k % PER == PER - 1 || k + 1 == nb;  // the buffer is complete
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < 4; kk++) mma_f8<BN>(tm + (PER * buf + k % PER) * BN, a + 2 * kk, b + 2 * kk, kk != 0);
                        if (last) umma_commit(&accfull[buf]);
                        umma_commit(&empty[st]);
                    }
                    __syncwarp();
                    if (++st == g.stages) st = 0, full_parity ^= 1;
                    if (last && ++buf == F_BUFS) buf = 0, free_parity ^= 1;
                }
        } else if (warp < 6) {
            const int quarter = warp & 3, row = 32 * quarter + lane;
            const uint32_t tl = tmem + ((uint32_t)(32 * quarter) << 16);
            int buf = 0;
            uint32_t parity = 0;
            bool ok = true;
            for (int tile = worker; tile < g.tiles && ok; tile += workers) {
                float acc[BN];
#pragma unroll
                for (int j = 0; j < BN; j++) acc[j] = 0.f;
                const float* sb = g.sb + (long long)tile * g.ld_sb + kb0;
                float sw32 = 0.f;
                for (int k = 0; k < nb; k += PER) {
                    if ((k & 31) == 0) sw32 = k + lane < nb ? sb[k + lane] : 0.f;  // a lane each for 32 blocks
                    float sw[PER];
#pragma unroll
                    for (int h = 0; h < PER; h++) sw[h] = __shfl_sync(0xffffffffu, sw32, (k + h) & 31);
                    ok = mbar_wait_warp(&accfull[buf], parity, g.err, F_WAIT);
                    if (!ok) break;
                    tc_fence_after();
                    uint32_t part[PER * BN];  // behind a single last block the second half is not used
#pragma unroll
                    for (int c = 0; c < PER * BN; c += 16) tmem_ld16_start(tl + buf * PER * BN + c, part + c);
                    tmem_ld_done(part);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive(&accempty[buf]);
                    if (++buf == F_BUFS) buf = 0, parity ^= 1;
#pragma unroll
                    for (int h = 0; h < PER; h++) {
                        if (k + h >= nb) break;
                        const float4* s4 = reinterpret_cast<const float4*>(xs + (k + h) * BN);
#pragma unroll
                        for (int j = 0; j < BN; j += 4) {
                            const float4 s = s4[j / 4];
                            const uint32_t* q = part + h * BN + j;
                            acc[j] = fmaf(__uint_as_float(q[0]), sw[h] * s.x, acc[j]);
                            acc[j + 1] = fmaf(__uint_as_float(q[1]), sw[h] * s.y, acc[j + 1]);
                            acc[j + 2] = fmaf(__uint_as_float(q[2]), sw[h] * s.z, acc[j + 2]);
                            acc[j + 3] = fmaf(__uint_as_float(q[3]), sw[h] * s.w, acc[j + 3]);
                        }
                    }
                }
                if (!ok) break;
                const int n = tile * 128 + row;
                if (g.splits == 1) {
                    if (n < g.N) {
#pragma unroll
                        for (int j = 0; j < BN; j++) {
                            if (j >= g.M) break;
                            store_as(g.y, g.out_dt, j * g.ldy + n, acc[j]);
                        }
                    }
                } else {  // one tile: every CTA of the cluster has started, its columns of the sums go to each
                    __syncwarp();
                    cluster_wait();
                    waited = true;
                    const int own = BN / g.splits;
#pragma unroll
                    for (int j = 0; j < BN; j++)
                        st_cluster_u32(&joined[(split * own + j % own) * 128 + row], j / own, __float_as_uint(acc[j]));
                }
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    if (g.splits > 1 && !waited) cluster_wait();
    __syncthreads();
    if (g.splits > 1) {
        cluster_arrive();
        cluster_wait();
        if (warp >= 2 && warp < 6) {
            const int row = 32 * (warp & 3) + lane, n = worker * 128 + row, own = BN / g.splits;
            for (int c = 0; c < own; c++) {
                const int m = split * own + c;
                if (m >= g.M || n >= g.N) break;
                float v = 0.f;
                for (int q = 0; q < g.splits; q++) v += joined[(q * own + c) * 128 + row];
                store_as(g.y, g.out_dt, m * g.ldy + n, v);
            }
        }
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(COLS) : "memory");
    }
}

struct FewPlan {
    int bn, nkb, tiles, splits, cap, stages, smem, grid;
};
// The quantized x of a CTA's share of K stays in its shared memory beside at least four weight blocks.  K is cut (2, 4 or 8 ways)
// where that takes it, and further while the CTAs all run at once (two an SM of at most 16 rows) with four blocks of K or more
// each.  False, for the other kernels, where more CTAs than that would each have to quantize their x, and for more than 32 rows:
// at 64 (one block a buffer, 88 us for 128256 x 2048) the 256-row tiles behind a separate quantization are faster (70 us a call).
bool plan_few(int M, int N, int K, int sms, FewPlan& p)
{
    if (M < 1 || M > F_ROWS || N < 1 || K < 1 || sms < 2) return false;
    p.bn = M <= 16 ? 16 : 32;
    p.nkb = (int)(((long long)K + QB - 1) / QB);
    p.tiles = (int)(((long long)N + 127) / 128);
    const int block = p.bn * (QB + 4), hand = p.bn * 512, fixed = 512 + 1024;  // bytes: x and its scales of a block; joined columns
    auto share = [&](int splits) { return (p.nkb + splits - 1) / splits; };
    auto need = [&](int splits, int stages) { return stages * F_STAGE + share(splits) * block + (splits > 1 ? hand : 0) + fixed; };
    if (p.bn > 16 && p.tiles < sms) return false;  // quantizing so much in every CTA pays where each then reads a row tile or more
    p.splits = 1;
    while (p.splits < 8 && need(p.splits, F_MIN_STAGES) > F_SMEM) p.splits *= 2;
    if (need(p.splits, F_MIN_STAGES) > F_SMEM || (p.splits > 1 && (long long)p.tiles * p.splits > sms)) return false;
    while (p.splits < 8 && p.nkb >= 8 * p.splits && (long long)p.tiles * p.splits * 2 <= sms) p.splits *= 2;
    int budget = F_SMEM;
    if (p.bn == 16 && p.splits < 8 && p.nkb >= 8 * p.splits && (long long)p.tiles * p.splits * 2 <= 2 * sms &&
        need(p.splits * 2, F_MIN_STAGES) <= F_SMEM / 2)
        p.splits *= 2, budget = F_SMEM / 2;
    p.cap = share(p.splits);
    const int blocks = p.splits > 1 || p.tiles <= sms ? p.cap : F_STAGES;  // that a CTA has to load
    p.stages = F_MIN_STAGES;
    while (p.stages < F_STAGES && p.stages < blocks && need(p.splits, p.stages + 1) <= budget) p.stages++;
    p.smem = need(p.splits, p.stages);
    p.grid = (p.splits > 1 || p.tiles < sms ? p.tiles : sms) * p.splits;
    if (p.bn > 16) p.grid &= ~1;
    return true;
}

template <typename T, int BN>
int run_few(const CUtensorMap& tw, const FewArgs& g, const FewPlan& p, cudaStream_t st)
{
    static std::atomic<int> ready[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
    auto k = gemm_few_kernel<T, BN>;
    if (!ready[dev].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, F_SMEM);
        if (e != cudaSuccess) return (int)e;
        ready[dev].store(1, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.grid);
    cfg.blockDim = dim3(F_THREADS);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {BN > 16 ? 2u : (unsigned)p.splits, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = BN > 16 || p.splits > 1 ? 1 : 0;
    return (int)cudaLaunchKernelEx(&cfg, k, tw, g);
}
template <typename T>
int few_type(const CUtensorMap& tw, const FewArgs& g, const FewPlan& p, cudaStream_t st)
{
    return p.bn == 16 ? run_few<T, 16>(tw, g, p, st) : run_few<T, 32>(tw, g, p, st);
}

}  // namespace

extern "C" int ltq_fp8_few_supported(int M, int N, int K)
{
    FewPlan p;
    return plan_few(M, N, K, sm_count(), p) ? 1 : 0;
}

extern "C" int ltq_fp8_few(const void* x, int dtype, long long ldx, const uint8_t* W, long long ldw, const float* sw, long long ld_sw,
                           void* y, int out_dtype, long long ldy, int M, int N, int K, int* err, void* stream)
{
    const int es = dt_bytes(dtype), eo = dt_bytes(out_dtype);
    if (!es || !eo || M < 0 || N < 0 || K < 1 || ldx < K || ldy < N || ld_sw < (K + QB - 1) / QB) return -1;
    if (M == 0 || N == 0) return 0;
    if (!x || (uintptr_t)x % es || bad_operand(W, ldw, K) || !sw || (uintptr_t)sw % 4 || !y || (uintptr_t)y % eo) return -1;
    FewPlan p;
    if (!plan_few(M, N, K, sm_count(), p)) return -1;
    CUtensorMap tw;
    if (!make_map_8(&tw, W, N, K, ldw, 128)) return -1;
    const int aligned = (uintptr_t)x % 16 == 0 && ldx * es % 16 == 0;
    const FewArgs g{x, ldx, sw, ld_sw, y, ldy, err, M, N, K, p.nkb, p.tiles, p.splits, p.cap, p.stages, out_dtype, aligned};
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F32) return few_type<float>(tw, g, p, st);
    if (dtype == DT_BF16) return few_type<__nv_bfloat16>(tw, g, p, st);
    return few_type<__half>(tw, g, p, st);
}
