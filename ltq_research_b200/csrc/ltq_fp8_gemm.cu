// Block-scaled products of e4m3 operands on the tensor cores (B200, sm_100a): tcgen05.mma kind::f8f6f4, TMA operand loads,
// the partial sums of each block of 128 joined under their scales in registers.
//
//     C[m, n] = sum_b sa[m, b] sb[n / 128, b] P_b[m, n],   P_b = sum over block b of A[m, k] B[n, k]
//
// The scales change from block to block of K, so tensor memory holds only the sum P_b of one block and the epilogue warps
// read it back, multiply and add it to fp32 registers while the next block's product runs into the other half of tensor
// memory.  A pair of CTAs works on a 256 x 256 tile (cta_group::2: each loads 128 rows of A and 128 of B and holds 128 rows
// of the sums): per block 32 KB of operands a CTA for 2 * 128^2 * 256 operations, 64 bytes a clock of L2 reads an SM at full rate,
// where one CTA with a 128 x 256 tile would need 96.
//
//   warp 8        TMA producer, A and B blocks into a ring of W_STAGES buffers (128-byte swizzle) on both CTAs; the bytes of both
//                 are counted on the first CTA's "full" mbarrier
//   warp 9        of the first CTA: four tcgen05.mma (K 32 each) a block; tcgen05.commit frees the buffers of both CTAs and hands
//                 the sum to both CTAs' epilogue warps
//   warps 0 .. 7  epilogue: lanes' quarter w % 4 of the rows, half w / 4 of the columns, 128 sums a thread
// Warps 8 and 9 run whole and one elected lane issues: from a single-lane branch the operands of the MMAs leave the uniform
// registers, which cost 800 cycles a block.
//
// What bounds it: a block's MMAs take 512 cycles a pair, and the chain sum complete -> read (two rounds of 64 columns, for which
// the registers beside the sums suffice) -> buffer handed back -> next MMAs about twice that, over two buffers.  8192 x 8192 x
// 4096: 267 us, 2060 TFLOP/s in a single launch (the MMAs alone, without epilogue, 160 us; a 256 x 128 tile with four buffers 290 us or
// more, for each hand-over costs the issuing warp the same).
//
// Pairs walk the tiles (rows first, so that neighbours share B in L2).  The tiles that are left after the last full round are cut
// along K into one equal share for each pair: as many slices of each tile as there are pairs for, and the rest of K of all tiles, cut
// across tiles, for the pairs that remain.  So all tiles' slices run through the same K at the same time and a block of A or B is
// read from memory once and by the other tiles from L2: 1003 x 2048 x 128256 250 us and 0.5 GB of reads, where shares that follow one
// another through the tiles took 266 us and 1.5 GB.  The parts go to a workspace and join_parts_kernel adds them in the order of K.  Every wait is bounded: when one runs out
// *err is set, the role stops and the CTAs still meet at their last barrier.
#include <algorithm>

#include "ltq_b200.h"
#include "fp8_tc.cuh"
#include "launch_next.cuh"
#include "vec_types.cuh"

namespace {

// ------------------------------------------------------------------------------------------------ cta_group::2 pieces

__device__ __forceinline__ uint32_t map_rank(const void* p, uint32_t rank)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
// Arrival on an mbarrier of either CTA.  What it guards is tensor memory, whose reads have completed (tcgen05.wait::ld) and are
// ordered by the tcgen05 fences; so it is relaxed: a cluster-wide release waits for the warp's outstanding loads and cost 2000
// cycles a block of K.
__device__ __forceinline__ void arrive_cluster(uint32_t addr)
{
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(addr) : "memory");
}
// the copy lands in this CTA's shared memory, its bytes are counted on the mbarrier at `bar` (of either CTA of the pair)
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void commit_pair(uint64_t* bar)  // arrives on both CTAs' mbarriers at this address
{
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void mma_f8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// waits for the reads issued so far; the registers pass through, so that no use of them moves above the wait
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_pin(uint32_t (&r)[32])
{
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];\n" ::"l"(map), "r"(smem_u32(src)),
                 "r"(x), "r"(y)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
}

// --------------------------------------------------------------------------------------------------- the wide kernel

constexpr int WT = 256;                                  // tile of a pair, both ways
constexpr int W_STAGES = 6;
constexpr int W_OP = 128 * QB, W_STAGE = 2 * W_OP;       // one operand's block of a CTA: 16 KB
constexpr int W_AHEAD = 8;                               // blocks whose scales are fetched together, one group ahead
constexpr int W_THREADS = 384;
// registers a thread: 168 at launch (384 x 168 = 64512 of the SM's 65536); the epilogue's eight warps take 232, the others keep 40
constexpr int W_REGS_EPILOGUE = 232, W_REGS_ROLES = 40;
static_assert(256 * W_REGS_EPILOGUE + 128 * W_REGS_ROLES <= W_THREADS * 168, "the shares fit the launch's registers");
constexpr int W_STORE = 4096;                            // staging of an epilogue warp: a 32-row box of 128 bytes
constexpr int W_SMEM = W_STAGES * W_STAGE + 8 * W_STORE + 256 + 1024;
static_assert(W_SMEM <= 232448, "shared memory of one CTA");
constexpr int PART_FLOATS = 128 * WT;                    // a CTA's rows of a partial tile

struct WideArgs {
    const float* sa;
    long long ld_sa;
    const float* sb;
    long long ld_sb;
    void* C;
    long long ldc;
    float* parts;  // [part][CTA][column / 4][row][4]
    int* err;
    int M, N, nkb, mt, whole, tma_c;  // whole: tiles done in one piece
    int cut;                          // tiles after them, of which pair g cut + r < slices cut takes blocks g slice .. of tile r;
    int slices, slice;                // the `tail` blocks behind a tile's slices, all tiles' in a row, are shared equally by the
    int tail, tailers;                // next `tailers` pairs (at least one block each)
};
// a pair's slice is part g cut + r; of the tails that of the q-th of its pairs in tile r is part slices cut + q + r (from share to share
// and tile to tile one of q and r grows, so no two are the same)
__host__ __device__ inline int part_count(int cut, int slices, int tail, int tailers)
{
    return cut * slices + (tail ? cut + tailers - 1 : 0);
}
__device__ __forceinline__ long long tail_share(const WideArgs& g, int q) { return (long long)g.cut * g.tail * q / g.tailers; }

struct Segment {
    int tile, k0, k1, part;
};
// the pieces of work of pair c of G, in order
struct Walk {
    const WideArgs& g;
    int c, pairs, t;
    bool slice;       // still to be done
    long long u, u1;  // blocks of the tails
    __device__ Walk(const WideArgs& g_, int c_, int pairs_)
        : g(g_), c(c_), pairs(pairs_), t(c_), slice(c_ < g_.slices * g_.cut), u(0), u1(0)
    {
        const int q = c - g.slices * g.cut;
        if (q >= 0 && q < g.tailers) u = tail_share(g, q), u1 = tail_share(g, q + 1);
    }
    __device__ bool next(Segment& s)
    {
        if (t < g.whole) {
            s = {t, 0, g.nkb, 0};
            t += pairs;
            return true;
        }
        if (slice) {
            const int k0 = c / g.cut * g.slice;
            s = {g.whole + c % g.cut, k0, k0 + g.slice, c};
            slice = false;
            return true;
        }
        if (u >= u1) return false;
        const int r = (int)(u / g.tail), k = (int)(u % g.tail), k0 = g.slices * g.slice + k;
        const long long left = u1 - u;
        s = {g.whole + r, k0, left < g.tail - k ? k0 + (int)left : g.nkb, c + r};
        u += s.k1 - s.k0;
        return true;
    }
};

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(W_THREADS, 1)
    gemm_wide_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmC, const WideArgs g)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* store = smem + W_STAGES * W_STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(store + 8 * W_STORE);
    uint64_t* empty = full + W_STAGES;
    uint64_t* accfull = empty + W_STAGES;
    uint64_t* accempty = accfull + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accempty + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < W_STAGES; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&accfull[i], 1);
            mbar_init(&accempty[i], 16);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 8) {
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];\n" ::"l"(&tmA) : "memory");
            asm volatile("prefetch.tensormap [%0];\n" ::"l"(&tmB) : "memory");
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    wait_for_previous();  // A and its scales are written
    next_may_start();     // the parts' join

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(W_REGS_ROLES));
        if (warp == 8) {
            Walk walk(g, pair, npairs);
            Segment s;
            int i = 0;
            bool ok = true;
            while (ok && walk.next(s)) {
                const int m0 = (s.tile % g.mt) * WT + rank * 128, n0 = (s.tile / g.mt) * WT + rank * 128;
                for (int k = s.k0; k < s.k1; k++, i++) {
                    const int st = i % W_STAGES;
                    if (i >= W_STAGES && !mbar_wait_warp(&empty[st], (i / W_STAGES - 1) & 1, g.err, WAIT_LIMIT)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bar = map_rank(&full[st], 0);
                    if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(&full[st], 2 * W_STAGE);  // both CTAs' bytes
                    tma_load_2d_pair(smem + st * W_STAGE, &tmA, k * QB, m0, bar);
                    tma_load_2d_pair(smem + st * W_STAGE + W_OP, &tmB, k * QB, n0, bar);
                    }
                    __syncwarp();
                }
            }
            // a buffer is free again once its copies have landed and been read: none is in flight when the CTA leaves
            for (int j = i > W_STAGES ? i - W_STAGES : 0; j < i; j++)
                mbar_wait_warp(&empty[j % W_STAGES], (j / W_STAGES) & 1, g.err, WAIT_LIMIT);
        }
        if (warp == 9 && rank == 0) {
            // the whole warp runs the loop and one elected lane issues: the operands then stay in uniform registers
            Walk walk(g, pair, npairs);
            Segment s;
            constexpr uint32_t ID = idesc_f8(256, WT);
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint64_t base = sw128_kmajor_desc(smem_u32(smem));
            int st = 0, buf = 0;
            uint32_t full_parity = 0, free_parity = 1;  // the first wait for either buffer passes at once
            bool ok = true;
            while (ok && walk.next(s))
                for (int k = s.k0; k < s.k1; k++) {
                    ok = mbar_wait_warp(&full[st], full_parity, g.err, WAIT_LIMIT) &&
                         mbar_wait_warp(&accempty[buf], free_parity, g.err, WAIT_LIMIT);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t a = base + (uint32_t)(st * (W_STAGE >> 4)), b = a + (W_OP >> 4);
                    const uint32_t d = tm + buf * WT;
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < 4; kk++) mma_f8_pair(d, a + 2 * kk, b + 2 * kk, ID, kk != 0);
                        commit_pair(&accfull[buf]);
                        commit_pair(&empty[st]);
                    }
                    __syncwarp();
                    if (++st == W_STAGES) st = 0, full_parity ^= 1;
                    if ((buf ^= 1) == 0) free_parity ^= 1;
                }
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(W_REGS_EPILOGUE));
        Walk walk(g, pair, npairs);
        Segment s;
        constexpr int BOX = 128 / sizeof(T);  // columns of a store box
        const int quarter = warp & 3, half = warp >> 2;
        uint8_t* box = store + warp * W_STORE;
        const uint32_t lane_base = tmem + ((uint32_t)(32 * quarter) << 16) + half * 128;
        const uint32_t free_bar[2] = {map_rank(&accempty[0], 0), map_rank(&accempty[1], 0)};
        int i = 0;
        bool ok = true;
        while (ok && walk.next(s)) {
            const int m0 = (s.tile % g.mt) * WT + rank * 128 + 32 * quarter, m = m0 + lane;
            const int n0 = (s.tile / g.mt) * WT + half * 128;
            const bool live = m < g.M && n0 < g.N;
            const float* pa = g.sa + m;
            const float* pb = g.sb + (long long)(n0 / QB) * g.ld_sb;
            float acc[128];
#pragma unroll
            for (int j = 0; j < 128; j++) acc[j] = 0.f;
            // sa of W_AHEAD blocks, and of as many more on their way: L2 answers later than several blocks take while the
            // operands stream.  sb comes for 32 blocks at a time, a lane each.  The loads go past L1, whose fills would take
            // shared-memory cycles from the MMAs' operands (23 us of 8192 x 8192 x 4096).
            float sa[W_AHEAD], na[W_AHEAD], sb32 = 0.f, nb32;
            auto fetch = [&](int k) {
#pragma unroll
                for (int j = 0; j < W_AHEAD; j++) na[j] = live && k + j < s.k1 ? __ldcg(pa + (k + j) * g.ld_sa) : 0.f;
            };
            auto fetch_b = [&](int k) { return n0 < g.N && k + lane < s.k1 ? __ldcg(pb + k + lane) : 0.f; };
            fetch(s.k0);
            nb32 = fetch_b(s.k0);
            for (int kq = s.k0; kq < s.k1 && ok; kq += W_AHEAD) {
                const int at = (kq - s.k0) & 31;
                if (at == 0) sb32 = nb32, nb32 = fetch_b(kq + 32);
#pragma unroll
                for (int j = 0; j < W_AHEAD; j++) sa[j] = na[j];
                fetch(kq + W_AHEAD);
#pragma unroll
                for (int kj = 0; kj < W_AHEAD; kj++) {
                    if (kq + kj >= s.k1) break;
                    const float sc = sa[kj] * __shfl_sync(0xffffffffu, sb32, at + kj);
                    const int buf = i & 1;
                    ok = mbar_wait_warp(&accfull[buf], (i / 2) & 1, g.err, WAIT_LIMIT);
                    i++;
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t t = lane_base + buf * WT;
                    uint32_t r[2][32];
                    tmem_ld32_issue(t, r[0]);
                    tmem_ld32_issue(t + 32, r[1]);
                    tmem_ld_wait(r[0]);
                    tmem_ld_pin(r[1]);
#pragma unroll
                    for (int j = 0; j < 32; j++) acc[j] = fmaf(__uint_as_float(r[0][j]), sc, acc[j]);
                    tmem_ld32_issue(t + 64, r[0]);
#pragma unroll
                    for (int j = 0; j < 32; j++) acc[32 + j] = fmaf(__uint_as_float(r[1][j]), sc, acc[32 + j]);
                    tmem_ld32_issue(t + 96, r[1]);
                    tmem_ld_wait(r[0]);
                    tmem_ld_pin(r[1]);
                    tc_fence_before();  // the sums are in registers: the buffer goes back to the MMAs
                    __syncwarp();
                    if (lane == 0) arrive_cluster(free_bar[buf]);
#pragma unroll
                    for (int j = 0; j < 32; j++) acc[64 + j] = fmaf(__uint_as_float(r[0][j]), sc, acc[64 + j]);
#pragma unroll
                    for (int j = 0; j < 32; j++) acc[96 + j] = fmaf(__uint_as_float(r[1][j]), sc, acc[96 + j]);
                }
            }
            if (!ok) break;
            if (s.k0 != 0 || s.k1 != g.nkb) {  // a part of the tile's sum
                float* part = g.parts + ((long long)s.part * 2 + rank) * PART_FLOATS;
#pragma unroll
                for (int c = 0; c < 32; c++)
                    *reinterpret_cast<float4*>(part + ((half * 32 + c) * 128 + 32 * quarter + lane) * 4) =
                        make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
                continue;
            }
#pragma unroll
            for (int c = 0; c < 128; c += BOX) {
                if (n0 + c >= g.N || m0 >= g.M) break;  // warp-uniform
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    float v[16 / sizeof(T)];
#pragma unroll
                    for (int e = 0; e < 16 / (int)sizeof(T); e++) v[e] = acc[c + q * (16 / sizeof(T)) + e];
                    *reinterpret_cast<uint4*>(box + lane * 128 + ((q ^ (lane & 7)) << 4)) = pack16(v, T());
                }
                if (g.tma_c) {
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    __syncwarp();
                    if (lane == 0) tma_store_2d(&tmC, box, n0 + c, m0);
                } else {  // rows that TMA cannot address: element by element, a row at a time
                    __syncwarp();
                    for (int r = 0; r < 32 && m0 + r < g.M; r++)
                        for (int e = lane; e < BOX && n0 + c + e < g.N; e += 32)
                            ((T*)g.C)[(long long)(m0 + r) * g.ldc + n0 + c + e] = *reinterpret_cast<const T*>(
                                box + r * 128 + (((e * (int)sizeof(T) / 16) ^ (r & 7)) << 4) + e * sizeof(T) % 16);
                    __syncwarp();
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Tiles whose K was cut: the parts of 32 rows and 64 columns, summed in the order of K.
constexpr int J_COLS = 64;
template <typename T>
__global__ void __launch_bounds__(256) join_parts_kernel(const WideArgs g)
{
    __shared__ float rows[32][J_COLS + 1];
    wait_for_previous();
    const int tile = g.whole + blockIdx.x, rank = blockIdx.y >> 2, r0 = (blockIdx.y & 3) * 32, col0 = blockIdx.z * J_COLS;
    const int m0 = (tile % g.mt) * WT + rank * 128 + r0, n0 = (tile / g.mt) * WT + col0;
    if (m0 >= g.M || n0 >= g.N) return;
    const int r = threadIdx.x & 31, q = threadIdx.x >> 5;
    float4 v[2] = {};
    auto add = [&](int index) {
        const float* part = g.parts + ((long long)index * 2 + rank) * PART_FLOATS + (col0 / 4 * 128LL + r0 + r) * 4;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float4 x = *reinterpret_cast<const float4*>(part + (q + 8 * h) * 512);
            v[h].x += x.x, v[h].y += x.y, v[h].z += x.z, v[h].w += x.w;
        }
    };
    const int cut_tile = blockIdx.x;
    for (int i = 0; i < g.slices; i++) add(i * g.cut + cut_tile);
    if (g.tail) {
        const long long a = (long long)cut_tile * g.tail, b = a + g.tail;
        int c = (int)(a * g.tailers / ((long long)g.cut * g.tail));  // the share that holds block a, or the one before it
        while (tail_share(g, c + 1) <= a) c++;
        for (; c < g.tailers && tail_share(g, c) < b; c++) add(g.slices * g.cut + c + cut_tile);
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float* o = &rows[r][4 * (q + 8 * h)];
        o[0] = v[h].x, o[1] = v[h].y, o[2] = v[h].z, o[3] = v[h].w;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * J_COLS; i += 256) {
        const int m = i / J_COLS, e = i % J_COLS;
        if (m0 + m < g.M && n0 + e < g.N) ((T*)g.C)[(long long)(m0 + m) * g.ldc + n0 + e] = from_f<T>(rows[m][e]);
    }
}

// ---------------------------------------------------------------------------------------------------------- host side

bool make_map_out(CUtensorMap* m, void* base, int es, long long rows, long long cols, long long ld)
{
    auto f = encode_fn();
    if (!f) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(ld * es)};
    cuuint32_t box[2] = {(cuuint32_t)(128 / es), 32}, one[2] = {1, 1};
    return f(m, es == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base, dims, strides, box, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct WidePlan {
    int mt, tiles, nkb, pairs, whole, cut, slices, slice, tail, tailers;
    size_t workspace;
};
// Whole tiles in rounds of one per pair; the tiles of a last round that would leave pairs idle are shared along K when that
// saves more than the parts cost (their traffic and a launch, about 10 us; a block of K takes 0.5 us).
WidePlan plan_wide(int M, int N, int K, int sms)
{
    WidePlan p{};
    p.mt = (M + WT - 1) / WT;
    p.tiles = p.mt * ((N + WT - 1) / WT);
    p.nkb = (K + QB - 1) / QB;
    p.pairs = sms / 2 > 0 ? sms / 2 : 1;
    const int rest = p.tiles % p.pairs;
    const bool share = rest && (double)(p.pairs - rest) / p.pairs * p.nkb * 0.5 > 10.0;
    p.whole = p.tiles;
    if (share) {
        const long long blocks = (long long)rest * p.nkb;
        p.slice = (int)std::max((blocks + p.pairs - 1) / p.pairs, 4LL);  // of at least 20 blocks, or it would not save so much
        p.slices = p.nkb / p.slice;  // rest < pairs: at least one, and at most pairs / rest
        p.tail = p.nkb - p.slices * p.slice;
        if (p.slices > 1 || p.tail) {
            p.cut = rest, p.whole -= rest;
            // not 0 where there is a tail: with a pair for each slice the slices would have taken all of K
            const long long tails = (long long)rest * p.tail, left = p.pairs - p.slices * rest;
            p.tailers = (int)std::min((tails + 3) / 4, left);
        }
    }
    if (!p.cut) p.slice = p.slices = p.tail = p.tailers = 0;
    const int sharers = p.slices * p.cut + p.tailers, busy = p.whole < sharers ? sharers : p.whole;
    if (busy < p.pairs) p.pairs = busy;
    p.workspace = (size_t)(p.cut ? part_count(p.cut, p.slices, p.tail, p.tailers) : 0) * 2 * PART_FLOATS * 4;
    return p;
}

template <typename T>
int run_wide(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const WideArgs& g, const WidePlan& p, cudaStream_t st)
{
    static std::atomic<int> ready[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
    if (!ready[dev].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(gemm_wide_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, W_SMEM);
        if (e != cudaSuccess) return (int)e;
        ready[dev].store(1, std::memory_order_release);
    }
    const cudaError_t e = launch_next(gemm_wide_kernel<T>, 2 * p.pairs, W_THREADS, W_SMEM, st, ta, tb, tc, g);
    if (e != cudaSuccess || !p.cut) return (int)e;
    return (int)launch_next(join_parts_kernel<T>, dim3(p.cut, 8, WT / J_COLS), 256, 0, st, g);
}

}  // namespace

extern "C" size_t ltq_fp8_gemm_workspace_bytes(int M, int N, int K)
{
    if (M < 1 || N < 1 || K < 1) return 0;
    return plan_wide(M, N, K, sm_count()).workspace;
}

extern "C" int ltq_fp8_gemm(const uint8_t* A, long long lda, const float* sa, long long ld_sa, const uint8_t* B, long long ldb,
                            const float* sb, long long ld_sb, void* C, int dtype, long long ldc, int M, int N, int K,
                            void* workspace, size_t workspace_bytes, int* err, void* stream)
{
    const int es = dt_bytes(dtype);
    if (!es || M < 0 || N < 0 || K < 1 || ldc < N || ld_sa < M || ld_sa % 4 || ld_sb < (K + QB - 1) / QB) return -1;
    if (M == 0 || N == 0) return 0;
    if (bad_operand(A, lda, K) || bad_operand(B, ldb, K) || !sa || (uintptr_t)sa % 16 || !sb || (uintptr_t)sb % 4 || !C ||
        (uintptr_t)C % es || K > 0x7fffffff - QB || (long long)((M + WT - 1LL) / WT) * ((N + WT - 1LL) / WT) > 0x3fffffff)
        return -1;
    const WidePlan p = plan_wide(M, N, K, sm_count());
    if (p.workspace && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < p.workspace)) return -1;
    CUtensorMap ta, tb, tc{};
    if (!make_map_8(&ta, A, M, K, lda, 128) || !make_map_8(&tb, B, N, K, ldb, 128)) return -1;
    const int tma_c = (uintptr_t)C % 16 == 0 && ldc * es % 16 == 0;
    if (tma_c && !make_map_out(&tc, C, es, M, N, ldc)) return -1;
    const WideArgs g{sa, ld_sa, sb, ld_sb, C, ldc, (float*)workspace, err, M, N, p.nkb, p.mt, p.whole, tma_c,
                     p.cut, p.slices, p.slice, p.tail, p.tailers};
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F32) return run_wide<float>(ta, tb, tc, g, p, st);
    if (dtype == DT_BF16) return run_wide<__nv_bfloat16>(ta, tb, tc, g, p, st);
    return run_wide<__half>(ta, tb, tc, g, p, st);
}
