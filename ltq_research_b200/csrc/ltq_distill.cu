// Divergence of a student from a teacher's top logits, and its gradient by the student's logits (B200, sm_100a).
//
// Row t has logits z [V], K slots (id_k, teacher logit u_k; a slot whose id is outside [0, V) is empty), a temperature
// tau and a weight w.  q = softmax(z / tau) is the student.  The teacher is, without its log-sum-exp,
//     p = softmax of u / tau over the live slots, no rest (p_r = 0);  with it (lse, at the same temperature)
//     p_k = exp(u_k / tau - lse),  p_r = max(0, 1 - sum p),  one outcome for all tokens outside the slots.
// With S = sum_j exp(z_j / tau), S_r the same sum over the tokens outside the slots, q_r = S_r / S, P = sum p + p_r:
//     L      = w [ sum_k p_k (log p_k - log q_{id_k}) + p_r (log p_r - log q_r) ]
//     dL/dz_j = (w / tau) (q_j P - sum_{k: id_k = j} p_k)   for j in the slots,   (w / tau) q_j (P - p_r / q_r)   else,
// so outside the slots the gradient is one factor times exp(z_j / tau), and the K slots are set afterwards.  S_r is summed
// over the tokens outside the slots (a bitmap of the slots' ids), not taken as S minus the slots, which would cancel.
//
// A term with p_k = 0 is 0.  A row of weight 0, or without a live slot, has loss 0 and gradient 0 (weight 0: its logits
// are not read).  Where q_{id_k} = 0 < p_k the loss is +inf and the gradient finite (q_j = 0).  NaN logits give NaN.
#include <float.h>
#include <atomic>
#include "ltq_b200.h"
#include "vec_types.cuh"

namespace {

constexpr int DK_MAX = 1024;          // slots of a row
constexpr int D_THREADS = 512;
constexpr int D_MAXCL = 8;
constexpr int D_SMEM = 200 * 1024;   // dynamic shared memory of a CTA at most
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
enum { M_LOSS = 0, M_BOTH = 1, M_GRAD = 2 };

struct DistillParams {
    const void* z;
    long long ld;
    const void* idx;
    long long ld_idx;
    const void* u;
    long long ld_u;
    const float* lse;     // teacher's log-sum-exp, or NULL
    const float* weight;  // or NULL
    const float* grad;    // M_GRAD: upstream gradient of the loss, or NULL
    long long s_grad;
    float* loss;
    float* stats;  // [T][2]: log S, log q_r (natural logarithms)
    void* dz;
    long long ld_d;
    int T, V, K, idx64, u_dt;
    float inv_tau;
    int cl;        // CTAs of a row (cluster size)
    int hold;      // M_BOTH: vectors of a CTA's slice that stay in shared memory between the passes
    int bit_words; // words of the bitmap, before the held vectors in shared memory
    int vec_out;   // dz rows have the alignment of z rows
};

// products and sums are written out (no contraction left to the compiler), so that every mode gives the same bits
__device__ __forceinline__ float ex2(float x)
{
    float y;  // ex2.approx: relative error 2^-22, results below 2^-126 are 0
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait()
{
    asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

// (m, s) <- s 2^m-scaled sums joined: the pair (m, s) stands for s * 2^m
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2)
{
    const float M = fmaxf(m, m2);
    const float b = M == -INFINITY ? 0.f : M;
    s = __fmaf_rn(s, ex2(m - b), __fmul_rn(s2, ex2(m2 - b)));
    m = M;
}

template <int OP>  // 0 max, 1 sum, over the lanes of a warp; every lane gets the result
__device__ __forceinline__ float warp_reduce(float v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = OP ? v + w : fmaxf(v, w);
    }
    return v;
}
__device__ __forceinline__ void warp_join(float& m, float& s)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
        join(m, s, m2, s2);
    }
}

__device__ __forceinline__ float load_u(const void* u, int dt, long long i)
{
    return dt == DT_F32 ? ((const float*)u)[i]
           : dt == DT_BF16 ? __bfloat162float(((const __nv_bfloat16*)u)[i])
                           : __half2float(((const __half*)u)[i]);
}

template <typename T, int MODE, bool REST>
__global__ void __launch_bounds__(D_THREADS, 3) distill_kernel(const DistillParams p)
{
    constexpr int VEC = 16 / sizeof(T), WARPS = D_THREADS / 32;
    extern __shared__ __align__(16) uint32_t dsm[];  // bitmap, held vectors, slots
    __shared__ float red[2][WARPS];
    __shared__ float slot_sums[6];  // sum p, p_r, sum p log p, and the pair of the slots' tokens in this CTA's slice
    __shared__ float xch[4][D_MAXCL];
    __shared__ int dup;
    uint32_t* bits = dsm;
    float* pr = reinterpret_cast<float*>(dsm + p.bit_words + 4 * p.hold);  // u / tau, then p_k
    float* zk = pr + p.K;  // z of the slot's token in units of log2 (slots of this CTA's slice; all slots on CTA 0)
    int* id = reinterpret_cast<int*>(zk + p.K);  // token or -1

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, K = p.K, V = p.V, cl = p.cl;
    const int rank = cl > 1 ? (int)cluster_rank() : 0;
    const long long row = blockIdx.x / cl;
    const T* z = (const T*)p.z + row * p.ld;
    T* dz = MODE == M_LOSS ? nullptr : (T*)p.dz + row * p.ld_d;
    const float w = p.weight ? p.weight[row] : 1.f;
    if (cl > 1) cluster_arrive();  // paired with the wait before the exchange: every CTA of the row has started

    // the row's 16-byte vectors: `head` elements before the first, nb vectors, the tail; this CTA's are [v0, v1), and
    // its elements [j0, j1)
    const int phase = (int)(((uintptr_t)z & 15) / sizeof(T));
    const int head = min(V, (VEC - phase) % VEC);
    const int nb = (V - head) / VEC;
    const int per = (nb + cl - 1) / cl;
    const int v0 = min(nb, rank * per), v1 = min(nb, v0 + per);
    const int j0 = rank == 0 ? 0 : head + v0 * VEC, j1 = rank == cl - 1 ? V : head + v1 * VEC;
    const int jb = head + (v0 - 1) * VEC;  // element of bit 0: vector v's bits start at (v - v0 + 1) VEC

    if (w == 0.f) {  // no loss, no gradient; the logits may be anything
        if (MODE != M_GRAD && rank == 0 && tid == 0) {
            p.loss[row] = 0.f;
            if (p.stats) p.stats[2 * row] = 0.f, p.stats[2 * row + 1] = 0.f;
        }
        if (MODE != M_LOSS) {
            if (p.vec_out) {
                for (int v = v0 + tid; v < v1; v += D_THREADS)
                    __stcs(reinterpret_cast<uint4*>(dz + head + (long long)v * VEC), make_uint4(0, 0, 0, 0));
                if (rank == 0 && tid < head) dz[tid] = from_f<T>(0.f);
                if (rank == cl - 1 && head + nb * VEC + tid < V) dz[head + nb * VEC + tid] = from_f<T>(0.f);
            } else
                for (int j = j0 + tid; j < j1; j += D_THREADS) dz[j] = from_f<T>(0.f);
        }
        if (cl > 1) cluster_wait();
        return;
    }

    const uint4* zv = reinterpret_cast<const uint4*>(z + head);
    // M_BOTH: the slice is on its way to shared memory (each thread copies and later reads its own vectors, so that no
    // barrier is needed) in four batches while the slots are worked on
    const uint32_t held = (uint32_t)__cvta_generic_to_shared(dsm + p.bit_words);
    const int nh = MODE == M_BOTH ? min(v1 - v0, p.hold) : 0;
    const int batch = MODE == M_BOTH ? (nh + 4 * D_THREADS - 1) / (4 * D_THREADS) * D_THREADS : 0;
    if (MODE == M_BOTH) {
#pragma unroll
        for (int b = 0; b < 4; b++) {
            for (int i = b * batch + tid; i < min(nh, (b + 1) * batch); i += D_THREADS) cp16(held + 16 * i, zv + v0 + i);
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        }
    }

    // slots: ids, teacher logits, the student's logits at them, the bitmap
    const float c = p.inv_tau * LOG2E;
    const int nwords = ((v1 - v0 + 2) * VEC + 31) / 32;
    for (int i = tid; i < nwords; i += D_THREADS) bits[i] = 0;
    if (tid == 0) dup = 0;
    __syncthreads();
    for (int k = tid; k < K; k += D_THREADS) {
        const long long i = p.idx64 ? ((const long long*)p.idx)[row * p.ld_idx + k] : ((const int*)p.idx)[row * p.ld_idx + k];
        const float u = load_u(p.u, p.u_dt, row * p.ld_u + k);
        const bool live = i >= 0 && i < V, own = live && i >= j0 && i < j1;
        id[k] = live ? (int)i : -1;
        pr[k] = live ? __fmul_rn(u, p.inv_tau) : -INFINITY;
        if (live && (rank == 0 || own)) zk[k] = __fmul_rn(to_f(z[i]), c);
        if (own) {
            const int b = (int)i - jb;
            if (atomicOr(&bits[b >> 5], 1u << (b & 31)) >> (b & 31) & 1u) dup = 1;
        }
    }
    __syncthreads();
    const bool any_dup = dup != 0;
    auto leads = [&](int k) {  // slot k is the first with its id: of slots with one id the lowest stands for the token
        if (any_dup)
            for (int q = 0; q < k; q++)
                if (id[q] == id[k]) return false;
        return true;
    };

    const uint8_t* bytes = reinterpret_cast<const uint8_t*>(bits);
    auto member_bits = [&](int v) -> uint32_t {
        const int b = v - v0 + 1;
        return VEC == 8 ? bytes[b] : (bytes[b >> 1] >> ((b & 1) * 4)) & 15u;
    };
    auto is_member = [&](int j) { return (bits[(j - jb) >> 5] >> ((j - jb) & 31)) & 1u; };

    // one pass: (m, s) with the running maximum, over the tokens outside the slots (REST) or all
    float m = -INFINITY, s = 0.f;
    if (MODE != M_GRAD) {
        auto add = [&](const uint4& raw, int v) {
            float x[VEC];
            unpack16(raw, x, T());
            if (REST) {
                const uint32_t mb = member_bits(v);
                if (mb)
#pragma unroll
                    for (int i = 0; i < VEC; i++)
                        if (mb >> i & 1u) x[i] = -INFINITY;
            }
            float vm = x[0];
#pragma unroll
            for (int i = 1; i < VEC; i++) vm = fmaxf(vm, x[i]);
            vm = __fmul_rn(vm, c);
            if (vm > m) {
                s *= ex2(m - vm);
                m = vm;
            }
            const float b = m == -INFINITY ? 0.f : m;
            float t[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) t[i] = ex2(fmaf(x[i], c, -b));
#pragma unroll
            for (int o = VEC / 2; o; o >>= 1)
#pragma unroll
                for (int i = 0; i < o; i++) t[i] += t[i + o];
            s += t[0];
        };
        if (MODE == M_BOTH) {
            auto held_batch = [&](int b) {
                for (int i = b * batch + tid; i < min(nh, (b + 1) * batch); i += D_THREADS) {
                    uint4 u;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n"
                                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                                 : "r"(held + 16 * i));
                    add(u, v0 + i);
                }
            };
            cp_wait<3>();
            held_batch(0);
            cp_wait<2>();
            held_batch(1);
            cp_wait<1>();
            held_batch(2);
            cp_wait<0>();
            held_batch(3);
        }
        int v = v0 + nh + tid;
        for (; v + 3 * D_THREADS < v1; v += 4 * D_THREADS) {
            uint4 u[4];
#pragma unroll
            for (int q = 0; q < 4; q++) u[q] = __ldg(zv + v + q * D_THREADS);
#pragma unroll
            for (int q = 0; q < 4; q++) add(u[q], v + q * D_THREADS);
        }
        for (; v < v1; v += D_THREADS) add(__ldg(zv + v), v);
        auto scalar = [&](int j) {
            if (!(REST && is_member(j))) {
                const float x = __fmul_rn(to_f(z[j]), c);
                const float M = fmaxf(m, x), b = M == -INFINITY ? 0.f : M;
                s = __fmaf_rn(s, ex2(m - b), ex2(x - b));
                m = M;
            }
        };
        if (rank == 0 && tid < head) scalar(tid);
        if (rank == cl - 1 && head + nb * VEC + tid < V) scalar(head + nb * VEC + tid);
        warp_join(m, s);
        if (lane == 0) red[0][warp] = m, red[1][warp] = s;
    }
    // the slots' sums, on the last warp: p_k into pr, P, the entropy term, the pair of this CTA's tokens
    if (warp == WARPS - 1) {
        float lt;  // the teacher's log-sum-exp
        if (REST) lt = p.lse[row];
        else {
            float um = -INFINITY, t = 0.f;
            for (int k = lane; k < K; k += 32) um = fmaxf(um, pr[k]);
            um = warp_reduce<0>(um);
            const float b = um == -INFINITY ? 0.f : um;
            for (int k = lane; k < K; k += 32) t += ex2(__fmul_rn(pr[k] - b, LOG2E));
            t = warp_reduce<1>(t);
            lt = t == 0.f ? 0.f : b + logf(t);  // no live slot, or all of them -inf: p = 0
        }
        float psum = 0.f, plogp = 0.f, mt = -INFINITY, st = 0.f, distinct = 0.f;
        for (int k = lane; k < K; k += 32) {
            const int i = id[k];
            float pk = 0.f;
            if (i >= 0) {
                const float lp = pr[k] - lt;
                pk = ex2(__fmul_rn(lp, LOG2E));
                psum += pk;
                if (!(pk == 0.f)) plogp = __fmaf_rn(pk, lp, plogp);
                if (REST && MODE != M_GRAD && i >= j0 && i < j1 && leads(k)) join(mt, st, zk[k], 1.f);
                if (REST && K >= V) {
                    bool first = true;
                    for (int q = 0; q < k && first; q++) first = id[q] != i;
                    distinct += first ? 1.f : 0.f;
                }
            }
            pr[k] = pk;
        }
        psum = warp_reduce<1>(psum);
        plogp = warp_reduce<1>(plogp);
        if (REST && MODE != M_GRAD) warp_join(mt, st);
        float prest = REST ? fmaxf(1.f - psum, 0.f) : 0.f;
        if (REST && K >= V && warp_reduce<1>(distinct) == (float)V) prest = 0.f;  // slots that hold every token leave no rest
        if (lane == 0) slot_sums[0] = psum, slot_sums[1] = prest, slot_sums[2] = plogp, slot_sums[3] = mt, slot_sums[4] = st;
    }
    __syncthreads();
    const float psum = slot_sums[0], prest = slot_sums[1];

    float log2S, log2qr;  // log2 of S and of q_r
    if (MODE != M_GRAD) {
        m = lane < WARPS ? red[0][lane] : -INFINITY;
        s = lane < WARPS ? red[1][lane] : 0.f;
        warp_join(m, s);
        float mt = slot_sums[3], st = slot_sums[4];
        if (cl > 1) {
            cluster_wait();
            if (tid < cl) {
                st_cluster_u32(&xch[0][rank], tid, __float_as_uint(m));
                st_cluster_u32(&xch[1][rank], tid, __float_as_uint(s));
                st_cluster_u32(&xch[2][rank], tid, __float_as_uint(mt));
                st_cluster_u32(&xch[3][rank], tid, __float_as_uint(st));
            }
            cluster_arrive();
            cluster_wait();
            m = mt = -INFINITY, s = st = 0.f;
            for (int q = 0; q < cl; q++) join(m, s, xch[0][q], xch[1][q]), join(mt, st, xch[2][q], xch[3][q]);
        }
        float ma = m, sa = s;
        if (REST) join(ma, sa, mt, st);
        log2S = ma + log2f(sa);
        log2qr = !REST || s == 0.f ? -INFINITY : m + log2f(s) - log2S;
        if (rank == 0 && warp == 0) {
            float l = 0.f;
            const float b = log2S == -INFINITY ? 0.f : log2S;
            for (int k = lane; k < K; k += 32)
                if (!(pr[k] == 0.f)) l = __fmaf_rn(-pr[k], __fmul_rn(zk[k] - b, LN2), l);
            l = warp_reduce<1>(l) + slot_sums[2];
            if (lane == 0) {
                if (prest > 0.f) l = __fmaf_rn(prest, __fmaf_rn(-log2qr, LN2, logf(prest)), l);
                p.loss[row] = __fmul_rn(w, l);
                if (p.stats) p.stats[2 * row] = log2S * LN2, p.stats[2 * row + 1] = log2qr * LN2;
            }
        }
    } else {
        log2S = p.stats[2 * row] * LOG2E;
        log2qr = p.stats[2 * row + 1] * LOG2E;
        if (cl > 1) cluster_wait();
    }

    if (MODE != M_LOSS) {
        const float g = MODE == M_GRAD && p.grad ? p.grad[row * p.s_grad] : 1.f;
        const float scale = g * w * p.inv_tau;
        const float P = psum + prest;
        // outside the slots: scale (P - p_r / q_r) 2^(z c - log2 S); a rest that the student gives nothing has q_j = 0
        const float cr = scale * (prest > 0.f ? (log2qr == -INFINITY ? 0.f : P - prest * ex2(-log2qr)) : P);
        const float b = log2S == -INFINITY ? 0.f : log2S;
        auto grad_of = [&](float x) { return cr * ex2(fmaf(x, c, -b)); };
        if (p.vec_out) {
            auto put = [&](const uint4& raw, int v) {
                float x[VEC];
                unpack16(raw, x, T());
#pragma unroll
                for (int i = 0; i < VEC; i++) x[i] = grad_of(x[i]);
                __stcs(reinterpret_cast<uint4*>(dz + head + (long long)v * VEC), pack16(x, T()));
            };
            for (int i = tid; i < nh; i += D_THREADS) {
                uint4 u;
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n"
                             : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                             : "r"(held + 16 * i));
                put(u, v0 + i);
            }
            // plain loads: the rows may be overwritten (dz = z), each vector by the thread that has read it
            int v = v0 + nh + tid;
            for (; v + 3 * D_THREADS < v1; v += 4 * D_THREADS) {
                uint4 u[4];
#pragma unroll
                for (int q = 0; q < 4; q++) u[q] = zv[v + q * D_THREADS];
#pragma unroll
                for (int q = 0; q < 4; q++) put(u[q], v + q * D_THREADS);
            }
            for (; v < v1; v += D_THREADS) put(zv[v], v);
            if (rank == 0 && tid < head) dz[tid] = from_f<T>(grad_of(to_f(z[tid])));
            if (rank == cl - 1 && head + nb * VEC + tid < V)
                dz[head + nb * VEC + tid] = from_f<T>(grad_of(to_f(z[head + nb * VEC + tid])));
        } else
            for (int j = j0 + tid; j < j1; j += D_THREADS) dz[j] = from_f<T>(grad_of(to_f(z[j])));
        __syncthreads();
        for (int k = tid; k < K; k += D_THREADS) {
            if (id[k] < 0 || id[k] < j0 || id[k] >= j1 || !leads(k)) continue;
            float pk = pr[k];
            if (any_dup)
                for (int q = k + 1; q < K; q++)
                    if (id[q] == id[k]) pk += pr[q];
            dz[id[k]] = from_f<T>(scale * (P * ex2(zk[k] - b) - pk));
        }
    }
}

template <typename T, int MODE, bool REST>
int launch(DistillParams p, int cl, cudaStream_t st)
{
    constexpr int VEC = 16 / sizeof(T);
    const int per = (p.V / VEC + cl - 1) / cl;
    p.bit_words = (((per + 2) * VEC + 31) / 32 + 3) / 4 * 4;
    p.hold = MODE == M_BOTH ? per : 0;
    const int fixed = p.bit_words * 4 + p.K * 12;
    if (fixed + p.hold * 16 > D_SMEM) p.hold = (D_SMEM - fixed) / 16;
    const int smem = fixed + p.hold * 16;
    auto k = distill_kernel<T, MODE, REST>;
    if (smem > 46 * 1024) {  // beyond the default 48 KB with the static arrays
        static std::atomic<int> ready[64];
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
        if (!ready[dev].load(std::memory_order_acquire)) {
            const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, D_SMEM);
            if (e != cudaSuccess) return (int)e;
            ready[dev].store(1, std::memory_order_release);
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long long)p.T * cl));
    cfg.blockDim = dim3(D_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)cl, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = cl > 1 ? 1 : 0;
    return (int)cudaLaunchKernelEx(&cfg, k, p);
}

// CTAs of a row.  Loss and gradient: as few as let a slice stay in 72 KB of shared memory (three CTAs an SM, one row's
// loads under another's exponentials and stores), so that the row is read from memory once; otherwise one.  Few rows: more, until
// the GPU's SMs have one each.
int row_ctas(long long T, int V, int es, int mode)
{
    int cl = 1;
    if (mode == M_BOTH)
        while (cl < D_MAXCL && (long long)V * es > 72 * 1024LL * cl) cl *= 2;
    while (cl < D_MAXCL && T * cl < 148 && (long long)V * es / cl > 16 * 1024) cl *= 2;
    return cl;
}

template <typename T>
int dispatch(const DistillParams& p, int mode, int cl, cudaStream_t st)
{
    const bool rest = p.lse != nullptr;
    if (mode == M_LOSS) return rest ? launch<T, M_LOSS, true>(p, cl, st) : launch<T, M_LOSS, false>(p, cl, st);
    if (mode == M_BOTH) return rest ? launch<T, M_BOTH, true>(p, cl, st) : launch<T, M_BOTH, false>(p, cl, st);
    return rest ? launch<T, M_GRAD, true>(p, cl, st) : launch<T, M_GRAD, false>(p, cl, st);
}

}  // namespace

extern "C" int ltq_distill_topk(const void* logits, int dtype, long long ld, const void* idx, int idx64, long long ld_idx,
                                const void* teacher, int teacher_dtype, long long ld_t, const float* teacher_lse,
                                const float* weight, const float* grad, long long grad_stride, int T, int V, int K,
                                float temperature, int mode, float* loss, float* stats, void* dlogits, long long ld_d,
                                void* stream)
{
    const int es = dt_bytes(dtype);
    if (!es || !dt_bytes(teacher_dtype) || T < 0 || V <= 0 || V > (1 << 20) || K < 1 || K > DK_MAX || mode < 0 || mode > 2 ||
        !(temperature > 0.f) || !(temperature <= FLT_MAX) || ld < V || ld_idx < K || ld_t < K)
        return -1;
    if (T == 0) return 0;
    if ((long long)T * D_MAXCL > 0x7fffffffLL) return -1;
    if (!logits || !idx || !teacher || ((uintptr_t)logits % es) || (mode != M_GRAD && !loss) || (mode == M_GRAD && !stats) ||
        (mode != M_LOSS && (!dlogits || ld_d < V || ((uintptr_t)dlogits % es))))
        return -1;
    DistillParams p{};
    p.z = logits, p.ld = ld, p.idx = idx, p.ld_idx = ld_idx, p.u = teacher, p.ld_u = ld_t, p.lse = teacher_lse;
    p.weight = weight, p.grad = grad, p.s_grad = grad_stride, p.loss = loss, p.stats = stats, p.dz = dlogits, p.ld_d = ld_d;
    p.T = T, p.V = V, p.K = K, p.idx64 = idx64 != 0, p.u_dt = teacher_dtype, p.inv_tau = 1.f / temperature;
    p.vec_out = mode != M_LOSS && ((uintptr_t)logits & 15) == ((uintptr_t)dlogits & 15) && ((ld - ld_d) * es) % 16 == 0;
    const int cl = p.cl = row_ctas(T, V, es, mode);
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F32) return dispatch<float>(p, mode, cl, st);
    if (dtype == DT_BF16) return dispatch<__nv_bfloat16>(p, mode, cl, st);
    return dispatch<__half>(p, mode, cl, st);
}
