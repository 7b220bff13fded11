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
#include "ltq_b200.h"
#include "vec_types.cuh"

namespace {

constexpr int DK_MAX = 1024;          // slots of a row
constexpr int D_THREADS = 512;
constexpr int D_MAXCL = 8;
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
    int vec_out;   // dz rows have the alignment of z rows
};

// products and sums are written out (no contraction left to the compiler), so that every mode gives the same bits
__device__ __forceinline__ float ex2(float x) { return exp2f(x); }

// (m, s) <- s 2^m-scaled sums joined: the pair (m, s) stands for s * 2^m
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2)
{
    const float M = fmaxf(m, m2);
    const float b = M == -INFINITY ? 0.f : M;
    s = __fmaf_rn(s, ex2(m - b), __fmul_rn(s2, ex2(m2 - b)));
    m = M;
}

template <int OP>  // 0 max, 1 sum; every thread gets the result; red: 32 floats of shared memory
__device__ __forceinline__ float block_reduce(float v, float* red)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = OP ? v + w : fmaxf(v, w);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < D_THREADS / 32 ? red[threadIdx.x & 31] : (OP ? 0.f : -INFINITY);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = OP ? v + w : fmaxf(v, w);
    }
    return v;
}

// joins the (m, s) pairs of all threads in a fixed order; every thread gets the result
__device__ __forceinline__ void block_join(float& m, float& s, float* red)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
        join(m, s, m2, s2);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m, red[32 + (threadIdx.x >> 5)] = s;
    __syncthreads();
    const int l = threadIdx.x & 31;
    m = l < D_THREADS / 32 ? red[l] : -INFINITY;
    s = l < D_THREADS / 32 ? red[32 + l] : 0.f;
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
__global__ void __launch_bounds__(D_THREADS) distill_kernel(const DistillParams p)
{
    constexpr int VEC = 16 / sizeof(T);
    extern __shared__ uint32_t dsm[];
    __shared__ float red[64];
    __shared__ float pr[DK_MAX];   // p_k
    __shared__ float zk[DK_MAX];   // z of the slot's token, in units of log2 (slots of this CTA; all slots on CTA 0)
    __shared__ int id[DK_MAX];     // token or -1
    __shared__ float xch[4][D_MAXCL];
    __shared__ int dup;
    uint32_t* bits = dsm;

    const int tid = threadIdx.x, K = p.K, V = p.V, cl = p.cl;
    const int rank = cl > 1 ? (int)cluster_rank() : 0;
    const long long row = blockIdx.x / cl;
    const T* z = (const T*)p.z + row * p.ld;
    T* dz = MODE == M_LOSS ? nullptr : (T*)p.dz + row * p.ld_d;
    const float w = p.weight ? p.weight[row] : 1.f;
    const float g = MODE == M_GRAD && p.grad ? p.grad[row * p.s_grad] : 1.f;
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
                    *reinterpret_cast<uint4*>(dz + head + (long long)v * VEC) = make_uint4(0, 0, 0, 0);
                if (rank == 0 && tid < head) dz[tid] = from_f<T>(0.f);
                if (rank == cl - 1 && head + nb * VEC + tid < V) dz[head + nb * VEC + tid] = from_f<T>(0.f);
            } else
                for (int j = j0 + tid; j < j1; j += D_THREADS) dz[j] = from_f<T>(0.f);
        }
        if (cl > 1) cluster_wait();
        return;
    }

    // slots: ids, p, the student's logits at them, the bitmap
    const float c = p.inv_tau * LOG2E;
    const int nwords = ((v1 - v0 + 2) * VEC + 31) / 32;
    for (int i = tid; i < nwords; i += D_THREADS) bits[i] = 0;
    if (tid == 0) dup = 0;
    float um = -INFINITY;
    for (int k = tid; k < K; k += D_THREADS) {
        const long long i = p.idx64 ? ((const long long*)p.idx)[row * p.ld_idx + k] : ((const int*)p.idx)[row * p.ld_idx + k];
        const bool live = i >= 0 && i < V;
        const float u = live ? __fmul_rn(load_u(p.u, p.u_dt, row * p.ld_u + k), p.inv_tau) : -INFINITY;
        id[k] = live ? (int)i : -1;
        pr[k] = u;
        if (live && (rank == 0 || (i >= j0 && i < j1))) zk[k] = __fmul_rn(to_f(z[i]), c);
        um = fmaxf(um, u);
    }
    float lt;  // the teacher's log-sum-exp
    if (REST) {
        lt = p.lse[row];
        __syncthreads();
    } else {
        um = block_reduce<0>(um, red);
        const float b = um == -INFINITY ? 0.f : um;
        float s = 0.f;
        for (int k = tid; k < K; k += D_THREADS) s += ex2(__fmul_rn(pr[k] - b, LOG2E));
        s = block_reduce<1>(s, red);
        lt = s == 0.f ? 0.f : b + logf(s);  // no live slot, or all of them -inf: p = 0
    }
    // pr: from u / tau to p; P and the entropy term need it all
    float psum = 0.f, plogp = 0.f;
    for (int k = tid; k < K; k += D_THREADS) {
        if (id[k] >= 0) {
            const float lp = pr[k] - lt, pk = ex2(__fmul_rn(lp, LOG2E));
            pr[k] = pk;
            psum += pk;
            if (!(pk == 0.f)) plogp = __fmaf_rn(pk, lp, plogp);
            const int b = id[k] - jb;
            if (id[k] >= j0 && id[k] < j1)
                if (atomicOr(&bits[b >> 5], 1u << (b & 31)) >> (b & 31) & 1u) dup = 1;
        } else
            pr[k] = 0.f;
    }
    psum = block_reduce<1>(psum, red);
    float prest = REST ? fmaxf(1.f - psum, 0.f) : 0.f;
    if (REST && K >= V) {  // slots that hold every token leave no rest
        float distinct = 0.f;
        for (int k = tid; k < K; k += D_THREADS) {
            bool first = id[k] >= 0;
            for (int q = 0; q < k && first; q++) first = id[q] != id[k];
            distinct += first ? 1.f : 0.f;
        }
        if (block_reduce<1>(distinct, red) == (float)V) prest = 0.f;
    }
    __syncthreads();
    // of slots with one id the lowest stands for the token
    const bool any_dup = dup != 0;
    auto leads = [&](int k) {  // slot k is the first with its id
        if (any_dup)
            for (int q = 0; q < k; q++)
                if (id[q] == id[k]) return false;
        return true;
    };

    const uint4* zv = reinterpret_cast<const uint4*>(z + head);
    const uint8_t* bytes = reinterpret_cast<const uint8_t*>(bits);
    auto member_bits = [&](int v) -> uint32_t {
        const int b = v - v0 + 1;
        return VEC == 8 ? bytes[b] : (bytes[b >> 1] >> ((b & 1) * 4)) & 15u;
    };
    auto is_member = [&](int j) { return (bits[(j - jb) >> 5] >> ((j - jb) & 31)) & 1u; };

    float log2S, log2qr;  // log2 of S and of q_r
    if (MODE != M_GRAD) {
        // one pass: (m, s) with the running maximum, over the tokens outside the slots (REST) or all
        float m = -INFINITY, s = 0.f;
        for (int v = v0 + tid; v < v1; v += D_THREADS) {
            float x[VEC];
            unpack16(__ldg(zv + v), x, T());
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
#pragma unroll
            for (int i = 0; i < VEC; i++) s += ex2(fmaf(x[i], c, -b));
        }
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
        block_join(m, s, red);
        float mt = -INFINITY, st = 0.f;  // the slots' tokens of this CTA
        if (REST) {
            for (int k = tid; k < K; k += D_THREADS)
                if (id[k] >= j0 && id[k] < j1 && leads(k)) join(mt, st, zk[k], 1.f);
            block_join(mt, st, red);
        }
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
        if (rank == 0) {
            float l = 0.f;
            const float b = log2S == -INFINITY ? 0.f : log2S;
            for (int k = tid; k < K; k += D_THREADS)
                if (!(pr[k] == 0.f)) l = __fmaf_rn(-pr[k], __fmul_rn(zk[k] - b, LN2), l);
            l = block_reduce<1>(l + plogp, red);
            if (tid == 0) {
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
        const float scale = g * w * p.inv_tau;
        const float P = psum + prest;
        // outside the slots: scale (P - p_r / q_r) 2^(z c - log2 S); a rest that the student gives nothing has q_j = 0
        const float cr = scale * (prest > 0.f ? (log2qr == -INFINITY ? 0.f : P - prest * ex2(-log2qr)) : P);
        const float b = log2S == -INFINITY ? 0.f : log2S;
        auto grad_of = [&](float x) { return cr * ex2(fmaf(x, c, -b)); };
        if (p.vec_out) {
            for (int v = v0 + tid; v < v1; v += D_THREADS) {
                float x[VEC];
                unpack16(__ldg(zv + v), x, T());
#pragma unroll
                for (int i = 0; i < VEC; i++) x[i] = grad_of(x[i]);
                *reinterpret_cast<uint4*>(dz + head + (long long)v * VEC) = pack16(x, T());
            }
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
int launch(const DistillParams& p, int cl, cudaStream_t st)
{
    constexpr int VEC = 16 / sizeof(T);
    const int per = (p.V / VEC + cl - 1) / cl;
    const int smem = (((per + 2) * VEC + 31) / 32) * 4;
    auto k = distill_kernel<T, MODE, REST>;
    if (smem > 32768) {  // beyond the default 48 KB with the static arrays
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return (int)e;
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
    const int cl = p.cl = 1;
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F32) return dispatch<float>(p, mode, cl, st);
    if (dtype == DT_BF16) return dispatch<__nv_bfloat16>(p, mode, cl, st);
    return dispatch<__half>(p, mode, cl, st);
}
