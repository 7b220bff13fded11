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
// The fast kernels take exponentials relative to a maximum in units of log2, z log2(e) / tau, rounded to fp32.  That holds while
// the maximum is below BIG in magnitude (what lies below -BIG counts as 0 there).  Where the student has less than 2^-60 of its mass
// outside the slots (a masked vocabulary), P - p_r / q_r and exponentials relative to the row's maximum would leave fp32's range, and
// the rest has a maximum of its own.  Other rows (masked with -1e10 or the type's lowest value, very low temperatures) are
// found by their statistics and done again by exact_row from differences of logits, which are exact where they count.
//
// A term with p_k = 0 is 0.  A row of weight 0, or without a live slot, has loss 0 and gradient 0 (weight 0: its logits
// are not read).  Where q_{id_k} = 0 < p_k the loss is +inf and the gradient finite (q_j = 0).  NaN logits give NaN.
#include <float.h>
#include <algorithm>
#include <atomic>
#include "launch_next.cuh"
#include "ltq_b200.h"
#include "vec_types.cuh"

namespace {

constexpr int DK_MAX = 1024;          // slots of a row
constexpr int D_THREADS = 256;
constexpr int D_MAXCL = 8;
constexpr long long D_ROW = 72 * 1024, D_SLICE = 52 * 1024;  // shared memory for a whole row of one CTA, for a cluster CTA's slice
constexpr int D_SMEM = 200 * 1024;   // dynamic shared memory of a CTA at most
constexpr float BIG = 0x1p30f;        // an exponent's rounding error, 2^-25 of it, stays far inside fp32's range
constexpr uint32_t TO_DO = 0x7fd15711u;  // a NaN that no arithmetic makes: loss of a row that exact_rows_kernel will do
constexpr float FAR_REST = -60.f;     // log2 q_r below which the rest's gradient is taken relative to the rest's own sum
constexpr double LOG2E_D = 1.4426950408889634, LN2_D = 0.6931471805599453;
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
    float* stats;  // [T][3]: S as sa 2^ma (ma, sa), log2 q_r
    void* dz;
    long long ld_d;
    int T, V, K, idx64, u_dt;
    float inv_tau;
    double inv_tau_d;
    int cl;         // CTAs of a row (cluster size)
    int hold;       // vectors of a slice that are held in shared memory
    int bit_words;  // words of the bitmap, before the held vectors in shared memory
    int vec_out;    // dz rows have the alignment of z rows
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

// (m, s) <- s 2^m-scaled sums joined: the pair (m, s) stands for s * 2^m; m is at least -BIG
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2)
{
    const float M = fmaxf(m, m2);
    s = __fmaf_rn(s, ex2(m - M), __fmul_rn(s2, ex2(m2 - M)));
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
// joins the pairs of groups of N lanes; the maximum first (NaN pairs do not raise it), then one rescaling and a sum
template <int N>
__device__ __forceinline__ void warp_join(float& m, float& s)
{
    float M = m;
#pragma unroll
    for (int o = N / 2; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    s = __fmul_rn(s, ex2(m - M));
#pragma unroll
    for (int o = N / 2; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    m = M;
}

__device__ __forceinline__ float load_u(const void* u, int dt, long long i)
{
    return dt == DT_F32 ? ((const float*)u)[i]
           : dt == DT_BF16 ? __bfloat162float(((const __nv_bfloat16*)u)[i])
                           : __half2float(((const __half*)u)[i]);
}

// The slice of a row that a CTA of the row's cluster works on: the row's 16-byte vectors begin `head` elements in, nb of them;
// this CTA's are [v0, v1), its elements [j0, j1) (the elements before and behind the vectors belong to the first and last CTA).
template <typename T>
struct Slice {
    const T* z;
    int head, nb, v0, v1, j0, j1;
    __device__ Slice(const DistillParams& p, long long row, int rank)
    {
        constexpr int VEC = 16 / sizeof(T);
        z = (const T*)p.z + row * p.ld;
        const int phase = (int)(((uintptr_t)z & 15) / sizeof(T));
        head = min(p.V, (VEC - phase) % VEC);
        nb = (p.V - head) / VEC;
        const int per = (nb + p.cl - 1) / p.cl;
        v0 = min(nb, rank * per), v1 = min(nb, v0 + per);
        j0 = rank == 0 ? 0 : head + v0 * VEC;
        j1 = rank == p.cl - 1 ? p.V : head + v1 * VEC;
    }
    __device__ int tail() const { return head + nb * (16 / (int)sizeof(T)); }
};

__device__ __forceinline__ void load_slot(const DistillParams& p, long long row, int k, int& id, float& u)
{
    const long long i = p.idx64 ? ((const long long*)p.idx)[row * p.ld_idx + k] : ((const int*)p.idx)[row * p.ld_idx + k];
    const float t = load_u(p.u, p.u_dt, row * p.ld_u + k);
    id = i >= 0 && i < p.V ? (int)i : -1;
    u = id >= 0 ? t : -INFINITY;
}

template <typename F>
__device__ __forceinline__ F warp_sum(F v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// p_k into pr (from u) on one warp, rounded to fp32; returns P's two parts and sum p log p.  In 64 bits: p_r is what the others leave
// of 1, and the loss is small beside its terms, so both of its sums take the same rounded p (a student that equals its teacher had
// losses of 3e-7 otherwise); K exponentials on one warp while the others read the row cost no time.
template <bool REST>
__device__ __forceinline__ void teacher_probabilities(const DistillParams& p, float lse, float* pr, const int* id, int lane,
                                                      double& psum, double& prest, double& plogp)
{
    const int K = p.K;
    double um = 0.0, lt = lse;  // without rest: the largest u / tau, and the log of the sum relative to it
    if (!REST) {
        float m = -INFINITY;
        for (int k = lane; k < K; k += 32) m = fmaxf(m, pr[k]);
        m = warp_reduce<0>(m);
        um = m == -INFINITY ? 0.0 : __dmul_rn(m, p.inv_tau_d);
        double t = 0.0;
        for (int k = lane; k < K; k += 32) t += exp(__fma_rn(pr[k], p.inv_tau_d, -um));
        t = warp_sum(t);
        lt = t == 0.0 ? 0.0 : log(t);  // 0: no live slot, or all of them -inf: p = 0
    }
    int distinct = 0;
    psum = plogp = 0.0;
    for (int k = lane; k < K; k += 32) {
        double pk = 0.0;
        if (id[k] >= 0) {
            const double lp = __fma_rn(pr[k], p.inv_tau_d, -um) - lt;
            pk = exp(lp);
            psum += pk;
            if (!((float)pk == 0.f)) plogp = __fma_rn((double)(float)pk, lp, plogp);  // p as it is held and meets log q
            if (REST && K >= p.V) {
                bool first = true;
                for (int q = 0; q < k && first; q++) first = id[q] != id[k];
                distinct += first;
            }
        }
        pr[k] = (float)pk;
    }
    psum = warp_sum(psum);
    plogp = warp_sum(plogp);
    prest = REST ? fmax(1.0 - psum, 0.0) : 0.0;
    if (REST && psum != psum) prest = psum;  // NaN
    if (REST && K >= p.V && warp_sum(distinct) == p.V) prest = 0.0;  // slots that hold every token leave no rest
}

// slot k is the first with its id: of slots with one id the lowest stands for the token
__device__ __forceinline__ bool leads(const int* id, int k)
{
    for (int q = 0; q < k; q++)
        if (id[q] == id[k]) return false;
    return true;
}

// what the gradient of a row needs, S = sa 2^ma: outside the slots cr 2^(z c - br), for a slot's token Pq 2^(z c - b) - scale sum p
struct GradScale {
    float scale, Pq, cr, b, br;
    __device__ GradScale(float scale_, float psum, float prest, float ma, float sa, float log2qr) : scale(scale_), b(ma), br(ma)
    {
        const float P = psum + prest, inv = 1.f / sa;
        Pq = scale * P * inv;
        cr = scale * (prest > 0.f ? P - prest * ex2(-log2qr) : P) * inv;
    }
    // a rest of which the student has so little that p_r / q_r overflows and 2^(z c - b) ends at 0: relative to its own pair (m, s)
    __device__ void far_rest(float psum, float prest, float log2qr, float m, float s)
    {
        br = m, cr = scale * ((psum + prest) * ex2(log2qr) - prest) / s;
    }
};
template <typename T>
__device__ __forceinline__ uint4 grad16(const uint4& raw, uint64_t cc, uint64_t bb, uint64_t rr)
{
    constexpr int VEC = 16 / sizeof(T);
    float x[VEC];
    unpack16(raw, x, T());
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
        const float2 e = unpair(fma2(pair(x[i], x[i + 1]), cc, bb));
        const float2 d = unpair(mul2(rr, pair(ex2(e.x), ex2(e.y))));
        x[i] = d.x, x[i + 1] = d.y;
    }
    return pack16(x, T());
}
template <typename T>
__device__ __forceinline__ void zero_slice(const DistillParams& p, const Slice<T>& w, T* dz, int rank, int tid, int threads)
{
    constexpr int VEC = 16 / sizeof(T);
    if (p.vec_out) {
        for (int v = w.v0 + tid; v < w.v1; v += threads)
            __stcs(reinterpret_cast<uint4*>(dz + w.head + (long long)v * VEC), make_uint4(0, 0, 0, 0));
        if (rank == 0 && tid < w.head) dz[tid] = from_f<T>(0.f);
        if (rank == p.cl - 1 && w.tail() + tid < p.V) dz[w.tail() + tid] = from_f<T>(0.f);
    } else
        for (int j = w.j0 + tid; j < w.j1; j += threads) dz[j] = from_f<T>(0.f);
}

// ------------------------------------------------------------------------------------- rows outside the fast kernels' range

// f(j, z_j) for the tokens of a slice outside the slots, in stretches of a bitmap of `words` words
template <typename T, typename F>
__device__ __forceinline__ void over_rest(const Slice<T>& sl, const int* id, int K, uint32_t* bits, int words, F f)
{
    constexpr int AHEAD = 8;  // loads in flight
    for (int a = sl.j0; a < sl.j1; a += 32 * words) {
        const int n = min(32 * words, sl.j1 - a), step = blockDim.x;
        for (int i = threadIdx.x; i < (n + 31) / 32; i += step) bits[i] = 0;
        __syncthreads();
        for (int k = threadIdx.x; k < K; k += step)
            if (id[k] >= a && id[k] < a + n) atomicOr(&bits[(id[k] - a) >> 5], 1u << ((id[k] - a) & 31));
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += AHEAD * step) {
            T z[AHEAD];
#pragma unroll
            for (int q = 0; q < AHEAD; q++)
                if (j + q * step < n) z[q] = sl.z[a + j + q * step];
#pragma unroll
            for (int q = 0; q < AHEAD; q++) {
                const int t = j + q * step;
                if (t < n && !(bits[t >> 5] >> (t & 31) & 1u)) f(a + t, to_f(z[q]));
            }
        }
        __syncthreads();
    }
}

// what the kernels find out about the slots of a row
struct SlotSums {
    float psum, prest, mt, st;  // sum p, p_r, the pair of the slots' tokens in the slice
    double plogp, prest64;
    int dup;  // slots may name one token more than once
};
__shared__ SlotSums sums;
__shared__ float xch[4][D_MAXCL];  // of the row's CTAs
extern __shared__ __align__(128) uint32_t dsm[];  // bitmap, held slice, then p_k, z and id of the slots

constexpr int PART_WARPS = 16, MIN_BIT_WORDS = 2 * PART_WARPS * 2;

// One row (a CTA's slice of it) whatever its logits' range: sums and gradient from exponentials of differences to the largest logit
// of the rest, of the slots and of the row, statistics in 64 bits.  Three passes over the row, element by element.  All threads of the row's CTAs come here together, with the slots in shared memory.
template <typename T, bool REST, int MODE>
__device__ __forceinline__ void exact_row(const DistillParams& p, long long row)
{
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5, K = p.K, cl = p.cl;
    const int rank = cl > 1 ? (int)cluster_rank() : 0;
    uint32_t* bits = dsm;
    // the warps' sums, where the bitmap is between two passes
    double(*dpart)[PART_WARPS] = reinterpret_cast<double(*)[PART_WARPS]>(dsm);
    float(*part)[PART_WARPS] = reinterpret_cast<float(*)[PART_WARPS]>(dsm);
    const float* pr = reinterpret_cast<const float*>(dsm + p.bit_words + 4 * p.hold);
    const float* zk = pr + K;
    const int* id = reinterpret_cast<const int*>(zk + K);
    const Slice<T> sl(p, row, rank);
    const float c = (float)(p.inv_tau_d * LOG2E_D), w = p.weight ? p.weight[row] : 1.f;
    const double prest = REST ? sums.prest64 : 0.0;
    auto counts = [&](int k) { return id[k] >= 0 && id[k] >= sl.j0 && id[k] < sl.j1 && (!sums.dup || leads(id, k)); };
    // four values of each of the row's CTAs to all of them
    auto exchange = [&](float v0, float v1, float v2, float v3) {
        const float v[4] = {v0, v1, v2, v3};
        if (cl > 1) {
            cluster_arrive(), cluster_wait();  // all CTAs have read what was there
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (tid < cl) st_cluster_u32(&xch[i][rank], tid, __float_as_uint(v[i]));
            cluster_arrive(), cluster_wait();
        } else {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (tid == 0) xch[i][0] = v[i];
            __syncthreads();
        }
    };
    float mr = -INFINITY, mt = -INFINITY;  // the largest logit outside the slots, and in them
    over_rest(sl, id, K, bits, p.bit_words, [&](int, float z) { mr = fmaxf(mr, z); });
    for (int k = tid; k < K; k += blockDim.x)
        if (counts(k)) mt = fmaxf(mt, zk[k]);
    mr = warp_reduce<0>(mr), mt = warp_reduce<0>(mt);
    if (lane == 0) part[0][warp] = mr, part[1][warp] = mt;
    __syncthreads();
    for (int w = 0; w < warps; w++) mr = fmaxf(mr, part[0][w]), mt = fmaxf(mt, part[1][w]);
    exchange(mr, mt, 0.f, 0.f);
    for (int q = 0; q < cl; q++) mr = fmaxf(mr, xch[0][q]), mt = fmaxf(mt, xch[1][q]);
    const float rr = mr == -INFINITY ? 0.f : mr, rt = mt == -INFINITY ? 0.f : mt;
    double sr = 0.0, st = 0.0;
    over_rest(sl, id, K, bits, p.bit_words, [&](int, float z) { sr += ex2(__fmul_rn(z - rr, c)); });
    for (int k = tid; k < K; k += blockDim.x)
        if (counts(k)) st += exp2(((double)zk[k] - rt) * c);
    sr = warp_sum(sr), st = warp_sum(st);
    if (lane == 0) dpart[0][warp] = sr, dpart[1][warp] = st;
    __syncthreads();
    sr = st = 0.0;
    for (int w = 0; w < warps; w++) sr += dpart[0][w], st += dpart[1][w];
    exchange((float)sr, (float)(sr - (float)sr), (float)st, (float)(st - (float)st));
    sr = st = 0.0;
    for (int q = 0; q < cl; q++) sr += (double)xch[0][q] + xch[1][q], st += (double)xch[2][q] + xch[3][q];
    // S = s 2^(zm c)
    const float zm = fmaxf(mr, mt);
    const double base = zm == -INFINITY ? 0.0 : zm;
    const double s = sr * exp2(((double)mr - base) * c) + st * exp2(((double)mt - base) * c);
    const double log2s = zm == -INFINITY ? 0.0 : log2(s);
    const double log2qr = sr == 0.0 ? -INFINITY : ((double)mr - base) * c + log2(sr) - log2s;
    if (MODE != M_GRAD && rank == 0 && warp == 0) {
        double l = 0.0;
        for (int k = lane; k < K; k += 32)
            if (!(pr[k] == 0.f)) l = __fma_rn(-(double)pr[k], (((double)zk[k] - base) * c - log2s) * LN2_D, l);
        l = warp_sum(l) + sums.plogp;
        if (lane == 0) {
            if (prest > 0.0) l = __fma_rn(prest, __fma_rn(-log2qr, LN2_D, log(prest)), l);
            p.loss[row] = (float)__dmul_rn(w, l);
            // out of range again for the gradient's kernel
            if (p.stats) p.stats[3 * row] = __fmul_rn(zm, c), p.stats[3 * row + 1] = (float)s, p.stats[3 * row + 2] = (float)log2qr;
        }
    }
    if (MODE == M_LOSS) return;
    T* dz = (T*)p.dz + row * p.ld_d;
    const float scale = MODE == M_GRAD ? (p.grad ? p.grad[row * p.s_grad] : 1.f) * w * p.inv_tau : __fmul_rn(w, p.inv_tau);
    const double P = sums.psum + prest, inv = s == 0.0 ? 0.0 : 1.0 / s;
    // outside the slots q_j P - p_r q_j / q_r = (q_r P - p_r) q_j / q_r; a rest that the student gives nothing has q_j = 0 throughout
    const float fr = sr == 0.0 ? 0.f : (float)(scale * (exp2(log2qr) * P - prest) / sr);
    over_rest(sl, id, K, bits, p.bit_words, [&](int j, float z) { dz[j] = from_f<T>(fr * ex2(__fmul_rn(z - rr, c))); });
    for (int k = tid; k < K; k += blockDim.x) {
        if (!counts(k)) continue;
        double pk = pr[k];
        if (sums.dup)
            for (int q = k + 1; q < K; q++)
                if (id[q] == id[k]) pk += pr[q];
        dz[id[k]] = from_f<T>((float)(scale * (P * exp2(((double)zk[k] - base) * c) * inv - pk)));
    }
}

// Losses, and with GRAD their gradients.  A cluster per row, each CTA a slice of it; with GRAD the slice stays in shared memory
// between the two passes, so that the row is read from memory once.  Several small CTAs an SM, not one large one: a row has
// latencies in a chain (its weight, its slots, the sums, the cluster's barrier) and only other rows can fill them.  The last warp
// works on the slots alone, while the others are in their first pass.
// Bound: the logits read once and the gradient written once; an exponential an element and pass (16 a clock and SM) and the
// instructions around it take 60 to 70 % of that time.  4096 x 128256 bf16 with the gradient, a quarter
// of the rows of weight 0: 385 us, 4.8 TB/s; 2048 rows, the loss alone: 98 us, 5.4 TB/s.
template <typename T, bool GRAD, bool REST>
__global__ void __launch_bounds__(D_THREADS + 32, REST && !GRAD ? 5 : 0) distill_rows_kernel(const __grid_constant__ DistillParams p)
{
    constexpr int VEC = 16 / sizeof(T), WARPS = D_THREADS / 32, ALL = D_THREADS + 32;
    __shared__ float red[2][WARPS];
    uint32_t* bits = dsm;
    float* pr = reinterpret_cast<float*>(dsm + p.bit_words + 4 * p.hold);  // u, then p_k
    float* zk = pr + p.K;  // z of the slot's token (slots of the slice; all of them on the first CTA)
    int* id = reinterpret_cast<int*>(zk + p.K);  // token or -1
    const uint32_t held = (uint32_t)__cvta_generic_to_shared(dsm + p.bit_words);
    if (GRAD) next_may_start();

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, K = p.K, V = p.V, cl = p.cl;
    const int rank = cl > 1 ? (int)cluster_rank() : 0;
    const long long row = blockIdx.x / cl;
    const float w = p.weight ? p.weight[row] : 1.f;
    int id0 = -1;
    float u0 = 0.f;
    if (tid < K) load_slot(p, row, tid, id0, u0);  // in flight together with the weight
    if (cl > 1) cluster_arrive_relaxed();          // paired with the wait before the exchange: every CTA of the row has started
    const Slice<T> sl(p, row, rank);
    T* dz = GRAD ? (T*)p.dz + row * p.ld_d : nullptr;
    if (w == 0.f) {  // no loss, no gradient; the logits may be anything
        if (rank == 0 && tid == 0) {
            p.loss[row] = 0.f;
            if (p.stats) p.stats[3 * row] = p.stats[3 * row + 1] = p.stats[3 * row + 2] = 0.f;
        }
        if (GRAD) zero_slice(p, sl, dz, rank, tid, ALL);
        if (cl > 1) cluster_wait();
        return;
    }
    // The slice is on its way to shared memory (each thread copies and later reads its own vectors: no barrier for them) in
    // four batches while the slots are set up.
    const int nvec = sl.v1 - sl.v0, nh = GRAD ? min(nvec, p.hold) : 0;
    const int bt = GRAD ? (nh + 4 * D_THREADS - 1) / (4 * D_THREADS) : 0;  // a thread's vectors in a batch
    const uint4* zt = reinterpret_cast<const uint4*>(sl.z + sl.head) + sl.v0 + tid;
    if (GRAD && tid < D_THREADS) {
#pragma unroll
        for (int b = 0; b < 4; b++) {
            for (int t = b * bt; t < (b + 1) * bt && tid + t * D_THREADS < nh; t++)
                cp16(held + 16 * tid + t * (16 * D_THREADS), zt + t * D_THREADS);
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        }
    }
    const int jb = sl.head + (sl.v0 - 1) * VEC;  // element of bit 0: vector v's bits start at (v - v0 + 1) VEC
    for (int i = tid; i < ((nvec + 2) * VEC + 31) / 32; i += ALL) bits[i] = 0;
    if (tid == 0) sums.dup = 0;
    __syncthreads();
    const float c = (float)(p.inv_tau_d * LOG2E_D);
    for (int k = tid; k < K; k += ALL) {
        if (k != tid) load_slot(p, row, k, id0, u0);
        const bool own = id0 >= 0 && id0 >= sl.j0 && id0 < sl.j1;
        id[k] = id0, pr[k] = u0;
        if (own || (rank == 0 && id0 >= 0)) zk[k] = to_f(sl.z[id0]);
        if (own) {
            const int b = id0 - jb;
            if (atomicOr(&bits[b >> 5], 1u << (b & 31)) >> (b & 31) & 1u) sums.dup = 1;
        }
    }
    __syncthreads();
    const bool any_dup = sums.dup != 0;

    const uint64_t cc = pair(c, c);
    auto held_vec = [&](int t) {
        uint4 u;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n"
                     : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                     : "r"(held + 16 * tid + t * (16 * D_THREADS)));
        return u;
    };
    // this thread's vectors: v0 + tid + t * D_THREADS for t < nt, the first nth of them in shared memory
    const int nt = tid < D_THREADS ? (nvec - tid + D_THREADS - 1) / D_THREADS : 0;
    const int nth = tid < D_THREADS ? max(0, (nh - tid + D_THREADS - 1) / D_THREADS) : 0;

    if (warp < WARPS) {
        // One pass: (m, s) with the running maximum, over the tokens outside the slots.  The slots' tokens, which hold most of
        // the mass, are summed apart and in 64 bits.
        float m = -BIG, s;
        uint64_t s2 = 0;  // two sums, by the elements' parity
        // the bits of this thread's vectors: at a fixed step (and, of four-element vectors, a fixed half of a byte)
        const uint8_t* bytes = reinterpret_cast<const uint8_t*>(bits) + (VEC == 8 ? tid + 1 : (tid + 1) >> 1);
        constexpr int step = VEC == 8 ? D_THREADS : D_THREADS / 2;
        auto masked = [&](uint4 raw, int t) {  // the slots' tokens as -infinity
            const uint32_t by = bytes[t * step], mb = VEC == 8 ? by : by >> (((tid + 1) & 1) * 4) & 15u;
            return mb ? mask16(raw, mb, T()) : raw;
        };
        auto raise = [&](float vm) {  // the running maximum
            if (vm > m) {
                const float f = ex2(m - vm);
                s2 = mul2(s2, pair(f, f));
                m = vm;
            }
        };
        auto sum = [&](const uint4& raw, uint64_t bb) {
            float x[VEC];
            unpack16(raw, x, T());
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
                const float2 e = unpair(fma2(pair(x[i], x[i + 1]), cc, bb));
                s2 = add2(s2, pair(ex2(e.x), ex2(e.y)));
            }
        };
        auto add = [&](uint4 raw, int t) {
            raw = masked(raw, t);
            raise(__fmul_rn(max16(raw, T()), c));
            sum(raw, pair(-m, -m));
        };
        auto add_both = [&](uint4 r0, uint4 r1, int t) {  // vectors t and t + 1, one look at the maximum
            r0 = masked(r0, t), r1 = masked(r1, t + 1);
            raise(__fmul_rn(fmaxf(max16(r0, T()), max16(r1, T())), c));
            const uint64_t bb = pair(-m, -m);
            sum(r0, bb);
            sum(r1, bb);
        };
        int t = 0;
        if (GRAD) {
            cp_wait<3>();
            for (const int e = min(nth, bt); t + 1 < e; t += 2) add_both(held_vec(t), held_vec(t + 1), t);
            cp_wait<2>();
            for (const int e = min(nth, 2 * bt); t + 1 < e; t += 2) add_both(held_vec(t), held_vec(t + 1), t);
            cp_wait<1>();
            for (const int e = min(nth, 3 * bt); t + 1 < e; t += 2) add_both(held_vec(t), held_vec(t + 1), t);
            cp_wait<0>();
            for (; t + 1 < nth; t += 2) add_both(held_vec(t), held_vec(t + 1), t);
            for (; t < nth; t++) add(held_vec(t), t);
        }
        for (; t + 4 <= nt; t += 4) {
            uint4 u[4];
#pragma unroll
            for (int q = 0; q < 4; q++) u[q] = __ldg(zt + (t + q) * D_THREADS);
#pragma unroll
            for (int q = 0; q < 4; q += 2) add_both(u[q], u[q + 1], t + q);
        }
        for (; t + 2 <= nt; t += 2) add_both(__ldg(zt + t * D_THREADS), __ldg(zt + (t + 1) * D_THREADS), t);  // the same pairs as above
        for (; t < nt; t++) add(__ldg(zt + t * D_THREADS), t);
        const float2 e = unpair(s2);
        s = e.x + e.y;
        auto scalar = [&](int j) {
            if (bits[(j - jb) >> 5] >> ((j - jb) & 31) & 1u) return;
            const float z = to_f(sl.z[j]), M = fmaxf(m, __fmul_rn(z, c));
            s = __fmaf_rn(s, ex2(m - M), ex2(__fmaf_rn(z, c, -M)));
            m = M;
        };
        if (rank == 0 && tid < sl.head) scalar(tid);
        if (rank == cl - 1 && sl.tail() + tid < V) scalar(sl.tail() + tid);
        warp_join<32>(m, s);
        if (lane == 0) red[0][warp] = m, red[1][warp] = s;
    } else {  // the slots' sums
        double psum, prest, plogp, t = 0.0;
        teacher_probabilities<REST>(p, REST ? p.lse[row] : 0.f, pr, id, lane, psum, prest, plogp);
        float mt = -BIG;
        auto counts = [&](int k) { return id[k] >= 0 && id[k] >= sl.j0 && id[k] < sl.j1 && (!any_dup || leads(id, k)); };
        for (int k = lane; k < K; k += 32)
            if (counts(k)) mt = fmaxf(mt, __fmul_rn(zk[k], c));
        mt = warp_reduce<0>(mt);
        for (int k = lane; k < K; k += 32)
            if (counts(k)) t += exp2(__fma_rn(zk[k], c, -(double)mt));
        t = warp_sum(t);
        if (lane == 0) {
            sums.psum = (float)psum, sums.prest = (float)prest, sums.mt = mt, sums.st = (float)t;
            sums.plogp = plogp, sums.prest64 = prest;
        }
    }
    __syncthreads();
    const float psum = sums.psum, prest = sums.prest;
    float m = red[0][lane & (WARPS - 1)], s = red[1][lane & (WARPS - 1)], mt = sums.mt, st = sums.st;
    warp_join<WARPS>(m, s);
    if (cl > 1) {
        cluster_wait();
        if (tid < cl) {
            st_cluster_u32(&xch[0][rank], tid, __float_as_uint(m));
            st_cluster_u32(&xch[1][rank], tid, __float_as_uint(s));
            st_cluster_u32(&xch[2][rank], tid, __float_as_uint(mt));
            st_cluster_u32(&xch[3][rank], tid, __float_as_uint(st));
        }
        if (warp == 0) cluster_arrive();
        else cluster_arrive_relaxed();
        cluster_wait();
        const int q = lane & (D_MAXCL - 1);
        m = q < cl ? xch[0][q] : -INFINITY, s = q < cl ? xch[1][q] : 0.f;
        warp_join<D_MAXCL>(m, s);
        mt = q < cl ? xch[2][q] : -INFINITY, st = q < cl ? xch[3][q] : 0.f;
        warp_join<D_MAXCL>(mt, st);
    }
    float ma = m, sa = s;
    join(ma, sa, mt, st);
    // S = sa 2^ma: the two stay apart, for log2 S itself would be rounded to the size of the logits
    const float log2qr = !REST || s == 0.f ? -INFINITY : (m - ma) + (log2f(s) - log2f(sa));
    // the same for all CTAs of the row: a largest logit, or a rest with some of the teacher's mass, outside the exponents' range
    if (!(fabsf(ma) < BIG) || (REST && prest > 0.f && s == 0.f)) {
        if (!GRAD) exact_row<T, REST, M_LOSS>(p, row);
        else if (rank == 0 && tid == 0) p.loss[row] = __uint_as_float(TO_DO);  // by exact_rows_kernel
        return;
    }
    if (rank == 0 && warp == WARPS) {
        double l = 0.0;
        const double shift = (double)ma + log2((double)sa);
        for (int k = lane; k < K; k += 32)
            if (!(pr[k] == 0.f)) l = __fma_rn(-(double)pr[k], __dmul_rn(__fma_rn(zk[k], c, -shift), LN2_D), l);
        l = warp_sum(l) + sums.plogp;
        if (lane == 0) {
            if (sums.prest64 > 0.0) l = __fma_rn(sums.prest64, __fma_rn(-(double)log2qr, LN2_D, log(sums.prest64)), l);
            p.loss[row] = (float)__dmul_rn(w, l);
            if (p.stats) p.stats[3 * row] = ma, p.stats[3 * row + 1] = sa, p.stats[3 * row + 2] = log2qr;
        }
    }
    if (GRAD) {
        GradScale g(__fmul_rn(w, p.inv_tau), psum, prest, ma, sa, log2qr);
        if (REST && prest > 0.f && log2qr < FAR_REST) g.far_rest(psum, prest, log2qr, m, s);
        if (p.vec_out) {
            const uint64_t bb = pair(-g.br, -g.br), rr = pair(g.cr, g.cr);
            uint4* dt = reinterpret_cast<uint4*>(dz + sl.head) + sl.v0 + tid;
            int t = 0;
#pragma unroll 2
            for (; t < nth; t++) __stcs(dt + t * D_THREADS, grad16<T>(held_vec(t), cc, bb, rr));
            // plain loads: the rows may be overwritten (dz = z), each vector by the thread that has read it
#pragma unroll 4
            for (; t < nt; t++) __stcs(dt + t * D_THREADS, grad16<T>(zt[t * D_THREADS], cc, bb, rr));
            auto scalar = [&](int j) { dz[j] = from_f<T>(g.cr * ex2(fmaf(to_f(sl.z[j]), c, -g.br))); };
            if (rank == 0 && tid < sl.head) scalar(tid);
            if (rank == cl - 1 && sl.tail() + tid < V) scalar(sl.tail() + tid);
        } else
            for (int j = sl.j0 + tid; j < sl.j1; j += ALL) dz[j] = from_f<T>(g.cr * ex2(fmaf(to_f(sl.z[j]), c, -g.br)));
        __syncthreads();
        for (int k = tid; k < K; k += ALL) {
            if (id[k] < 0 || id[k] < sl.j0 || id[k] >= sl.j1 || (any_dup && !leads(id, k))) continue;
            float pk = pr[k];
            if (any_dup)
                for (int q = k + 1; q < K; q++)
                    if (id[q] == id[k]) pk += pr[q];
            dz[id[k]] = from_f<T>(__fmaf_rn(g.Pq, ex2(__fmaf_rn(zk[k], c, -g.b)), -__fmul_rn(g.scale, pk)));
        }
    }
}

// The slots of a row into shared memory, and p_k, by a CTA that has the whole row.
template <typename T, bool REST>
__device__ __forceinline__ void load_slots(const DistillParams& p, long long row, const T* z)
{
    const int tid = threadIdx.x, K = p.K;
    float* pr = reinterpret_cast<float*>(dsm + p.bit_words);
    float* zk = pr + K;
    int* id = reinterpret_cast<int*>(zk + K);
    for (int k = tid; k < K; k += blockDim.x) {
        load_slot(p, row, k, id[k], pr[k]);
        if (id[k] >= 0) zk[k] = to_f(z[id[k]]);
    }
    __syncthreads();
    if (tid < 32) {
        double psum, prest, plogp;
        teacher_probabilities<REST>(p, REST ? p.lse[row] : 0.f, pr, id, tid, psum, prest, plogp);
        if (tid == 0) sums.psum = (float)psum, sums.prest = (float)prest, sums.plogp = plogp, sums.prest64 = prest, sums.dup = 1;
    }
    __syncthreads();
}

// 4096 x 128256 bf16 with all rows masked by -1e10 outside the slots: 4.2 ms, 0.46 in range; the gradient alone 2.1 ms against 0.40.
// The rows that the kernel of losses and gradients left to do (their losses hold TO_DO), a CTA each.  A launch of its own, for
// exact_row inside that kernel makes its fast path slower (4096 x 128256 bf16 386 us: 412 as part of it, 400 as a call; the launch
// costs 2); the others carry it at no cost.
template <typename T, bool REST>
__global__ void __launch_bounds__(D_THREADS) exact_rows_kernel(const __grid_constant__ DistillParams p)
{
    __shared__ int found;
    wait_for_previous();
    for (long long r0 = blockIdx.x; r0 < p.T; r0 += (long long)D_THREADS * gridDim.x) {
        const long long mine = r0 + (long long)threadIdx.x * gridDim.x;
        bool todo = mine < p.T && __float_as_uint(p.loss[mine]) == TO_DO;
        while (__syncthreads_or(todo)) {
            if (threadIdx.x == 0) found = D_THREADS;
            __syncthreads();
            if (todo) atomicMin(&found, (int)threadIdx.x);
            __syncthreads();
            const int f = found;
            todo = todo && f != (int)threadIdx.x;
            const long long row = r0 + (long long)f * gridDim.x;
            load_slots<T, REST>(p, row, (const T*)p.z + row * p.ld);
            exact_row<T, REST, M_BOTH>(p, row);
        }
    }
}

// the gradient alone, from the statistics: one pass, a CTA per row.  CTAs an SM as many as before exact_row was part of it: 2048 x
// 128256 bf16 215 us, 226 with the registers that it would take
template <typename T, bool REST>
__global__ void __launch_bounds__(D_THREADS, sizeof(T) == 4 ? 6 : 5) distill_grad_kernel(const __grid_constant__ DistillParams p)
{
    float* pr = reinterpret_cast<float*>(dsm + p.bit_words);
    float* zk = pr + p.K;
    int* id = reinterpret_cast<int*>(zk + p.K);
    const int tid = threadIdx.x, K = p.K, V = p.V;
    const long long row = blockIdx.x;
    const Slice<T> sl(p, row, 0);
    T* dz = (T*)p.dz + row * p.ld_d;
    const float w = p.weight ? p.weight[row] : 1.f;
    if (w == 0.f) {
        zero_slice(p, sl, dz, 0, tid, D_THREADS);
        return;
    }
    const float c = (float)(p.inv_tau_d * LOG2E_D);
    load_slots<T, REST>(p, row, sl.z);
    const float up = p.grad ? p.grad[row * p.s_grad] : 1.f;
    const float scale = up * w * p.inv_tau, ma = p.stats[3 * row], log2qr = p.stats[3 * row + 2];
    if (!(fabsf(ma) < BIG) || (REST && sums.prest > 0.f && log2qr < FAR_REST)) {  // the statistics do not hold the rest's own pair
        exact_row<T, REST, M_GRAD>(p, row);
        return;
    }
    const GradScale g(scale, sums.psum, sums.prest, ma, p.stats[3 * row + 1], log2qr);
    if (p.vec_out) {
        const uint64_t cc = pair(c, c), bb = pair(-g.br, -g.br), rr = pair(g.cr, g.cr);
        // plain loads: the rows may be overwritten (dz = z), each vector by the thread that has read it
        const uint4* zt = reinterpret_cast<const uint4*>(sl.z + sl.head);
        uint4* dt = reinterpret_cast<uint4*>(dz + sl.head);
        int v = tid;
        for (; v + 3 * D_THREADS < sl.nb; v += 4 * D_THREADS) {
            uint4 u[4];
#pragma unroll
            for (int q = 0; q < 4; q++) u[q] = zt[v + q * D_THREADS];
#pragma unroll
            for (int q = 0; q < 4; q++) __stcs(dt + v + q * D_THREADS, grad16<T>(u[q], cc, bb, rr));
        }
        for (; v < sl.nb; v += D_THREADS) __stcs(dt + v, grad16<T>(zt[v], cc, bb, rr));
        auto scalar = [&](int j) { dz[j] = from_f<T>(g.cr * ex2(fmaf(to_f(sl.z[j]), c, -g.br))); };
        if (tid < sl.head) scalar(tid);
        if (sl.tail() + tid < V) scalar(sl.tail() + tid);
    } else
        for (int j = tid; j < V; j += D_THREADS) dz[j] = from_f<T>(g.cr * ex2(fmaf(to_f(sl.z[j]), c, -g.br)));
    __syncthreads();
    for (int k = tid; k < K; k += D_THREADS) {
        if (id[k] < 0 || !leads(id, k)) continue;
        float pk = pr[k];
        for (int q = k + 1; q < K; q++)
            if (id[q] == id[k]) pk += pr[q];
        dz[id[k]] = from_f<T>(__fmaf_rn(g.Pq, ex2(__fmaf_rn(zk[k], c, -g.b)), -__fmul_rn(g.scale, pk)));
    }
}

// CTAs of a row.  With gradient one where the row fits D_ROW (three CTAs an SM and no cluster barrier: 4096 x 32000 fp16 111 us,
// two CTAs of half a row 123 us), else as few as let a slice stay in D_SLICE (four an SM: 4096 x 128256 bf16 384 us with 52 KB
// slices, 397 us with 36, 395 us with 66 KB).  Without gradient one.  Few rows: more, until the GPU's SMs have one each.
int row_ctas(long long T, int V, int es, bool grad)
{
    const long long bytes = (long long)V * es;
    int cl = grad && bytes > D_ROW ? (int)((bytes + D_SLICE - 1) / D_SLICE) : 1;
    while (cl < D_MAXCL && T * cl < 148 && bytes / cl > 16 * 1024) cl *= 2;
    return cl < D_MAXCL ? cl : D_MAXCL;
}

// for kernels whose CTAs have whole rows and hold nothing of them but the slots
constexpr int WHOLE_BITS = 1024;  // words of exact_row's bitmap
void whole_row(DistillParams& p) { p.cl = 1, p.bit_words = WHOLE_BITS, p.hold = 0; }
int slots_smem(int K) { return WHOLE_BITS * 4 + K * 12; }

template <typename T, bool GRAD, bool REST>
int launch_rows(DistillParams p, cudaStream_t st)
{
    constexpr int VEC = 16 / sizeof(T);
    auto k = distill_rows_kernel<T, GRAD, REST>;
    p.cl = row_ctas(p.T, p.V, sizeof(T), GRAD);
    const int per = (p.V / VEC + p.cl - 1) / p.cl;
    // whole 256 bytes: 1024 x 128256 fp32 226 us, up to 250 when the held slice behind them begins elsewhere
    p.bit_words = (((per + 2) * VEC + 31) / 32 + MIN_BIT_WORDS - 1) / MIN_BIT_WORDS * MIN_BIT_WORDS;
    const int fixed = p.bit_words * 4 + p.K * 12;
    p.hold = GRAD ? per : 0;
    if (fixed + p.hold * 16 > D_SMEM) p.hold = (D_SMEM - fixed) / 16;
    const int smem = fixed + p.hold * 16;
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
    cfg.gridDim = dim3((unsigned)((long long)p.T * p.cl));
    cfg.blockDim = dim3(D_THREADS + 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)p.cl, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = p.cl > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, k, p);
    if (!GRAD || e != cudaSuccess) return (int)e;
    whole_row(p);
    return (int)launch_next(exact_rows_kernel<T, REST>, std::min(p.T, 296), D_THREADS, slots_smem(p.K), st, p);
}

template <typename T, bool REST>
int launch_grad(DistillParams p, cudaStream_t st)
{
    whole_row(p);
    distill_grad_kernel<T, REST><<<p.T, D_THREADS, slots_smem(p.K), st>>>(p);
    return (int)cudaGetLastError();
}

template <typename T>
int dispatch(const DistillParams& p, int mode, cudaStream_t st)
{
    const bool rest = p.lse != nullptr;
    if (mode == M_LOSS) return rest ? launch_rows<T, false, true>(p, st) : launch_rows<T, false, false>(p, st);
    if (mode == M_BOTH) return rest ? launch_rows<T, true, true>(p, st) : launch_rows<T, true, false>(p, st);
    return rest ? launch_grad<T, true>(p, st) : launch_grad<T, false>(p, st);
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
    p.T = T, p.V = V, p.K = K, p.idx64 = idx64 != 0, p.u_dt = teacher_dtype, p.inv_tau = 1.f / temperature, p.inv_tau_d = 1.0 / temperature;
    p.vec_out = mode != M_LOSS && ((uintptr_t)logits & 15) == ((uintptr_t)dlogits & 15) && ((ld - ld_d) * es) % 16 == 0;
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F32) return dispatch<float>(p, mode, st);
    if (dtype == DT_BF16) return dispatch<__nv_bfloat16>(p, mode, st);
    return dispatch<__half>(p, mode, st);
}
