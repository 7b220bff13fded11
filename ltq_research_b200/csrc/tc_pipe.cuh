// Building blocks of the tensor-core pipelines (sm_100a): mbarriers with bounded waits, TMA loads, operand descriptors of
// tcgen05.mma, reads of tensor memory.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <atomic>

namespace {

constexpr uint32_t GEMM_WAIT_LIMIT = 1u << 26;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint64_t* b, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* b, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* b, uint32_t parity)
{
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
// bounded wait for the phase with parity `parity`; false after `limit` polls (the timeout is recorded in *err)
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, int* err, uint32_t limit = GEMM_WAIT_LIMIT)
{
    for (uint32_t i = 0; i < limit; i++)
        if (mbar_try_wait(b, parity)) return true;
    if (err) atomicExch(err, 1);
    return false;
}
// The same for a whole warp, with one answer for all of its lanes: a phase may end between two lanes' last polls, and lanes that
// went different ways would wait without limit at the next instruction of the whole warp (shfl, elect, tcgen05.ld).  A vote a poll
// keeps the loop uniform; 8192 x 8192 x 4096 in 8 bits: 267 us (311 back to back), 257 (308) with lanes that poll each for themselves;
// 366 back to back with these joined after the loop (the epilogue spills then).
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* b, uint32_t parity, int* err, uint32_t limit = GEMM_WAIT_LIMIT)
{
    for (uint32_t i = 0; i < limit; i++)
        if (__all_sync(0xffffffffu, mbar_try_wait(b, parity))) return true;
    if (err) atomicExch(err, 1);
    return false;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}

// shared-memory matrix descriptor (tcgen05): K-major tile of rows x 64 bf16 with the 128-byte swizzle, as TMA writes it:
// 8-row atoms of 1024 bytes one after the other (stride byte offset 1024), the second 16-byte column chunk adjacent
// (leading byte offset 16), descriptor version 1, layout 2 (128-byte swizzle).  `addr` may step through the atom's
// row in 32-byte units (one K = 16 slice of bf16), the hardware applying the swizzle to the computed address.
__device__ __forceinline__ uint64_t sw128_kmajor_desc(uint32_t addr)
{
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ void umma_commit(uint64_t* bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16])
{
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn()
{
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> fn{nullptr};
    PFN_cuTensorMapEncodeTiled_v12000 f = fn.load(std::memory_order_acquire);
    // the encoder is a driver call: a thread whose first CUDA call it is (autograd's, say) has no context current yet
    static thread_local bool bound = false;
    if (!bound) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return nullptr;
        bound = true;
    }
    if (!f) {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return nullptr;
        f = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
        fn.store(f, std::memory_order_release);
    }
    return f;
}

}  // namespace
