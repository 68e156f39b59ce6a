// Fifth-generation tensor cores: what the kernels that issue tcgen05 instructions share (barriers with
// bounded waits, descriptors, tensor-memory loads, tensor maps).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <string>

#include "../../include/lokiscan.h"
#include "lk_common.cuh"

namespace lk {

constexpr long long GWAIT_CLOCKS = 4000000000ll;  // ~2 s at 2 GHz

__device__ __forceinline__ unsigned g_smem(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void g_mbar_init(unsigned long long *bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(g_smem(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void g_mbar_expect_tx(unsigned long long *bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(g_smem(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void g_mbar_arrive(unsigned long long *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(g_smem(bar)) : "memory");
}
// Bounded wait for the phase with the given parity; false when the clock ran out or
// another role of this CTA has already given up.
__device__ __forceinline__ bool g_mbar_wait(unsigned long long *bar, unsigned parity, volatile int *cta_failed) {
    {   // usually the phase is already complete: no clock read on that path
        unsigned ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(g_smem(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
    }
    const long long t0 = clock64();
    for (;;) {
        // the thread sleeps inside the instruction until the phase completes or the hint (in ns) runs
        // out: a waiting role issues next to nothing and leaves shared memory to the tensor core
        unsigned ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(g_smem(bar)), "r"(parity), "r"(4000u)
            : "memory");
        if (ok) return true;
        if (*cta_failed != 0 || clock64() - t0 > GWAIT_CLOCKS) {
            *cta_failed = 1;
            return false;
        }
    }
}
// The whole (converged) warp waits for a phase, but only lane 0 polls the barrier: 18 warps of
// pollers would compete with the MMAs' operand reads for shared memory.
__device__ __forceinline__ bool g_mbar_wait_warp(unsigned long long *bar, unsigned parity, volatile int *cta_failed) {
    int ok = 0;
    if ((threadIdx.x & 31) == 0) ok = g_mbar_wait(bar, parity, cta_failed) ? 1 : 0;
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}
// One lane of the (converged) warp: the issuer of a single-thread instruction.
__device__ __forceinline__ bool g_elect_one() {
    unsigned pred;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(pred));
    return pred != 0;
}
// Address of `local` (a shared-memory address of this CTA) as it sits in the pair's leader CTA.
__device__ __forceinline__ unsigned g_leader_addr(unsigned local) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(local));
    return r;
}
__device__ __forceinline__ unsigned g_cta_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// One arrival on a barrier of the leader CTA (which may be this CTA).
__device__ __forceinline__ void g_mbar_arrive_leader(unsigned long long *bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(g_leader_addr(g_smem(bar))) : "memory");
}
// All threads of both CTAs of the pair.
__device__ __forceinline__ void g_pair_sync() {
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
// Shared-memory matrix descriptor: K-major operand, 128-byte swizzle, 8-row groups 1024 B apart.
__device__ __forceinline__ unsigned long long g_smem_desc(unsigned addr) {
    unsigned long long d = 0;
    d |= (unsigned long long)((addr & 0x3ffffu) >> 4);        // start address
    d |= (unsigned long long)1 << 16;                          // leading byte offset (unused with swizzle)
    d |= (unsigned long long)(1024 >> 4) << 32;                // stride byte offset between 8-row groups
    d |= (unsigned long long)1 << 46;                          // descriptor version
    d |= (unsigned long long)2 << 61;                          // SWIZZLE_128B
    return d;
}
// Arrive on the barrier at this address in BOTH CTAs of the pair once the MMAs issued so far are done.
__device__ __forceinline__ void g_mma_commit(unsigned long long *bar) {
    const unsigned short both = 3;
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     g_smem(bar)),
                 "h"(both)
                 : "memory");
}
__device__ __forceinline__ void g_tmem_ld32(unsigned taddr, int (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (no link against libcuda)
typedef CUresult (*encode_fn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                              const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline encode_fn get_encode() {
    static const encode_fn fn = [] {  // looked up once; threads that come meanwhile wait for it
        void *p = nullptr;
        cudaDriverEntryPointQueryResult qr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr) != cudaSuccess) {
            cudaGetLastError();
            return encode_fn(nullptr);
        }
        return qr == cudaDriverEntryPointSuccess ? reinterpret_cast<encode_fn>(p) : encode_fn(nullptr);
    }();
    return fn;
}

// rows x row_bytes, rows `stride` bytes apart (a multiple of 16, like the base): boxes of box_rows rows x 128
// bytes, 128-byte swizzle; what lies outside reads as zero, the end of a row to the byte.
inline int encode_rows(CUtensorMap *tm, const void *base, long long rows, long long row_bytes, long long stride, int box_rows) {
    encode_fn enc = get_encode();
    if (!enc) return fail(LK_ECUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t dims[2] = {(cuuint64_t)row_bytes, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LK_ECUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
    return 0;
}

}  // namespace lk
