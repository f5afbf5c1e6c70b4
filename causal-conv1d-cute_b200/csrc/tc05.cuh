// 5th-generation tensor core (tcgen05) and mbarrier primitives for sm_100a, as inline PTX.
//
// Shared-memory operand images are rows of 128 (or 64) bytes whose 16-byte units are permuted
// within groups of eight rows: unit u of row r lies at u ^ (r & 7) (u ^ ((r >> 1) & 3) for 64-byte
// rows). The same bytes serve as a K-major operand (rows along M or N) or an MN-major one (rows
// along K), by the descriptor and the major bits of the instruction descriptor alone.
#pragma once

#include <cuda.h>  // CUtensorMap

#include "common.cuh"

namespace cc1d {

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}

// ---------------------------------------------------------------------------------------- barriers

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
// One arrival, announcing bytes that bulk copies will bring.
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
                 : "memory");
}
// Wait until the phase of the given parity has completed, for limit_ns at most. When one wait of the
// CTA has run out, *abort is set and every later wait returns at once, so that the CTA runs to its end:
// it starts no further copy, waits for what is in flight (drain), says that its results are invalid and
// frees its TMEM.
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
static __device__ __noinline__ void mbar_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort,
                                                   int64_t limit_ns) {
    unsigned long long start, now;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(start));
    while (!*abort) {
        for (int i = 0; i < 64; ++i)
            if (mbar_try(bar, parity)) return;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
        if (now - start > (unsigned long long)limit_ns) *abort = 1;
    }
}
__device__ __forceinline__ void mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort,
                                          int64_t limit_ns) {
    for (int i = 0; i < 16; ++i)
        if (mbar_try(bar, parity)) return;
    mbar_wait_slow(bar, parity, abort, limit_ns);
}
// Barrier of `threads` threads (whole warps) of the CTA.
__device__ __forceinline__ void named_sync(int id, int threads) {
    __syncwarp();
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// Makes this thread's shared-memory writes visible to the tensor core.
__device__ __forceinline__ void fence_async_smem() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// One box of a tensor map at (x, y, z) into shared memory, counted on the mbarrier.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                         uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

// `bytes` contiguous bytes (a multiple of 16, both sides 16-byte aligned) into shared memory.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
        "l"(src), "r"(bytes), "r"(bar)
        : "memory");
}

// -------------------------------------------------------------------------------- tensor memory

__device__ __forceinline__ void tmem_alloc(uint32_t smem_result, int columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_result),
                 "r"(columns)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t tmem, int columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns)
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// 16 fp32 columns of the warp's 32 lanes: lane l of the warp gets row l. The address carries the
// warp's first lane in its upper half. The load and its wait are one statement, so that no use of
// the registers can come before it.
#define CC1D_LD16(first, addr)                                                                \
    "tcgen05.ld.sync.aligned.32x32b.x16.b32 {" first "}, [" addr "];\n\t"
#define CC1D_16REGS(r)                                                                           \
    "=f"((r)[0].x), "=f"((r)[0].y), "=f"((r)[1].x), "=f"((r)[1].y), "=f"((r)[2].x),              \
        "=f"((r)[2].y), "=f"((r)[3].x), "=f"((r)[3].y), "=f"((r)[4].x), "=f"((r)[4].y),          \
        "=f"((r)[5].x), "=f"((r)[5].y), "=f"((r)[6].x), "=f"((r)[6].y), "=f"((r)[7].x),          \
        "=f"((r)[7].y)
#define CC1D_R0 "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15"

__device__ __forceinline__ void tmem_ld16(uint32_t t0, float2* f) {
    __syncwarp();
    asm volatile(CC1D_LD16(CC1D_R0, "%16") "tcgen05.wait::ld.sync.aligned;"
                 : CC1D_16REGS(f)
                 : "r"(t0)
                 : "memory");
}
// The same without the wait: after tmem_wait_ld() and tmem_ready() of each the values may be used.
__device__ __forceinline__ void tmem_ld16_async(uint32_t t0, float2* f) {
    __syncwarp();
    asm volatile(CC1D_LD16(CC1D_R0, "%16") : CC1D_16REGS(f) : "r"(t0) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// Keeps uses of the registers behind the wait that stands before it.
__device__ __forceinline__ void tmem_ready(float2* f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+f"(f[i].x), "+f"(f[i].y));
}
__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// ------------------------------------------------------------------------------------------ MMA

enum : uint64_t { kSwizzle128 = 2, kSwizzle64 = 4 };

// Operand descriptor: start address, byte offset between 64-element atoms along MN (MN-major
// operands wider than one atom), byte offset between groups of eight rows, row swizzle.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t atom, uint32_t group,
                                            uint64_t swizzle) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(atom >> 4) << 16) |
           ((uint64_t)(group >> 4) << 32) | (1ull << 46) | (swizzle << 61);
}

// Instruction descriptor: bf16 x bf16 -> fp32, M = 128.
__host__ __device__ constexpr uint32_t mma_desc(int n, bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) |
           ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

// D (TMEM, fp32) (+)= A B for one K step of 16; one thread issues it.
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t desc,
                                         bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
// kSteps K steps, the operands' descriptors moving on by kA and kB 16-byte units. Unrolled: with
// the descriptors at fixed offsets a step issues in 46 cycles, in a loop it took above 100.
template <int kSteps, int kA, int kB>
__device__ __forceinline__ void mma_steps(uint32_t d, uint64_t a, uint64_t b, uint32_t desc,
                                          bool accumulate) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) mma_bf16(d, a + i * kA, b + i * kB, desc, accumulate || i > 0);
}
// The same with A in tensor memory: 128 lanes, a row of M each, two K elements to a column.
__device__ __forceinline__ void mma_bf16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc,
                                            bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(desc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
template <int kSteps, int kB>
__device__ __forceinline__ void mma_steps_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc,
                                             bool accumulate) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) mma_bf16_ts(d, a + i * 8, b + i * kB, desc, accumulate || i > 0);
}
// Arrive on the mbarrier when all MMAs this thread has issued so far are complete.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
        : "memory");
}

// ----------------------------------------------------------------------------- three-part bf16

// x minus the bf16 pair h, exactly: the products with -1 are exact and so is the difference, as h is
// within an ulp of x. One mixed-precision FMA each (the shift and mask that widen a half would be
// two more instructions on the half-rate integer pipe).
__device__ __forceinline__ float2 rest2(float2 x, uint32_t h) {
    float2 r;
    asm("{\n\t.reg .b16 l, h, m;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "mov.b16 m, 0xbf80;\n\t"  // -1
        "fma.rn.f32.bf16 %0, l, m, %3;\n\t"
        "fma.rn.f32.bf16 %1, h, m, %4;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "r"(h), "f"(x.x), "f"(x.y));
    return r;
}
__device__ __forceinline__ uint32_t bf16x2(float2 f) {
    uint32_t v;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(f.y), "f"(f.x));
    return v;
}
// Two values as two bf16 pairs, within 2^-17 of them: exact for fp16 values (11 bits).
__device__ __forceinline__ void split2(float2 f, uint32_t& hi, uint32_t& lo) {
    hi = bf16x2(f);
    lo = bf16x2(rest2(f, hi));
}
// Two values as three bf16 pairs, whose sum holds the 24 bits of fp32: 8 bits and a sign each.
// The low halves hold f.x.
__device__ __forceinline__ void split3(float2 f, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
    p0 = bf16x2(f);
    f = rest2(f, p0);
    p1 = bf16x2(f);
    p2 = bf16x2(rest2(f, p1));
}
// A pair of T (bf16 or fp16) plus two fp32 values.
template <typename T>
__device__ __forceinline__ float2 add_pair(uint32_t v, float2 f) {
    float2 r;
    if constexpr (std::is_same<T, f16>::value) {
        asm("{\n\t.reg .b16 l, h;\n\t"
            "mov.b32 {l, h}, %2;\n\t"
            "add.rn.f32.f16 %0, l, %3;\n\t"
            "add.rn.f32.f16 %1, h, %4;\n\t}"
            : "=f"(r.x), "=f"(r.y)
            : "r"(v), "f"(f.x), "f"(f.y));
        return r;
    }
    asm("{\n\t.reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "add.rn.f32.bf16 %0, l, %3;\n\t"
        "add.rn.f32.bf16 %1, h, %4;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "r"(v), "f"(f.x), "f"(f.y));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

}  // namespace cc1d
