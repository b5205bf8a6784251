// Instructions of sm_100a that C++ has no words for, as the attention kernels use them: mbarriers, tensor copies into shared memory,
// matrix products with accumulators in tensor memory (TMEM).
//
// Operand tiles in shared memory are panels of 64 columns of 16 bits: rows of 128 bytes with the 128-byte swizzle that the tensor
// copy writes, 8 rows = 1024 bytes = one swizzle atom.  A panel [rows][64] serves both ways:
//   "K-major", the 64 columns are summed over:   16 columns further = 32 bytes, 8 rows further = 1024 bytes
//   "MN-major", the rows are summed over:        16 rows further = 2048 bytes, the next 64 columns = the next panel
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace rode {

#ifdef __CUDACC__

__device__ __forceinline__ uint32_t shared_address(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// --- mbarriers ------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_init_done() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
// Waits for the phase of this parity, for about two seconds at most; false: given up.  By whole warps, whose lanes are together again behind the branch.
// (A __syncwarp or a vote here costs 4 % of forward_tiles.)
//
// A wait tells phases apart by their parity alone, so that no waiter may fall two phases behind: for every barrier here, the phase after the next one
// needs the waiter's own progress.
constexpr long long kWaitClocks = 1ll << 32;
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity) {
    bool done = barrier_try(bar, parity);
    if (!done) {
        const long long start = clock64();
        do done = barrier_try(bar, parity);
        while (!done && clock64() - start < kWaitClocks);
    }
    return done;
}

// Writes of this thread to shared memory become visible to tensor copies and matrix products.
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// --- tensor copies --------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// --- tensor memory --------------------------------------------------------------------------------------------------------------

// One warp; the address is written to shared memory.
__device__ __forceinline__ void tmem_alloc(uint32_t where, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t address, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of the thread's own lane (warp w of a warpgroup: lanes 32 (w % 4) and up, which the address names).
#define RODE_R32(r, o)                                                                                                            \
    "=r"(r[o + 0]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]),               \
        "=r"(r[o + 7]), "=r"(r[o + 8]), "=r"(r[o + 9]), "=r"(r[o + 10]), "=r"(r[o + 11]), "=r"(r[o + 12]), "=r"(r[o + 13]),       \
        "=r"(r[o + 14]), "=r"(r[o + 15]), "=r"(r[o + 16]), "=r"(r[o + 17]), "=r"(r[o + 18]), "=r"(r[o + 19]), "=r"(r[o + 20]),    \
        "=r"(r[o + 21]), "=r"(r[o + 22]), "=r"(r[o + 23]), "=r"(r[o + 24]), "=r"(r[o + 25]), "=r"(r[o + 26]), "=r"(r[o + 27]),    \
        "=r"(r[o + 28]), "=r"(r[o + 29]), "=r"(r[o + 30]), "=r"(r[o + 31])
#define RODE_W32(r, o)                                                                                                            \
    "r"(r[o + 0]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7]),       \
        "r"(r[o + 8]), "r"(r[o + 9]), "r"(r[o + 10]), "r"(r[o + 11]), "r"(r[o + 12]), "r"(r[o + 13]), "r"(r[o + 14]),             \
        "r"(r[o + 15]), "r"(r[o + 16]), "r"(r[o + 17]), "r"(r[o + 18]), "r"(r[o + 19]), "r"(r[o + 20]), "r"(r[o + 21]),           \
        "r"(r[o + 22]), "r"(r[o + 23]), "r"(r[o + 24]), "r"(r[o + 25]), "r"(r[o + 26]), "r"(r[o + 27]), "r"(r[o + 28]),           \
        "r"(r[o + 29]), "r"(r[o + 30]), "r"(r[o + 31])
// registers o .. o + 31 of r
template <int o, int n>
__device__ __forceinline__ void tmem_load32(uint32_t address, uint32_t (&r)[n]) {
    static_assert(o + 32 <= n, "32 registers");
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : RODE_R32(r, o)
        : "r"(address));
}
// Waits for the thread's loads.  The registers pass through it, so that nothing that uses them can be moved in front of it.
#define RODE_RW32(r, o)                                                                                                           \
    "+r"(r[o + 0]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), "+r"(r[o + 5]), "+r"(r[o + 6]),               \
        "+r"(r[o + 7]), "+r"(r[o + 8]), "+r"(r[o + 9]), "+r"(r[o + 10]), "+r"(r[o + 11]), "+r"(r[o + 12]), "+r"(r[o + 13]),       \
        "+r"(r[o + 14]), "+r"(r[o + 15]), "+r"(r[o + 16]), "+r"(r[o + 17]), "+r"(r[o + 18]), "+r"(r[o + 19]), "+r"(r[o + 20]),    \
        "+r"(r[o + 21]), "+r"(r[o + 22]), "+r"(r[o + 23]), "+r"(r[o + 24]), "+r"(r[o + 25]), "+r"(r[o + 26]), "+r"(r[o + 27]),    \
        "+r"(r[o + 28]), "+r"(r[o + 29]), "+r"(r[o + 30]), "+r"(r[o + 31])
template <int o, int n>
__device__ __forceinline__ void tmem_wait_load32(uint32_t (&r)[n]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : RODE_RW32(r, o)::"memory");
}
template <int o, int n>
__device__ __forceinline__ void tmem_store32(uint32_t address, const uint32_t (&r)[n]) {
    static_assert(o + 32 <= n, "32 registers");
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::RODE_W32(r, o),
        "r"(address)
        : "memory");
}

// The same with 16 columns.
#define RODE_W16(r, o)                                                                                                            \
    "r"(r[o + 0]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7]),       \
        "r"(r[o + 8]), "r"(r[o + 9]), "r"(r[o + 10]), "r"(r[o + 11]), "r"(r[o + 12]), "r"(r[o + 13]), "r"(r[o + 14]), "r"(r[o + 15])
template <int o, int n>
__device__ __forceinline__ void tmem_store16(uint32_t address, const uint32_t (&r)[n]) {
    static_assert(o + 16 <= n, "16 registers");
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::RODE_W16(
            r, o),
        "r"(address)
        : "memory");
}

// --- matrix products ------------------------------------------------------------------------------------------------------------

// Descriptor of an operand tile in shared memory: address, distance of the panels (MN-major only) and of the 8-row groups in units of
// 16 bytes, constant 1 in bits 46-48, 128-byte swizzle.
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t address, uint32_t panel_bytes) {
    return static_cast<uint64_t>((address >> 4) & 0x3fff) | static_cast<uint64_t>((panel_bytes >> 4) & 0x3fff) << 16 |
           static_cast<uint64_t>(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// 128 x n product of two operands of one 16-bit type into 32-bit accumulators; b_rows: the rows of b's tile are summed over.
template <typename T>
__device__ __forceinline__ uint32_t product_descriptor(int n, bool b_rows) {
    const uint32_t type = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return 1u << 4 | type << 7 | type << 10 | (b_rows ? 1u << 16 : 0u) | static_cast<uint32_t>(n >> 3) << 17 | (128u >> 4) << 24;
}

// One thread of a warp issues products and their arrivals.  The whole warp runs the code, with its operands in uniform registers, and the
// instruction is predicated on the elected thread: 64 clocks per 128 x 128 x 16 product, the tensor core's own time, where code
// behind a branch on the lane took 70 (128 x 64: 37 instead of 72).
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t one;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one;
}
// d (+)= a b over 16 summands; a in shared memory, or in tensor memory (two elements per column).
__device__ __forceinline__ void product(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(
            d),
        "l"(a), "l"(b), "r"(shape), "r"(static_cast<uint32_t>(add)), "r"(one)
        : "memory");
}
__device__ __forceinline__ void product_from_tmem(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, "
        "p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(shape), "r"(static_cast<uint32_t>(add)), "r"(one)
        : "memory");
}
// The barrier gets one arrival when all products that this thread has issued are complete.
__device__ __forceinline__ void products_arrive(uint32_t one, uint32_t bar) {
    asm volatile(
        "{\n.reg .pred q;\nsetp.ne.b32 q, %1, 0;\n@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar),
        "r"(one)
        : "memory");
}
// The value of lane 0, for the compiler to know that it is the same in all lanes.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }

// Two numbers rounded to the 16-bit type, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    uint32_t r;
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

#endif  // __CUDACC__

}  // namespace rode
