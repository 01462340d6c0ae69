// The tensor cores of sm_100a and what feeds them, in PTX: barriers in shared memory, tiled copies, tensor memory and
// tcgen05 products.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace mtxc {

__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// True in one thread of a converged warp, the same one each time.  Behind a comparison of lanes a product took 125 to 160
// cycles to issue, behind this about 40.
__device__ __forceinline__ bool elected() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// ------------------------------------------------------------------------------------------
// Barriers
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {  // the hardware waits a while itself
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
// Waits for the phase of this parity to end.  Where it does not within some seconds (2^20 tries, which take 4 us each), *failed
// is set, and no thread waits for anything any more: the block runs to its end, with outputs that count for nothing.  False: the
// phase has not ended.
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, volatile int* failed) {
    if (barrier_try(bar, parity)) return true;
    for (uint32_t i = 0; i < 1u << 20; ++i) {
        if (barrier_try(bar, parity)) return true;
        if (*failed) return false;
    }
    *failed = 1;
    return false;
}
// What threads have written to shared memory becomes visible to copies and products.
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ------------------------------------------------------------------------------------------
// Tiled copies (three axes)
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ void copy_tile(uint32_t to, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(to),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// ------------------------------------------------------------------------------------------
// Tensor memory: 128 lanes (bits 16 and up of an address) x 512 columns of 32 bits; warp w of a group of four reaches
// lanes 32 w .. 32 w + 31.
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ void tensor_alloc(uint32_t to, uint32_t columns) {  // a whole warp
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tensor_free(uint32_t address, uint32_t columns) {  // a whole warp
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
}
__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tensor_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define MTX_REGS32(c, v, o)                                                                                              \
    c((v)[(o) + 0]), c((v)[(o) + 1]), c((v)[(o) + 2]), c((v)[(o) + 3]), c((v)[(o) + 4]), c((v)[(o) + 5]), c((v)[(o) + 6]),  \
        c((v)[(o) + 7]), c((v)[(o) + 8]), c((v)[(o) + 9]), c((v)[(o) + 10]), c((v)[(o) + 11]), c((v)[(o) + 12]),           \
        c((v)[(o) + 13]), c((v)[(o) + 14]), c((v)[(o) + 15]), c((v)[(o) + 16]), c((v)[(o) + 17]), c((v)[(o) + 18]),        \
        c((v)[(o) + 19]), c((v)[(o) + 20]), c((v)[(o) + 21]), c((v)[(o) + 22]), c((v)[(o) + 23]), c((v)[(o) + 24]),        \
        c((v)[(o) + 25]), c((v)[(o) + 26]), c((v)[(o) + 27]), c((v)[(o) + 28]), c((v)[(o) + 29]), c((v)[(o) + 30]),        \
        c((v)[(o) + 31])
#define MTX_LIST32                                                                                                       \
    "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, " \
    "%25, %26, %27, %28, %29, %30, %31}"

// 32 columns of this thread's lane; valid after tensor_wait_load.
template <int N>
__device__ __forceinline__ void tensor_load32(uint32_t address, float (&v)[N], int at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 " MTX_LIST32 ", [%32];" : MTX_REGS32("=f", v, at) : "r"(address));
}
template <int N>
__device__ __forceinline__ void tensor_store32(uint32_t address, const float (&v)[N], int at) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], " MTX_LIST32 ";" ::MTX_REGS32("f", v, at), "r"(address) : "memory");
}
template <int N>
__device__ __forceinline__ void tensor_store32(uint32_t address, const uint32_t (&v)[N], int at) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], " MTX_LIST32 ";" ::MTX_REGS32("r", v, at), "r"(address) : "memory");
}

// ------------------------------------------------------------------------------------------
// Products of half types, accumulated in 32 bits
// ------------------------------------------------------------------------------------------
// A tile in shared memory, of rows of 128 bytes with their 16-byte units swapped by the row (as a tiled copy with the
// 128-byte swizzle leaves it), eight rows in 1,024 bytes: `step` bytes from eight rows to the next, `wide` from 128 bytes
// of a row to the next (where the rows, and not the columns, are summed over).
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t address, uint32_t step, uint32_t wide) {
    return (uint64_t)(address >> 4 & 0x3FFF) | (uint64_t)(wide >> 4 & 0x3FFF) << 16 | (uint64_t)(step >> 4 & 0x3FFF) << 32 |
           1ull << 46 | 2ull << 61;
}
// What a product of m x n x 16 is: the operands' type, and whether the second one's rows are what is summed over.
constexpr uint32_t product_descriptor(bool bf16, int m, int n, bool rows_summed) {
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (rows_summed ? 1u << 16 : 0u) | (uint32_t)(n / 8) << 17 | (uint32_t)(m / 16) << 24;
}
// One thread; both operands in shared memory.
__device__ __forceinline__ void product(uint32_t to, uint64_t a, uint64_t b, uint32_t what, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(to),
        "l"(a), "l"(b), "r"(what), "r"((uint32_t)add)
        : "memory");
}
// The first operand in tensor memory, two elements a column.
__device__ __forceinline__ void product(uint32_t to, uint32_t a, uint64_t b, uint32_t what, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(to),
        "r"(a), "l"(b), "r"(what), "r"((uint32_t)add)
        : "memory");
}
// The barrier is arrived at when all products that this thread has issued are done.
__device__ __forceinline__ void product_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

template <int N>
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN where one of them is
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace mtxc
