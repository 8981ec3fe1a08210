// tcgen05 in the few forms that the attention kernels use: 16-bit operands, fp32 accumulators of 128 rows in tensor memory.
//
// Operand tiles lie in shared memory as blocks of rows of 64 values (128 bytes) whose 16-byte pieces are exchanged by the row's lower
// three bits (the 128-byte swizzle).  The same block serves as an operand whose rows are summed over (values contiguous along the sum,
// "K-major") and as one whose columns are ("MN-major"): only the descriptor differs.
#pragma once

#include <stdint.h>

#include "lutgemm_waits.cuh"

namespace lutgemm {

// One lane of a whole warp.  Products are issued from `if (elect_one())` in code that the warp enters together, with the operand sizes as
// constants: the compiler then keeps their operands in uniform registers.  128 x 64 x 16 products take 33 clocks (first operand
// from tensor memory) and 49 (from shared memory) that way, 94 from `if (lane == 0)`.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// this thread's warp, the same register for all its lanes
__device__ __forceinline__ int warp_index() { return __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0); }

// ---- tensor memory ----------------------------------------------------------------------------------------------------
// by one warp; the address of `columns` (a power of two from 32 on) goes to *slot in shared memory
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}
__device__ __forceinline__ void tmem_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_loads_done() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_stores_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this thread's row (the warp's 32 rows are lanes 32 * (warp % 4) on; the address carries that offset)
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
        "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
          "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
          "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
          "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
          "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const float (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
        "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]),
        "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// ---- products ------------------------------------------------------------------------------------------------------------
// Descriptor of an operand in shared memory, 128-byte swizzle.  K-major: eight rows (of 128 bytes) lie `step` = 1024 bytes apart and
// a block is 64 values of the sum.  MN-major: eight rows of the sum lie 1024 bytes apart, blocks of 64 values of the other axis
// `block` bytes.
__device__ __forceinline__ uint64_t smem_descriptor(uint32_t addr, uint32_t block) {
    return (uint64_t)((addr & 0x3ffffu) >> 4) | (uint64_t)(block >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// the descriptor of the operand `bytes` further on (a product's operands lie at fixed distances from the first: one thread issues them all, and
// building every descriptor anew would take longer than the products)
__device__ __forceinline__ uint64_t descriptor_at(uint64_t descriptor, uint32_t bytes) { return descriptor + (bytes >> 4); }
// 128 x N products of two operands of one 16-bit type into fp32; `b_mn`: the second operand is MN-major
constexpr uint32_t mma_descriptor(bool bf16, int N, bool b_mn) {
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (b_mn ? 1u << 16 : 0u) | (uint32_t)(N >> 3) << 17 | (128u >> 4) << 24;
}
// both from shared memory; one thread
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
        : "memory");
}
// the first from tensor memory (two values to a 32-bit column)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
        : "memory");
}
// the barrier takes one arrival when every product issued so far by this thread is done
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// ---- copies into shared memory ---------------------------------------------------------------------------------------------
// 16 bytes, or zeros
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// what this thread wrote to shared memory is seen by the tensor cores
__device__ __forceinline__ void writes_to_tensor_cores() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

}  // namespace lutgemm
