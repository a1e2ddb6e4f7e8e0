// PTX of sm_100a that the operators use: mbarriers with bounded waits, TMA tile loads, and fifth-generation tensor cores.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "number_types.cuh"

namespace ptwm {

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// One try suspends the thread for up to 20 us.
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity), "r"(20000u) : "memory");
    return done != 0;
}
__device__ __forceinline__ uint64_t nanoseconds() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Waits are bounded: one that lasts for two seconds raises *failed (shared memory), after which every wait of the block returns at once.
constexpr uint64_t WAIT_NS = 2000000000ull;
constexpr uint32_t WAIT_TRIES = 1u << 24;  // in case that clock stands still
__device__ __noinline__ bool mbar_wait_long(uint32_t bar, uint32_t parity, volatile uint32_t* failed) {
    const uint64_t began = nanoseconds();
    for (uint32_t i = 0; !mbar_try(bar, parity); ++i)
        if (*failed || i == WAIT_TRIES || nanoseconds() - began > WAIT_NS) { *failed = 1; return false; }
    return true;
}
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
// False: given up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile uint32_t* failed) { return mbar_test(bar, parity) || mbar_wait_long(bar, parity, failed); }
// For a thread that has issued copies and will not see them land: time for them to.
__device__ __forceinline__ void let_copies_land() {
    for (uint32_t i = 0; i < 65536; ++i) __nanosleep(64);
}

// A box of a 2-D tensor map into shared memory; rows and columns outside the tensor are zeros.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}

__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) { asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols)); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Arrives at the barrier once every MMA issued so far by this thread is done.
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"(uint32_t(accumulate))
                 : "memory");
}
// The same with the first operand in tensor memory: row r in lane r, two values of k to a column.
__device__ __forceinline__ void mma_f16_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
                 "r"(uint32_t(accumulate))
                 : "memory");
}
// 16 columns of this thread's lane (those of a warp: 32 times its number modulo 4, and on).
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
                   "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Shared-memory descriptor of an operand in 128-byte swizzled lines, eight lines (1024 bytes) to a repeating unit.
//   K-major: a line holds 64 k of one row; `stride` is from one unit of eight rows to the next (the other offset is unused).
//   MN-major: a line holds 64 rows of one k; `lead` is from one unit of 64 rows to the next, `stride` from eight k to the next eight.
// 16 bytes further on is one more.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
    return uint64_t((addr & 0x3FFFF) >> 4) | uint64_t(lead >> 4) << 16 | uint64_t(stride >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// Instruction descriptor: bf16 operands, fp32 sums, M = 128 rows, N = n; `a_mn`: the first operand is MN-major.
__device__ __forceinline__ uint32_t instruction_desc(uint32_t n, bool a_mn) { return 1u << 4 | 1u << 7 | 1u << 10 | uint32_t(a_mn) << 15 | (n >> 3) << 17 | (128u >> 4) << 24; }

}  // namespace ptwm
