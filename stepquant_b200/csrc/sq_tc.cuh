// tcgen05, TMA and mbarrier wrappers of the block-scaled product (sq_matmul.cu) and of prompts' attention
// (sq_attention_prompt.cu).
#pragma once

#include <cuda.h>

#include "sq_common.cuh"

namespace sq {
namespace tc {

constexpr int64_t kWaitClocks = int64_t(1) << 32;  // a wait gives up after about two seconds, unless the call says otherwise

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void bar_init(uint64_t *bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory"); }
__device__ __forceinline__ void bar_expect(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
// Waits for the phase of `parity`; false when `limit` clocks ran out (sets `abort`) or another warp
// set `abort`.  Both are looked at after the first try that fails and every 16th from there (a
// negative limit: never again).  A try suspends the thread for a while that the hardware chooses: an
// explicit time made the products 3 to 8 % slower, and so did a look after every try.  (The cycle
// counter bounds it: a read of the global timer takes longer than a block's products.)
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, volatile int *abort, int64_t limit) {
    int64_t since = 0;
    for (uint32_t it = 1;; ++it) {
        uint32_t done;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (done) return true;
        if ((it & 15) == 1) {
            if (*abort) return false;
            const int64_t now = clock64();
            if (since == 0) since = now;
            if (now - since > limit) {
                *abort = 1;
                return false;
            }
        }
    }
}

// The same, but a negative limit allows one look, which suspends nothing: a copy just begun is not there yet, so
// that the way out can be tested.
__device__ __forceinline__ bool bar_wait_or_look(uint64_t *bar, uint32_t parity, volatile int *abort, int64_t limit) {
    if (limit >= 0) return bar_wait(bar, parity, abort, limit);
    uint32_t done;
    asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    if (!done) *abort = 1;
    return done;
}

// One lane of the (converged) warp.
__device__ __forceinline__ bool elected() {
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}

// Box of a 2-D tensor map at (x, y) into shared memory, completing on `bar`.
__device__ __forceinline__ void tma_load(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y) : "memory");
}

// `bytes` (a multiple of 16) from src to dst, both 16-byte aligned, completing on `bar`.
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// K-major operand tile of 128-byte rows under the 128-byte swizzle, 8-row groups of 1024 bytes.
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
    return uint64_t((addr >> 4) & 0x3FFF) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// e4m3 x e4m3 -> fp32, M = 128, both operands K-major.
__device__ __forceinline__ constexpr uint32_t e4m3_product(int n) { return (1u << 4) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24); }

__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)) : "memory");
}
// f16 operands -> fp32, M = 128; B K-major, or MN-major (its rows are K).
__device__ __forceinline__ constexpr uint32_t half_product(int n, bool b_mn) {
    return (1u << 4) | (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}
// Operand tile of 128-byte rows (64 values) under the 128-byte swizzle whose rows are K: `lead` bytes to
// the next 64 values.
__device__ __forceinline__ uint64_t operand_mn(uint32_t addr, uint32_t lead) {
    return uint64_t((addr >> 4) & 0x3FFF) | (uint64_t(lead >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// K-major operand tile of 16 values of K without a swizzle: two pieces of 16 bytes a row, `lead` bytes
// apart, each 8 rows of them contiguous.
__device__ __forceinline__ uint64_t operand_narrow(uint32_t addr, uint32_t lead) {
    return uint64_t((addr >> 4) & 0x3FFF) | (uint64_t(lead >> 4) << 16) | (uint64_t(128 >> 4) << 32) | (1ull << 46);
}
__device__ __forceinline__ void mma_half(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)) : "memory");
}
// A in tensor memory: lanes are its rows, a column holds two values of K.
__device__ __forceinline__ void mma_half_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)) : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(slot)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(addr), "r"(columns));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }

// Eight or sixteen consecutive fp32 columns of the thread's lane; valid after tmem_wait().
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(addr));
}
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
#define SQ_R8(i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define SQ_W8(i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : SQ_R8(0), SQ_R8(8), SQ_R8(16), SQ_R8(24) : "r"(addr));
}
// Stores are in tensor memory after tmem_stored().
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n"
                 ::"r"(addr), SQ_W8(0), SQ_W8(8) : "memory");
}
#undef SQ_R8
#undef SQ_W8
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// The registers pass through the wait, so that no use of theirs moves before it.
template <int N>
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

}  // namespace tc
}  // namespace sq
