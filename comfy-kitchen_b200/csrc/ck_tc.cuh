// Wrappers around the instructions that a TMA / tcgen05 pipeline of one CTA uses (cta_group::1, 16-bit operands).
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "ck_common.cuh"

namespace ck {
namespace tc {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_init_done() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
// A look that does not suspend the thread (try_wait takes some 150 clocks even where the phase is over).
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
constexpr uint32_t kSpinLimit = 1u << 22;   // polls before giving up (a fraction of a second)

// One lane of a converged warp, chosen by the hardware.  The roles that issue copies and MMAs run their loops with the
// whole warp and choose a lane only around a run of issues: addresses and descriptors then stay in uniform registers, where
// the instructions want them (a loop run by lane 0 alone: 240 clocks an MMA; this way: 85; a lane chosen for each: 148).
__device__ __forceinline__ bool elect_one() {
    uint32_t pred;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(pred));
    return pred != 0;
}

// Bounded wait of one thread.  False when the limit ran out (recorded in *status) or another role of the CTA has given up.
__device__ __forceinline__ bool mbar_wait_one(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
    if (mbar_test_wait(bar, parity)) return true;
    for (uint32_t i = 0; i < kSpinLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 1023u) == 1023u && *abort_flag) return false;
    }
    if (!*abort_flag) {
        *abort_flag = 1;
        atomicCAS(status, 0, (code << 16) | (int)(blockIdx.x & 0xffff));
    }
    return false;
}
// The same by a whole warp; every lane gets the same answer.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
    return __all_sync(0xffffffffu, mbar_wait_one(bar, parity, abort_flag, status, code));
}
// A place in a ring of stages and the parity of its current round (kept by counting: dividing a running number by a
// stage count that is known at run time only costs more than the rest of a loop's step).  A consumer waits for parity
// `round`, a producer for the other one, which a fresh barrier grants at once.
struct Ring {
    int at = 0;
    uint32_t round = 0;
    __device__ __forceinline__ void next(int stages) {
        if (++at == stages) { at = 0; round ^= 1u; }
    }
};

// What a role that gives up does for its copies and MMAs in flight: they end before shared memory and TMEM go.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < kSpinLimit && !mbar_try_wait(bar, parity); ++i) {}
}
// The copies of the last `issued` (at most all) stages before `ring`'s place.
__device__ __forceinline__ void ring_drain(uint64_t* full, Ring ring, uint32_t issued, int stages) {
    for (uint32_t i = 0; i < issued && i < (uint32_t)stages; ++i) {
        if (--ring.at < 0) { ring.at = stages - 1; ring.round ^= 1u; }
        mbar_drain(&full[ring.at], ring.round);
    }
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(c0), "r"(c1), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar)) : "memory");
}
// 16-byte aligned addresses and size.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// Shared -> global (clipped at the tensor's edges), one bulk group of the issuing thread per call of tma_store_commit().
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(map), "r"(smem_u32(src)), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kLeft) : "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// All threads of the cluster; what they have written before, global memory included, is seen after it.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A kernel launched with programmatic stream serialization may start once every CTA of the one before has called the first,
// and sees that kernel's results behind the second.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_dependency() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// TMEM columns (a power of two from 32 on); both by one whole warp, the same one.
__device__ __forceinline__ void tmem_alloc(uint32_t* base_in_smem, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(base_in_smem)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}

// Operand tiles: K-major rows of 128 bytes (64 elements), 128-byte swizzle, groups of 8 rows 1024 bytes apart.  The low
// word of a descriptor is the address / 16 (16 elements of K further on: + 2) and the unused leading offset.
constexpr uint32_t kDescHi = 64u | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(const void* tile) { return ((smem_u32(tile) & 0x3ffffu) >> 4) | (1u << 16); }

// D[128, n] (+)= A[128, 16] . B[n, 16]^T, both f16 or both bf16, fp32 accumulator.  By one thread (elect_one()), which issues
// a whole run of them and their commit.
__device__ __forceinline__ uint32_t idesc(bool bf16, int n) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_16bit(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{ .reg .pred p; .reg .b64 da, db; setp.ne.b32 p, %4, 0;\n"
        "mov.b64 da, {%1, %5}; mov.b64 db, {%2, %5};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p; }"
        ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(kDescHi) : "memory");
}
// Arrives on the barrier once the MMAs that this thread has issued so far are complete.
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// 16 consecutive fp32 columns of this lane's TMEM row.
__device__ __forceinline__ void ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ------------------------------------------------------------------ host: tensor maps

using EncodeFn = PFN_cuTensorMapEncodeTiled_v12000;

inline EncodeFn get_encode() {
    static EncodeFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeFn>(sym);
    });
    return fn;
}

// A 16-bit tensor of `rank` dimensions (innermost first; strides in bytes from the second on), boxes of 64 elements x
// box_rows, 128-byte swizzle, zeros outside.
inline bool make_map_16bit(CUtensorMap* map, const void* base, int rank, const int64_t* dims, const int64_t* strides, int box_rows) {
    EncodeFn enc = get_encode();
    if (!enc) return false;
    cuuint64_t d[3], s[2];
    cuuint32_t box[3] = {64u, (cuuint32_t)box_rows, 1u}, step[3] = {1u, 1u, 1u};
    for (int i = 0; i < rank; ++i) d[i] = (cuuint64_t)dims[i];
    for (int i = 0; i + 1 < rank; ++i) s[i] = (cuuint64_t)strides[i];
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, (cuuint32_t)rank, const_cast<void*>(base), d, s, box, step,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tc
}  // namespace ck
