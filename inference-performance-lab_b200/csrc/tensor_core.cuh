// tcgen05 (5th-generation tensor core) and tensor-map TMA helpers for sm_100a.
#pragma once

#include "ipl_common.cuh"

#include <cuda.h>

namespace ipl {

// ---- TMA, tiled form (no multicast) ------------------------------------------------------------

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void prefetch_tensor_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// Orders this thread's shared-memory writes before later reads by the tensor core or TMA.
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- tensor memory -------------------------------------------------------------------------------

// All columns of the SM's tensor memory; the address lands at `slot` in shared memory. A whole warp.
constexpr uint32_t kTmemColumns = 512;
__device__ __forceinline__ void tmem_alloc(uint32_t slot) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "n"(kTmemColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t address) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "n"(kTmemColumns) : "memory");
}
__device__ __forceinline__ void tcgen05_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this thread's lane (the warp's lane quarter is in the address). The values are there
// after tmem_wait_loads.
__device__ __forceinline__ void tmem_load_32(uint32_t address, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(address));
}
__device__ __forceinline__ void tmem_load_16(uint32_t address, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(address));
}
__device__ __forceinline__ void tmem_store_16(uint32_t address, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(address)
        : "memory");
}

// Moves registers between the warpgroups of a CTA (every warp of the warpgroup executes it): the sum over
// them must not exceed what the CTA was launched with, or the takers wait for good.
template <int kRegisters>
__device__ __forceinline__ void warpgroup_take_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegisters));
}
template <int kRegisters>
__device__ __forceinline__ void warpgroup_leave_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegisters));
}

// ---- tcgen05.mma -----------------------------------------------------------------------------------

// Shared-memory matrix descriptor of a tile in rows of 128 bytes, 128-byte swizzled as TMA writes it
// (the pattern repeats every 8 rows = 1024 bytes, to which the tile is aligned). Descriptor fields:
// address, leading and stride offsets in 16-byte units, version 1 at bit 46, swizzle mode 2 at bit 61.
// * operand along rows (K-major): `stride` = 1024, the next 8 rows; the leading offset is unused;
// * operand across rows (MN-major): `leading` = bytes to the next 64 elements of a row, `stride` = 1024.
// The address field takes sums in 16-byte units, so a descriptor moves by adding to its low word.
__device__ __forceinline__ uint32_t smem_descriptor_low(uint32_t address, uint32_t leading) {
    return ((address & 0x3ffffu) >> 4) | (leading >> 4) << 16;
}
constexpr uint32_t smem_descriptor_high(uint32_t stride) { return (stride >> 4) | 1u << 14 | 2u << 29; }
__device__ __forceinline__ uint64_t smem_descriptor(uint32_t low, uint32_t high) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "r"(high));
    return d;
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_lane() {
    uint32_t elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
    return elected != 0;
}
// kind::f16 instruction descriptor: fp32 accumulator, bf16 operands, A K-major, B K-major or MN-major.
constexpr uint32_t mma_descriptor(int m, int n, bool b_mn_major) {
    return 1u << 4 | 1u << 7 | 1u << 10 | (b_mn_major ? 1u << 16 : 0u) | static_cast<uint32_t>(n / 8) << 17 |
           static_cast<uint32_t>(m / 16) << 24;
}
// D[tmem] (+)= A[smem] B[smem], 16 elements of the inner dimension. One thread.
__device__ __forceinline__ void mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t descriptor, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(descriptor), "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}
// The same with A in tensor memory: two bf16 of a row in each 32-bit column.
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t descriptor, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(descriptor), "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}
// Arrives at `bar` once every tcgen05 operation this thread has issued is complete.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

}  // namespace ipl
