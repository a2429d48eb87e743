// attn_tc.cuh -- what the paired-CTA tensor-core attention kernels share: cluster addressing, 2-CTA tcgen05 forms,
// swizzled operand descriptors, TMA loads and bounded waits with cluster scope.
#pragma once
#include <cuda.h>
#include "moe_device.cuh"
#include "tcgen05.cuh"
#include "attn_internal.h"

namespace lk {

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
// The .aligned forms below (barriers, tensor-memory loads and stores) are undefined in a diverged warp, and a warp may
// leave a polling loop (wait_phase) lane by lane: each is preceded by __syncwarp().
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive() { __syncwarp(); asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { __syncwarp(); asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// the shared::cluster address of the same shared variable in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// Arrivals and waits have CTA scope: what they order is this CTA's shared memory, handed to the tensor core by
// fence.proxy.async, or tensor memory, ordered by the tcgen05 fences.  With cluster scope each arrival cost ~700 cycles
// and each wait ~150 on a B200 (a unit of work of k_tree 15 000 cycles).
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" :: "r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void arrive_expect_at(uint32_t cluster_bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" :: "r"(cluster_bar), "r"(bytes) : "memory");
}
// one thread waits for the phase of `parity`; false once WAIT_LIMIT_NS passes (recorded) or another role has given up
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* gave_up, int* err) {
    for (int i = 0; i < 64; ++i) if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (*gave_up) return false;
        if (globaltimer_ns() - t0 > WAIT_LIMIT_NS) { att_error(err, DEV_ERR_TIMEOUT_FULL); *gave_up = 1; return false; }
    }
    return true;
}

// the same by a whole warp, converged again afterwards
__device__ __forceinline__ bool warp_wait_phase(uint64_t* bar, uint32_t parity, volatile int* gave_up, int* err) {
    const bool ok = wait_phase(bar, parity, gave_up, err);
    __syncwarp();
    return ok;
}

// barrier 1 of 256 threads, and the same with the OR of a predicate
__device__ __forceinline__ void group_sync() { __syncwarp(); named_bar_sync(1, 256); }
__device__ __forceinline__ bool group_or(bool pred) { __syncwarp(); return named_bar_or(1, 256, pred); }

// ---- 2-CTA tcgen05: M = 128 rows are 64 of each CTA, N columns half of each.  The accumulator of a CTA's 64 rows uses
// all 128 lanes: row i, column n is lane i + 64 * (n >= N/2), column n % (N/2).
__device__ __forceinline__ void tmem_alloc2(uint32_t* dst_smem, uint32_t ncols) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(dst_smem)), "r"(ncols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc2(uint32_t taddr, uint32_t ncols) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(taddr), "r"(ncols) : "memory");
}
// Operand tiles of 128-byte rows with the 128-byte swizzle (8-row groups of 1 KB; 16-byte column c of row r at c ^ (r % 8)).
// K-major: row = M/N index, 64 16-bit values of K; a 16-deep K step is +32 bytes.
// MN-major: row = K index, 64 values of M/N; blocks of 64 M/N values `lbo` bytes apart; a 16-deep K step is +2048 bytes.
// Descriptor: low word start >> 4 and lbo >> 4, high word 8-row stride, version and swizzle.
constexpr uint32_t SW128_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t sw128_lo(uint32_t smem_addr, uint32_t lbo) { return ((smem_addr >> 4) & 0x3FFFu) | ((lbo >> 4) << 16); }
// true in one lane of a converged warp.  The single-thread roles branch on this: behind an ordinary lane test the compiler
// cannot know that one thread is active and serialises every TMA and MMA over the possible ones (~200 cycles each).
__device__ __forceinline__ bool elect_one() {
    uint32_t e = 0;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\t@p mov.u32 %0, 1;\n\t}" : "+r"(e));
    return e != 0;
}
// four 16-deep K steps of D[tmem] (+)= A x B^T, A_STEP and B_STEP bytes apart; the first overwrites D where !accumulate
template <uint32_t IDESC, uint32_t A_STEP, uint32_t B_STEP>
__device__ __forceinline__ void umma2_x4(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b32 al, bl;\n\t.reg .b64 ad, bd;\n\t"
                 "setp.ne.b32 p, %3, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"
                 "mov.b64 ad, {%1, %4};\n\tmov.b64 bd, {%2, %4};\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, p;\n\t"
                 "add.u32 al, %1, %6;\n\tadd.u32 bl, %2, %7;\n\tmov.b64 ad, {al, %4};\n\tmov.b64 bd, {bl, %4};\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, q;\n\t"
                 "add.u32 al, al, %6;\n\tadd.u32 bl, bl, %7;\n\tmov.b64 ad, {al, %4};\n\tmov.b64 bd, {bl, %4};\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, q;\n\t"
                 "add.u32 al, al, %6;\n\tadd.u32 bl, bl, %7;\n\tmov.b64 ad, {al, %4};\n\tmov.b64 bd, {bl, %4};\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, q;\n\t}"
                 :: "r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(accumulate), "n"(SW128_HI), "n"(IDESC), "n"(A_STEP >> 4), "n"(B_STEP >> 4) : "memory");
}
// the same with the instruction descriptor in a register, both operands K-major
__device__ __forceinline__ void umma2_x4_n(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b32 al, bl;\n\t.reg .b64 ad, bd;\n\t"
                 "setp.ne.b32 p, %3, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"
                 "mov.b64 ad, {%1, %4};\n\tmov.b64 bd, {%2, %4};\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, p;\n\t"
                 "add.u32 al, %1, 2;\n\tadd.u32 bl, %2, 2;\n\tmov.b64 ad, {al, %4};\n\tmov.b64 bd, {bl, %4};\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, q;\n\t"
                 "add.u32 al, al, 2;\n\tadd.u32 bl, bl, 2;\n\tmov.b64 ad, {al, %4};\n\tmov.b64 bd, {bl, %4};\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, q;\n\t"
                 "add.u32 al, al, 2;\n\tadd.u32 bl, bl, 2;\n\tmov.b64 ad, {al, %4};\n\tmov.b64 bd, {bl, %4};\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, q;\n\t}"
                 :: "r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(accumulate), "n"(SW128_HI), "r"(idesc) : "memory");
}
// arrive on this barrier in both CTAs when every tcgen05.mma issued so far has completed
__device__ __forceinline__ void commit2(uint64_t* bar) {
    asm volatile("{\n\t.reg .b16 m;\n\tmov.b16 m, 3;\n\t"
                 "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}"
                 :: "r"(smem_u32(bar)) : "memory");
}
__host__ __device__ constexpr uint32_t att_idesc(int M, int N, bool bf16, bool b_mn_major) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}
// box at (x, y) -> this CTA's shared memory; completes on a barrier of either CTA of the pair
__device__ __forceinline__ void tma_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t cluster_bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(cluster_bar) : "memory");
}

__device__ __forceinline__ void tma_3d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t cluster_bar) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(cluster_bar) : "memory");
}

// ---- 32 lanes x 32 columns
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    __syncwarp();
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    __syncwarp();
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
                 :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                   "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                   "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { __syncwarp(); asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { __syncwarp(); asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_approx(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&h;
}

}  // namespace lk
