// The 5th-generation tensor cores (tcgen05, TMEM): PTX wrappers, descriptors and the
// GEMM epilogue that pk_gemm.cu and pk_adapter.cu share.
#pragma once

#include "pk_common.cuh"

namespace pk {
namespace {

constexpr int kBM = 128, kBK = 64;
constexpr int kABytes = kBM * kBK * 2;   // 16 KB per stage

__device__ __forceinline__ void tma_load_2d(void *dst, const CUtensorMap *map, uint64_t *bar,
                                            int32_t c0, int32_t c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar))
        : "memory");
}

// Shared-memory matrix descriptor of a K-major operand tile written by TMA
// with 128B swizzle (rows of 128 bytes, 8-row swizzle atoms of 1024 bytes):
// start address >> 4, leading byte offset 1 (unused for swizzled K-major),
// stride byte offset 1024 >> 4 between 8-row groups, descriptor version 1,
// layout type 2 = 128B swizzle.  The tile base is 1024-byte aligned, so the
// base offset is 0; a K step of 16 elements inside the atom advances the start
// address by 32 bytes.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) |
           ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// Instruction descriptor, kind::f16: D fp32 (bits 4-5 = 1), A and B bf16
// (bits 7-9, 10-12 = 1), both K-major (bits 15, 16 = 0), N >> 3 at bit 17,
// M >> 4 at bit 24.
constexpr uint32_t idesc_bf16(int m, int n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void umma_bf16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                          uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void mbar_arrive_cta(uint64_t *bar) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// arrive on `bar` when every tcgen05.mma issued so far by this thread is done
__device__ __forceinline__ void umma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     smem_u32(bar))
                 : "memory");
}

// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r));
    return r != 0;
}

// The .aligned instructions are the whole warp's: the wrappers join its lanes, whatever
// branches some of them took before (one thread sets the barriers up).
__device__ __forceinline__ void tmem_alloc(uint32_t *dst, uint32_t ncols) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(dst)),
                 "r"(ncols)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// 32 consecutive fp32 columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    __syncwarp();
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
        "%28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Epilogue staging: each epilogue warp owns a 32-row tile of 64 bf16 columns
// in shared memory (rows padded to 144 bytes: a row-per-lane 16-byte access
// and a row-segment access are both free of bank conflicts).
constexpr int kStageRow = 144;
constexpr int kStageBytes = 32 * kStageRow;

// The epilogue of accumulator columns [col, col + 64) of the warp's tile rows
// row0 .. row0 + 31 (TMEM lane l of taddr = row row0 + l).  The arithmetic runs
// a row per lane, as the accumulator comes out of TMEM; the residual rows are
// read and the output rows written through the warp's staging tile as whole
// 128-byte row segments (four rows per warp access), where a row per lane would
// touch 32 rows per access.
constexpr bool is_residual(int epi) {
    return epi == PK_GEMM_RESIDUAL || epi == PK_GEMM_RESIDUAL_RELU;
}

// Where a tile's rows 0 .. 31 of a warp lie in C and R: consecutive from row0, and
// nowhere (-1) past the last one.
struct LinearRows {
    int row0, M;
    __device__ __forceinline__ int operator()(int r, int) const {
        return row0 + r < M ? row0 + r : -1;
    }
};

// This lane's share of the residual rows of the same 64 columns, as row
// segments (piece i: row row0 + 4 i + lane / 8, bytes (lane % 8) * 16 ..):
// loaded ahead of the columns' epilogue so that the load latency overlaps work.
template <typename Rows>
__device__ __forceinline__ void load_residual64(uint4 (&rv)[8], const Rows &rows, int col,
                                                const __nv_bfloat16 *R, int64_t ldr) {
    const int lane = threadIdx.x & 31;
    const int sr = lane >> 3, sb = (lane & 7) * 16;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = rows(i * 4 + sr, i);
        rv[i] = make_uint4(0u, 0u, 0u, 0u);
        if (row >= 0)
            rv[i] = *reinterpret_cast<const uint4 *>(
                reinterpret_cast<const char *>(R + (int64_t)row * ldr + col) + sb);
    }
}

template <int EPI, typename Rows>
__device__ __forceinline__ void epilogue_tile64(uint32_t taddr, const Rows &rows, int col,
                                                __nv_bfloat16 *C, int64_t ldc,
                                                const uint4 (&rv)[8], const __nv_bfloat16 *bias,
                                                float alpha, uint8_t *stage) {
    constexpr bool kRes = is_residual(EPI);
    const int lane = threadIdx.x & 31;
    const int sr = lane >> 3, sb = (lane & 7) * 16;   // row-segment phase: row in 4, byte
    if (kRes) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4 *>(stage + (i * 4 + sr) * kStageRow + sb) = rv[i];
    }
    float v[64];
    tmem_ld32(taddr, *reinterpret_cast<float(*)[32]>(v));
    tmem_ld32(taddr + 32, *reinterpret_cast<float(*)[32]>(v + 32));
    __syncwarp();   // residual rows staged
    uint8_t *mine = stage + lane * kStageRow;
    if (EPI == PK_GEMM_SILU) {
#pragma unroll
        for (int i = 0; i < 64; ++i) v[i] = __fdividef(v[i], 1.f + __expf(-v[i]));
    } else if (kRes) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            float f[8];
            unpack16(*reinterpret_cast<const uint4 *>(mine + q * 16), f, bias);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float t = f[i] + alpha * v[q * 8 + i];
                v[q * 8 + i] = EPI == PK_GEMM_RESIDUAL_RELU ? fmaxf(t, 0.f) : t;
            }
        }
    } else if (EPI == PK_GEMM_BIAS) {
        const uint4 *bp = reinterpret_cast<const uint4 *>(bias + col);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            float f[8];
            unpack16(bp[q], f, bias);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[q * 8 + i] += f[i];
        }
    }
    __syncwarp();   // every lane's residual row read
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        uint4 o;
        __nv_bfloat162 *h = reinterpret_cast<__nv_bfloat162 *>(&o);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            h[i] = __floats2bfloat162_rn(v[q * 8 + 2 * i], v[q * 8 + 2 * i + 1]);
        *reinterpret_cast<uint4 *>(mine + q * 16) = o;
    }
    __syncwarp();   // output rows staged
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + sr, row = rows(r, i);
        if (row >= 0)
            *reinterpret_cast<uint4 *>(reinterpret_cast<char *>(C + (int64_t)row * ldc + col) + sb) =
                *reinterpret_cast<const uint4 *>(stage + r * kStageRow + sb);
    }
    __syncwarp();   // staging tile free again
}

// ---------------------------------------------------------------- CTA pairs
__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// shared::cluster address of the same shared-memory object in CTA `rank`
__device__ __forceinline__ uint32_t mapa_rank(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// arrive on an mbarrier of either CTA of the cluster (release at cluster scope)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr)
                 : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "n"(kSuspendNs)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_cluster_bounded(uint64_t *bar, uint32_t parity,
                                                          uint64_t limit_ns) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait_cluster(bar, parity)) {
        if (globaltimer_ns() - t0 > limit_ns) return false;
    }
    return true;
}
// 2-D tile load into this CTA's shared memory, completion on an mbarrier of
// either CTA of the pair (bar: shared::cluster address)
__device__ __forceinline__ void tma_load_2d_pair(void *dst, const CUtensorMap *map, uint32_t bar,
                                                 int32_t c0, int32_t c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void umma_bf16_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                               uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// arrive on `bar` (same offset) in both CTAs of the pair when the MMAs issued so
// far by this thread are done
__device__ __forceinline__ void umma_commit_pair(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)0x3)
        : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t *dst, uint32_t ncols) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(dst)),
                 "r"(ncols)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
                 : "memory");
}

}  // namespace
}  // namespace pk
