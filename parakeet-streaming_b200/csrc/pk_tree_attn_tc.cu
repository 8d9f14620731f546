// Tree attention (see pk_tree_attn.cu) for row tiles of up to 128 query rows, bf16,
// on the 5th-generation tensor cores.
//
// Bound by reading K and V as long as a request's rows fit one tile: 128 keys of a
// 128-wide head are 64 KB, 2800 cycles of an SM's share of the memory rate, for some
// 1400 cycles of MMAs and 1024 of exponentials (without either the kernel takes as long).
// But a tile is a chain - S, the softmax (loads from TMEM, maximum, exp2, sum,
// conversions), O - and beginning and ending a row tile another.  So one CTA an SM with
// two workers, each with a share of the step's line, a ring of its own and its own warps,
// and S of the next tile (of 64 keys) under the softmax of this one:
//   warps 0, 2   pages of K and V by TMA into a ring of slots (a slot: one tile of K or
//                of V), running ahead over the worker's units
//   warps 1, 3   S = Q K^T (both from shared memory, fp32 in TMEM) and O += P V (P
//                from TMEM, V from shared memory as it lies: a row-major [keys][dim]
//                tile is the MN-major operand), O in TMEM
//   warps 4..11  four a worker, a thread per row (TMEM lane): the row's scores without a
//                shuffle, maximum, exp2, P as bf16 over the scores, fp32 sum; the next
//                unit's queries ahead of the epilogue
// Two groups that took every other tile (of 128 keys) of one worker's units and met at
// their ends took 140 us for 32 requests x 8 heads of 128 with up to 128 rows and 8000
// tokens, this takes 125 (4.8 TB/s); 160 x 8 heads of 64 with 21 rows and 2000 tokens: 171
// and 128; 160 x 8 heads of 128 with 33 rows and 500 tokens: 135 and 93; a single request
// of 131,000 tokens, whose shares are cut twice as often: 98 and 103 (5.2 TB/s).
// The running maximum is raised, and O scaled for it, only when a row's scores pass
// the one in use by more than 2^8: weights stay below 256, which the fp32 sums and
// bf16's exponent hold, and most tiles touch O in the MMA alone.
#include <math.h>

#include "pk_tree.cuh"
#include "pk_umma.cuh"

namespace pk {
namespace {

constexpr int kRows = 128, kKeys = 64, kTcThreads = 128 + 256;
constexpr float kRaise = 8.f;   // log2 of how far scores may pass the maximum in use

template <int DH>
struct TcShape {
    static constexpr int kSlot = kKeys * DH * 2;       // one tile of K or V
    static constexpr int kQ = kRows * DH * 2;
    static constexpr int kGroup = DH / 64 * 1024;      // 8 rows of one
    static constexpr int kSlots = DH == 64 ? 10 : 5;   // a worker's, beside its Q
    static constexpr int kWorker = kQ + kSlots * kSlot;
    static constexpr int kSmem = 2 * kWorker + 1024;
    // TMEM columns: each worker's S, twice (P over it), each worker's O
    static constexpr int kS = 0, kO = 4 * kKeys, kTmem = 512;
    // barriers of a worker: slots full and empty, then
    // (S, P and O of even and odd tiles have barriers of their own: two tiles are under way)
    enum {
        kQFull = 2 * kSlots,
        kIdle,
        kODone,
        kSFull = kODone + 2,
        kPFull = kSFull + 2,
        kBars = kPFull + 2
    };
};

// O += P V: A from TMEM (bf16 pairs), B MN-major
__device__ __forceinline__ void umma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc,
                                             uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Descriptor of a tile of tma_load_rows: 128B swizzle, `group` bytes between groups of
// 8 rows (SBO).  As a K-major operand (rows x 64 columns of the dim) the LBO is unused;
// as an MN-major one (the dim x keys) it is the 1024 bytes between 64-column blocks.
__device__ __forceinline__ uint64_t tile_desc(uint32_t saddr, uint32_t group) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(1024 >> 4) << 16) |
           ((uint64_t)(group >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    __syncwarp();
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
        "%28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// a row's scores: one wait for their loads
__device__ __forceinline__ void tmem_ld_scores(uint32_t taddr, float (&v)[kKeys]) {
    __syncwarp();
    uint32_t r[kKeys];
#pragma unroll
    for (int c = 0; c < kKeys; c += 32)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
            "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
            "%28, %29, %30, %31}, [%32];"
            : "=r"(r[c]), "=r"(r[c + 1]), "=r"(r[c + 2]), "=r"(r[c + 3]), "=r"(r[c + 4]),
              "=r"(r[c + 5]), "=r"(r[c + 6]), "=r"(r[c + 7]), "=r"(r[c + 8]), "=r"(r[c + 9]),
              "=r"(r[c + 10]), "=r"(r[c + 11]), "=r"(r[c + 12]), "=r"(r[c + 13]), "=r"(r[c + 14]),
              "=r"(r[c + 15]), "=r"(r[c + 16]), "=r"(r[c + 17]), "=r"(r[c + 18]), "=r"(r[c + 19]),
              "=r"(r[c + 20]), "=r"(r[c + 21]), "=r"(r[c + 22]), "=r"(r[c + 23]), "=r"(r[c + 24]),
              "=r"(r[c + 25]), "=r"(r[c + 26]), "=r"(r[c + 27]), "=r"(r[c + 28]), "=r"(r[c + 29]),
              "=r"(r[c + 30]), "=r"(r[c + 31])
            : "r"(taddr + c));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < kKeys; ++i) v[i] = __uint_as_float(r[i]);
}
// two fp32 operations an instruction
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    return (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float low2(uint64_t a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float high2(uint64_t a) { return __uint_as_float((uint32_t)(a >> 32)); }
__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// barrier of one worker's softmax warps (four) that also ORs a flag over them
__device__ __forceinline__ bool group_any(int group, bool v) {
    uint32_t r;
    __syncwarp();
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, %2, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v), "r"(2 + group)
        : "memory");
    return r != 0;
}
// Bits of keys rel0 .. rel0 + 31 of the step's own tokens that a row sees.
__device__ __forceinline__ uint32_t seen_bits(int trees, uint64_t mask, int node, int rel0) {
    if (rel0 <= -32) return 0xffffffffu;
    if (!trees) {
        const int n = node - rel0 + 1;   // keys up to the row's own
        return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u);
    }
    if (rel0 >= 64) return 0u;
    if (rel0 >= 0) return (uint32_t)(mask >> rel0);
    return (uint32_t)(mask << -rel0) | ((1u << -rel0) - 1u);
}

template <int DH>
__global__ void __launch_bounds__(kTcThreads, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ TreeParams p) {
    using S = TcShape<DH>;
    constexpr int NS = S::kSlots;
    extern __shared__ uint8_t tree_smem[];
    __shared__ __align__(8) uint64_t bars[2][S::kBars];   // of each worker
    __shared__ uint32_t tmem_base;
    __shared__ volatile int failed;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // worker 0: warps 0 and 1 (copies, MMAs) and 4 .. 7 (softmax); worker 1: 2, 3, 8 .. 11
    const int w = warp < 4 ? warp >> 1 : (warp >> 2) - 1;
    uint8_t *sq = reinterpret_cast<uint8_t *>(
                      (reinterpret_cast<uintptr_t>(tree_smem) + 1023) & ~uintptr_t(1023)) +
                  w * S::kWorker;
    uint8_t *ring = sq + S::kQ;
    uint64_t *full = bars[w], *empty = full + NS, *q_full = full + S::kQFull,
             *s_full = full + S::kSFull, *p_full = full + S::kPFull, *o_done = full + S::kODone,
             *idle = full + S::kIdle;
    if (threadIdx.x == 0) {
        for (int v = 0; v < 2; ++v)
            for (int s = 0; s < S::kBars; ++s)
                mbar_init(&bars[v][s], s == S::kQFull || s >= S::kPFull ? 4 : 1);
        failed = 0;
        fence_mbar_init();
        prefetch_tmap(&kv_map);
    }
    if (warp == 0) {
        tmem_alloc(&tmem_base, S::kTmem);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base;
    grid_dep_wait();
    grid_dep_launch();
    const int worker = w * gridDim.x + blockIdx.x;   // neighbouring shares on different SMs

    auto produce = [&]() {
        // lanes issue a tile's boxes, K then V
        const int ps = 1 << p.ps_shift, rows_box = min(ps, kTokRowsBox);
        const int box_of = lane;
        const uint32_t bytes = rows_box * DH * 2;
        int it = 0;
        bool stop = false;   // the warp's, so that its lanes stay together
        Work work(p, worker);
        Pages pages, then;
        bool more = work.next();
        Unit u = work.u;
        if (more) pages.open(p, u);
        while (more && !stop) {
            more = work.next();
            if (more) then.open(p, work.u);
            // K of a tile ahead of V of the one before: the order of their products
            const int len = u.ctx + u.count;
            int last = 0;   // the page of this lane's box of the tile before
            for (int t = u.t0; t <= u.t1 && u.t0 < u.t1 && !stop; ++t) {
                int page = last;
                if (t < u.t1) {
                    const int k0 = t * kKeys, n = (min(kKeys, len - k0) + rows_box - 1) / rows_box;
                    // lanes without a box ask for the last one's page
                    page = pages.get((k0 + min(box_of, n - 1) * rows_box) >> p.ps_shift);
                    if (page < 0 || page >= p.num_pages) {
                        raise(p.error, PK_DEV_BAD_PAGE);
                        page = 0;
                    }
                }
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const int tile = t - v;   // V of the tile before
                    if (tile < u.t0 || tile >= u.t1) continue;
                    const int k0 = tile * kKeys, n = (min(kKeys, len - k0) + rows_box - 1) / rows_box;
                    const int s = it % NS, use = it / NS;
                    ++it;
                    if (use) ring_wait(&empty[s], (use - 1) & 1, &failed, p.error);
                    stop = __any_sync(0xffffffffu, failed != 0);
                    if (stop) {
                        --it;
                        break;
                    }
                    if (lane == 0) mbar_arrive_expect_tx(&full[s], n * bytes);
                    __syncwarp();
                    if (box_of < n)
                        tma_load_rows(ring + s * S::kSlot + box_of * bytes, &kv_map, &full[s],
                                      (k0 + box_of * rows_box) & (ps - 1),
                                      (((v ? last : page) * p.num_layers + p.layer) * 2 + v) * p.kv_heads +
                                          u.head);
                }
                last = page;
            }
            u = work.u;
            pages = then;
        }
        if (stop)   // leave no copy in flight
            for (int s = 0; s < NS; ++s)
                if (it > s) mbar_wait_bounded(&full[s], ((it - 1 - s) / NS) & 1, kWaitLimitNs);
    };
    auto multiply = [&]() {
        Work work(p, worker);
        constexpr uint32_t id_s = idesc_bf16(kRows, kKeys);
        constexpr uint32_t id_o = idesc_bf16(kRows, DH) | (1u << 16);   // B MN-major
        const uint64_t q0 = tile_desc(smem_u32(sq), S::kGroup), ring0 = tile_desc(smem_u32(ring), S::kGroup);
        const uint32_t st = tmem + S::kS + w * 2 * kKeys, ot = tmem + S::kO + w * DH;
        // the whole warp walks along, so that indexes and descriptors are uniform
        const bool one = elect_one();
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            return __all_sync(0xffffffffu, ring_wait(bar, parity, &failed, p.error));
        };
        int s = 0, unit = 0;   // ring slot, unit of this worker
        uint32_t phase = 0, j = 0;   // of the ring, tile of this worker
        bool ok = true;
        auto next = [&]() {
            if (++s == NS) {
                s = 0;
                phase ^= 1;
            }
        };
        // S of a tile, over the P of the tile two before: the products issued so far, of
        // tiles below j, have to be done with it
        auto scores = [&](uint32_t tile) {
            ok = ok && (j == 0 || wait(&o_done[(j - 1) & 1], ((j - 1) >> 1) & 1)) && wait(&full[s], phase);
            if (!ok) return;
            tc_fence_after();
            if (one) {
                const uint64_t k0 = ring0 + s * (S::kSlot >> 4);
#pragma unroll
                for (int kk = 0; kk < DH / 16; ++kk) {
                    const uint32_t off = ((kk / 4) * 1024 + (kk % 4) * 32) >> 4;
                    umma_bf16(st + (tile & 1) * kKeys, q0 + off, k0 + off, id_s, kk != 0);
                }
                umma_commit(&empty[s]);
                umma_commit(&s_full[tile & 1]);
            }
            __syncwarp();
            next();
        };
        while (ok && work.next()) {
            const int n = work.u.t1 - work.u.t0;
            if (n <= 0) continue;
            ok = wait(q_full, unit & 1);
            ++unit;
            scores(j);
            for (int i = 0; i < n && ok; ++i, ++j) {
                if (i + 1 < n) scores(j + 1);
                ok = ok && wait(&full[s], phase) && wait(&p_full[j & 1], (j >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
                if (one) {
                    const uint64_t v0 = ring0 + s * (S::kSlot >> 4);
#pragma unroll
                    for (int kk = 0; kk < kKeys / 16; ++kk)
                        umma_bf16_ts(ot, st + (j & 1) * kKeys + kk * 8, v0 + kk * (2 * S::kGroup >> 4),
                                     id_o, (i > 0) | (kk != 0));
                    umma_commit(&empty[s]);
                    umma_commit(&o_done[j & 1]);
                }
                __syncwarp();
                next();
            }
        }
        if (one) umma_commit(idle);   // no MMA is left when the CTA frees its TMEM
        __syncwarp();
        mbar_wait_bounded(idle, 0, kWaitLimitNs);
    };

    if (warp < 4) {
        if (warp & 1) multiply();
        else produce();
    } else {
        Work work(p, worker);
        // thread = row (TMEM lane) 32 (warp % 4) + lane of the tile
        const int quad = warp & 3, rt = quad * 32 + lane;
        const int gt = threadIdx.x & 127;   // thread in the group
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const uint32_t st0 = tmem + lanes + S::kS + w * 2 * kKeys, ot = tmem + lanes + S::kO + w * DH;
        const __nv_bfloat16 *q = static_cast<const __nv_bfloat16 *>(p.q);
        __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out);
        // this thread's row of a unit
        struct Row {
            Unit u;
            int node;   // -1: none
            int64_t row, qh;
            uint64_t mask;
        } now, then;
        bool more;
        // the next unit's row, its query to shared memory: ahead of the epilogue of the unit
        // before, whose scores have all been read
        auto advance = [&](Row &x) {
            more = work.next();
            if (!more) return;
            x.u = work.u;
            const int r = x.u.rt * kRows + rt;
            const bool live = r < x.u.count * p.group;
            x.node = live ? r / p.group : -1;
            x.row = x.u.row0 + (live ? x.node : 0);
            x.qh = (int64_t)x.u.head * p.group + (live ? r - x.node * p.group : 0);
            x.mask = 0;
            if (live && p.trees) x.mask = reinterpret_cast<const uint64_t *>(p.step + p.l.mask)[x.row];
            if (x.u.t1 <= x.u.t0) return;
            const uint4 *src = reinterpret_cast<const uint4 *>(q + x.row * p.q_rs + x.qh * p.q_hs);
#pragma unroll
            for (int c = 0; c < DH / 8; ++c)
                *reinterpret_cast<uint4 *>(sq + tile_at<DH>(rt, c)) =
                    live ? src[c] : make_uint4(0u, 0u, 0u, 0u);
            fence_async_proxy();
            __syncwarp();
            if (lane == 0) arrive(q_full);
        };
        advance(now);
        uint32_t it = 0, j = 0;   // ring use and tile of this worker where the unit begins
        while (more) {
            const Unit &u = now.u;
            const int len = u.ctx + u.count;
            float m = -INFINITY, l = 0.f;   // the maximum in use (scaled), the sum
            bool odd = false;               // a value that is not finite among the own rows
            const int n = u.t1 - u.t0;
            for (int i = 0; i < n; ++i, ++j) {
                const int k0 = (u.t0 + i) * kKeys;
                const uint32_t st = st0 + (j & 1) * kKeys;
                ring_wait(&s_full[j & 1], (j >> 1) & 1, &failed, p.error);
                __syncwarp();
                tc_fence_after();
                float sc[kKeys];
                tmem_ld_scores(st, sc);
                if (k0 + kKeys > u.ctx) {   // some of the step's own tokens, or the end
#pragma unroll
                    for (int c = 0; c < kKeys / 32; ++c) {
                        const uint32_t bits =
                            seen_bits(p.trees, now.mask, now.node, k0 + c * 32 - u.ctx);
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(bits >> e & 1)) sc[c * 32 + e] = -INFINITY;
                    }
                    // V rows past the end hold what the page held before, and a token's
                    // values may be inf or NaN: zero in the product, where a weight of
                    // zero would not keep them out; the epilogue adds the latter to the
                    // rows that see them
                    const uint32_t use = it + (i + 1 < n ? 2 * i + 2 : 2 * i + 1);
                    ring_wait(&full[use % NS], (use / NS) & 1, &failed, p.error);
                    uint8_t *vs = ring + use % NS * S::kSlot;
                    bool bad = false;
                    for (int c = max(u.ctx - k0, 0) * (DH / 8) + gt; c < kKeys * DH / 8; c += 128) {
                        const int vr = c / (DH / 8), ch = c % (DH / 8), key = k0 + vr;
                        uint4 *at = reinterpret_cast<uint4 *>(vs + tile_at<DH>(vr, ch));
                        uint4 x = make_uint4(0u, 0u, 0u, 0u);
                        if (key < len) {
                            x = *at;
                            uint32_t *e = &x.x;
                            bool here = false;
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                if ((e[k] & 0x7f80u) == 0x7f80u) {
                                    e[k] &= 0xffff0000u;
                                    here = true;
                                }
                                if ((e[k] & 0x7f800000u) == 0x7f800000u) {
                                    e[k] &= 0x0000ffffu;
                                    here = true;
                                }
                            }
                            if (!here) continue;
                            bad = true;
                        }
                        *at = x;
                    }
                    fence_async_proxy();
                    odd |= group_any(w, bad);
                }
                float tops[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
                for (int e = 4; e < kKeys; ++e) tops[e & 3] = fmaxf(tops[e & 3], sc[e]);
                float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                top = top == -INFINITY ? top : __fmul_rn(top, p.scale_log2);
                const bool raise_it = top > m + kRaise || (m == -INFINITY && top > m);
                if (__any_sync(0xffffffffu, raise_it)) {
                    const float keep = raise_it ? ex2(m - top) : 1.f;
                    if (raise_it) m = top;
                    l *= keep;
                    if (i > 0) {   // O has the unit's tiles before
                        ring_wait(&o_done[(j - 1) & 1], ((j - 1) >> 1) & 1, &failed, p.error);
                        __syncwarp();
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < DH / 32; ++c) {
                            float o[32];
                            tmem_ld32(ot + c * 32, o);
                            uint32_t x[32];
#pragma unroll
                            for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(o[e] * keep);
                            tmem_st32(ot + c * 32, x);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : m;
                const uint64_t scale2 = pair2(p.scale_log2, p.scale_log2), base2 = pair2(-base, -base);
                uint64_t sum[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < kKeys / 64; ++c) {
                    uint32_t x[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const uint64_t y =
                            fma2(pair2(sc[c * 64 + 2 * e], sc[c * 64 + 2 * e + 1]), scale2, base2);
                        const float a = ex2(low2(y)), b = ex2(high2(y));
                        sum[e & 1] = add2(sum[e & 1], pair2(a, b));
                        x[e] = pack2(a, b);
                    }
                    tmem_st32(st + c * 32, x);   // P over the scores, all of them read
                }
                l += (low2(sum[0]) + high2(sum[0])) + (low2(sum[1]) + high2(sum[1]));
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive(&p_full[j & 1]);
            }
            it += 2 * max(n, 0);
            advance(then);
            // O after the unit's last tile
            if (n > 0) {
                ring_wait(&o_done[(j - 1) & 1], ((j - 1) >> 1) & 1, &failed, p.error);
                __syncwarp();
                tc_fence_after();
            }
            const float inv = 1.f / l;
            float *dst = p.ws_o + ((int64_t)u.part * kRows + rt) * DH;
            __nv_bfloat16 *o_row = out + now.row * p.o_rs + now.qh * p.o_hs;
#pragma unroll 1
            for (int c = 0; c < DH / 32; ++c) {
                float o[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0.f;
                __syncwarp();
                if (n > 0) tmem_ld32(ot + c * 32, o);
                if (now.node < 0) continue;
                if (odd) {
                    // the values that were kept out of the product, for the keys that
                    // the row sees: they make the sum inf or NaN, whatever their weight
#pragma unroll 1
                    for (int key = max(u.ctx, u.t0 * kKeys); key < min(len, u.t1 * kKeys); ++key) {
                        if (!(seen_bits(p.trees, now.mask, now.node, key - u.ctx) & 1)) continue;
                        const __nv_bfloat16 *v = value_row<DH>(p, u, key) + c * 32;
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float y = __bfloat162float(v[e]);
                            if (!isfinite(y)) o[e] += y;
                        }
                    }
                }
                if (u.part >= 0) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        reinterpret_cast<float4 *>(dst + c * 32)[e] =
                            make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        reinterpret_cast<uint4 *>(o_row + c * 32)[e] = make_uint4(
                            pack2(o[8 * e] * inv, o[8 * e + 1] * inv),
                            pack2(o[8 * e + 2] * inv, o[8 * e + 3] * inv),
                            pack2(o[8 * e + 4] * inv, o[8 * e + 5] * inv),
                            pack2(o[8 * e + 6] * inv, o[8 * e + 7] * inv));
                }
            }
            if (u.part >= 0 && now.node >= 0)
                *reinterpret_cast<float2 *>(p.ws_ml + ((int64_t)u.part * kRows + rt) * 2) =
                    make_float2(m, l);
            tc_fence_before();   // O is free again when this group's next P is there
            __syncwarp();
            now = then;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, S::kTmem);
    }
}

template <int DH>
cudaError_t launch(const pk_token_kv *kv, const TreeParams &p, int workers, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(tree_tc_kernel<DH>, TcShape<DH>::kSmem, done);
    if (e != cudaSuccess) return e;
    const int ctas = workers < kv->sms ? workers : kv->sms;   // few workers: an SM each
    return launch_pdl(tree_tc_kernel<DH>, dim3(ctas), dim3(kTcThreads), TcShape<DH>::kSmem, s,
                      kv->kv_map, p);
}

}  // namespace

cudaError_t launch_tree_tc(const pk_token_kv *kv, const TreeParams &p, int workers, cudaStream_t s) {
    return kv->d.head_dim == 64 ? launch<64>(kv, p, workers, s) : launch<128>(kv, p, workers, s);
}

}  // namespace pk
