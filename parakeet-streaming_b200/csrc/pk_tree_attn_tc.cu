// Tree attention (see pk_tree_attn.cu) for row tiles of up to 128 query rows, bf16,
// on the 5th-generation tensor cores.
//
// Bound by reading K and V as long as a request's rows fit one tile: 128 keys of a
// 128-wide head are 64 KB, 2800 cycles of an SM's share of the memory rate, for
// 1024 cycles of MMAs and 1024 of exponentials, but some 2400 of a warpgroup's whole
// softmax (loads from TMEM, maximum, sum, conversions).  So one CTA an SM, and two
// softmax warpgroups that take every other tile:
//   warp 0      pages of K and V by TMA into a ring of slots (a slot: one tile of
//               K or of V), running ahead over the CTA's units
//   warp 1      one thread issues S_j = Q K_j^T (both from shared memory, fp32 in
//               TMEM, two buffers) and O += P_j V_j (P from TMEM, V from shared
//               memory as it lies: a row-major [keys][dim] tile is the MN-major
//               operand), O in TMEM, one for the even tiles and one for the odd
//   warps 4..11 a thread per row (TMEM lane), warps 4..7 for the even tiles: the row's
//               scores without a shuffle, maximum, exp2, P as bf16 over the scores,
//               fp32 sum; maxima, sums and O of the two meet at the end of a unit
// The running maximum is raised, and O scaled for it, only when a row's scores pass
// the one in use by more than 2^8: weights stay below 256, which the fp32 sums and
// bf16's exponent hold, and most tiles touch O in the MMA alone.
#include <math.h>

#include "pk_tree.cuh"
#include "pk_umma.cuh"

namespace pk {
namespace {

constexpr int kRows = 128, kKeys = 128, kTcThreads = 128 + 256;
constexpr float kRaise = 8.f;   // log2 of how far scores may pass the maximum in use

template <int DH>
struct TcShape {
    static constexpr int kSlot = kKeys * DH * 2;       // one tile of K, V or Q
    static constexpr int kGroup = DH / 64 * 1024;      // 8 rows of one
    static constexpr int kSlots = 5 * (128 / DH);      // 160 KB
    static constexpr int kSmem = (kSlots + 1) * kSlot + 1024;
    // TMEM columns: S twice (P over it), O twice
    static constexpr int kS = 0, kO = 2 * kKeys, kTmem = 512;
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
__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// barrier of one softmax group (four warps) that also ORs a flag over them
__device__ __forceinline__ bool group_any(int group, bool v) {
    uint32_t r;
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
// barrier of both groups
__device__ __forceinline__ void groups_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

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
    uint8_t *sq = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(tree_smem) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = sq + S::kSlot;
    __shared__ __align__(8) uint64_t full[NS], empty[NS], q_full, s_full[2], p_full[2], o_done[2],
        idle;
    __shared__ float s_max[2][kRows], s_sum[2][kRows];
    __shared__ int s_odd[2];
    __shared__ uint32_t tmem_base;
    __shared__ volatile int failed;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&q_full, 8);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_done[i], 1);
        }
        mbar_init(&idle, 1);
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
    auto produce = [&]() {
        // producer: lanes issue a tile's boxes, K then V
        const int ps = 1 << p.ps_shift, rows_box = min(ps, kTokRowsBox);
        const int box_of = lane;
        const uint32_t bytes = rows_box * DH * 2;
        int it = 0;
        bool stop = false;   // the warp's, so that its lanes stay together
        Work work(p, blockIdx.x);
        Pages pages, then;
        bool more = work.next();
        Unit w = work.u;
        if (more) pages.open(p, w);
        while (more && !stop) {
            more = work.next();
            if (more) then.open(p, work.u);
            const int len = w.ctx + w.count;
            for (int t = w.t0; t < w.t1 && !stop; ++t) {
                const int k0 = t * kKeys, n = (min(kKeys, len - k0) + rows_box - 1) / rows_box;
                // lanes without a box ask for the last one's page
                int page = pages.get((k0 + min(box_of, n - 1) * rows_box) >> p.ps_shift);
                if (page < 0 || page >= p.num_pages) {
                    raise(p.error, PK_DEV_BAD_PAGE);
                    page = 0;
                }
                const int in_page = (k0 + box_of * rows_box) & (ps - 1);
#pragma unroll
                for (int v = 0; v < 2; ++v, ++it) {
                    const int s = it % NS, use = it / NS;
                    if (use) ring_wait(&empty[s], (use - 1) & 1, &failed, p.error);
                    stop = __any_sync(0xffffffffu, failed != 0);
                    if (stop) break;
                    if (lane == 0) mbar_arrive_expect_tx(&full[s], n * bytes);
                    __syncwarp();
                    if (box_of < n)
                        tma_load_rows(ring + s * S::kSlot + box_of * bytes, &kv_map, &full[s], in_page,
                                      ((page * p.num_layers + p.layer) * 2 + v) * p.kv_heads + w.head);
                }
            }
            w = work.u;
            pages = then;
        }
        if (stop)   // leave no copy in flight
            for (int s = 0; s < NS; ++s)
                if (it > s) mbar_wait_bounded(&full[s], ((it - 1 - s) / NS) & 1, kWaitLimitNs);
    };
    auto multiply = [&]() {
        Work work(p, blockIdx.x);
        constexpr uint32_t id_s = idesc_bf16(kRows, kKeys);
        constexpr uint32_t id_o = idesc_bf16(kRows, DH) | (1u << 16);   // B MN-major
        const uint64_t q0 = tile_desc(smem_u32(sq), S::kGroup), ring0 = tile_desc(smem_u32(ring), S::kGroup);
        // the whole warp walks along, so that indexes and descriptors are uniform
        const bool one = elect_one();
        int it = 0, j = 0, unit = 0;   // ring use, tile and unit of this CTA
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            return __all_sync(0xffffffffu, ring_wait(bar, parity, &failed, p.error));
        };
        bool ok = true;
        // S of a tile whose K is ring use `use`, over the P of the tile two before, whose
        // product has to be done with it
        auto scores = [&](int use, int tile) {
            const int s = use % NS;
            if (tile >= 2) ok = ok && wait(&o_done[tile & 1], ((tile >> 1) - 1) & 1);
            ok = ok && wait(&full[s], (use / NS) & 1);
            if (!ok) return;
            tc_fence_after();
            if (one) {
                const uint64_t k0 = ring0 + s * (S::kSlot >> 4);
#pragma unroll
                for (int kk = 0; kk < DH / 16; ++kk) {
                    const uint32_t off = ((kk / 4) * 1024 + (kk % 4) * 32) >> 4;
                    umma_bf16(tmem + S::kS + (tile & 1) * kKeys, q0 + off, k0 + off, id_s, kk != 0);
                }
                umma_commit(&empty[s]);
                umma_commit(&s_full[tile & 1]);
            }
            __syncwarp();
        };
        while (ok && work.next()) {
            const int n = work.u.t1 - work.u.t0;
            if (n <= 0) continue;
            ok = wait(&q_full, unit & 1);
            ++unit;
            tc_fence_after();
            scores(it, j);
            for (int i = 0; i < n && ok; ++i, ++j, it += 2) {
                if (i + 1 < n) scores(it + 2, j + 1);
                const int s = (it + 1) % NS;
                ok = ok && wait(&full[s], ((it + 1) / NS) & 1) && wait(&p_full[j & 1], (j >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
                if (one) {
                    const uint64_t v0 = ring0 + s * (S::kSlot >> 4);
#pragma unroll
                    for (int kk = 0; kk < kKeys / 16; ++kk)
                        umma_bf16_ts(tmem + S::kO + (j & 1) * DH,
                                     tmem + S::kS + (j & 1) * kKeys + kk * 8,
                                     v0 + kk * (2 * S::kGroup >> 4), id_o, (i > 1) | (kk != 0));
                    umma_commit(&empty[s]);
                    umma_commit(&o_done[j & 1]);
                }
                __syncwarp();
            }
        }
        if (one) umma_commit(&idle);   // no MMA is left when the CTA frees its TMEM
        __syncwarp();
        mbar_wait_bounded(&idle, 0, kWaitLimitNs);
    };

    // a row's scores take 128 registers: 208 for the softmax warps out of the launch's
    // 168 x 384, 88 for the other warpgroup (128 x 88 + 256 x 208 = 64512)
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 0) produce();
        else if (warp == 1) multiply();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        Work work(p, blockIdx.x);
        // softmax group g takes the CTA's tiles j with j % 2 == g; thread = row (TMEM
        // lane) 32 (warp % 4) + lane of the tile
        const int g = (warp >> 2) - 1, quad = warp & 3, rt = quad * 32 + lane;
        const int gt = threadIdx.x & 127;   // thread in the group
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const uint32_t st = tmem + lanes + S::kS + g * kKeys, ot = tmem + lanes + S::kO + g * DH;
        const __nv_bfloat16 *q = static_cast<const __nv_bfloat16 *>(p.q);
        __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out);
        int it = 0, j = 0;   // ring use and tile of the unit's first tile
        while (work.next()) {
            const Unit &w = work.u;
            const int r = w.rt * kRows + rt, n = w.t1 - w.t0, len = w.ctx + w.count;
            const bool live = r < w.count * p.group;
            const int node = live ? r / p.group : -1;
            const int64_t row = w.row0 + (live ? node : 0);
            const int64_t qh = (int64_t)w.head * p.group + (live ? r - node * p.group : 0);
            uint64_t mask = 0;
            if (live && p.trees) mask = reinterpret_cast<const uint64_t *>(p.step + p.l.mask)[row];
            float m = -INFINITY, l = 0.f;   // the maximum in use (scaled), the sum
            bool odd = false;               // a value that is not finite among the own rows
            if (n > 0) {
                // the tile's queries, half a group; the MMAs that read the last ones are
                // done, since both groups have read their scores
                const uint4 *src = reinterpret_cast<const uint4 *>(q + row * p.q_rs + qh * p.q_hs);
#pragma unroll
                for (int i = 0; i < DH / 16; ++i) {
                    const int c = g * (DH / 16) + i;
                    *reinterpret_cast<uint4 *>(sq + tile_at<DH>(rt, c)) =
                        live ? src[c] : make_uint4(0u, 0u, 0u, 0u);
                }
                fence_async_proxy();
                __syncwarp();
                if (lane == 0) arrive(&q_full);
            }
            int mine = 0;   // tiles of this group in the unit
            for (int i = (g ^ j) & 1; i < n; i += 2, ++mine) {
                const int tile = j + i, use = it + 2 * i;
                const int k0 = (w.t0 + i) * kKeys;
                ring_wait(&s_full[g], (tile >> 1) & 1, &failed, p.error);
                __syncwarp();
                tc_fence_after();
                float s[kKeys];
#pragma unroll
                for (int c = 0; c < kKeys / 32; ++c)
                    tmem_ld32(st + c * 32, *reinterpret_cast<float(*)[32]>(s + c * 32));
                if (k0 + kKeys > w.ctx) {   // some of the step's own tokens, or the end
                    const int sv = (use + 1) % NS;
#pragma unroll
                    for (int c = 0; c < kKeys / 32; ++c) {
                        const uint32_t bits = seen_bits(p.trees, mask, node, k0 + c * 32 - w.ctx);
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(bits >> e & 1)) s[c * 32 + e] = -INFINITY;
                    }
                    // V rows past the end hold what the page held before, and a token's
                    // values may be inf or NaN: zero in the product, where a weight of
                    // zero would not keep them out; the epilogue adds the latter to the
                    // rows that see them
                    ring_wait(&full[sv], ((use + 1) / NS) & 1, &failed, p.error);
                    uint8_t *vs = ring + sv * S::kSlot;
                    bool bad = false;
                    for (int c = gt; c < kKeys * DH / 8; c += 128) {
                        const int vr = c / (DH / 8), ch = c % (DH / 8), key = k0 + vr;
                        if (key < w.ctx) continue;
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
                    odd |= group_any(g, bad);
                }
                float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int e = 4; e < kKeys; ++e) tops[e & 3] = fmaxf(tops[e & 3], s[e]);
                float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                top = top == -INFINITY ? top : __fmul_rn(top, p.scale_log2);
                const bool raise_it = top > m + kRaise || (m == -INFINITY && top > m);
                if (__any_sync(0xffffffffu, raise_it)) {
                    const float keep = raise_it ? ex2(m - top) : 1.f;
                    if (raise_it) m = top;
                    l *= keep;
                    if (mine > 0) {   // O has the group's tiles before
                        ring_wait(&o_done[g], ((tile >> 1) - 1) & 1, &failed, p.error);
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
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t x[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const float a = ex2(s[c * 64 + 2 * e] * p.scale_log2 - base);
                        const float b = ex2(s[c * 64 + 2 * e + 1] * p.scale_log2 - base);
                        sum[(2 * e) & 3] += a;
                        sum[(2 * e + 1) & 3] += b;
                        x[e] = pack2(a, b);
                    }
                    tmem_st32(st + c * 32, x);   // P over the scores, all of them read
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive(&p_full[g]);
            }
            // the last tile of each group in O, and the groups' maxima and sums
            const int last = j + n - 1;   // the CTA's last tile; the other group's is the one before
            if (n > 0) {
                if (n > 1 || (last & 1) == 0)
                    ring_wait(&o_done[0], ((last & 1 ? last - 1 : last) >> 1) & 1, &failed, p.error);
                if (n > 1 || (last & 1) == 1)
                    ring_wait(&o_done[1], ((last & 1 ? last : last - 1) >> 1) & 1, &failed, p.error);
                __syncwarp();
                tc_fence_after();
            }
            j += n > 0 ? n : 0;
            it += n > 0 ? 2 * n : 0;
            s_max[g][rt] = m;
            s_sum[g][rt] = l;
            if (gt == 0) s_odd[g] = odd;
            groups_sync();
            odd = s_odd[0] | s_odd[1];
            // a group without a tile has O that was never written: a factor of 0 and no
            // product with it
            const float ma = s_max[0][rt], mb = s_max[1][rt], mm = fmaxf(ma, mb);
            const float ref = mm == -INFINITY ? 0.f : mm;
            const float fa = ex2(ma - ref), fb = ex2(mb - ref);
            const float ls = fa * s_sum[0][rt] + fb * s_sum[1][rt];
            const bool has_a = n > 1 || (n == 1 && (last & 1) == 0),
                       has_b = n > 1 || (n == 1 && (last & 1) == 1);
            const float inv = 1.f / ls;
            float *dst = p.ws_o + ((int64_t)w.part * kRows + rt) * DH;
            __nv_bfloat16 *o_row = out + row * p.o_rs + qh * p.o_hs;
#pragma unroll 1
            for (int c = g * (DH / 64); c < (g + 1) * (DH / 64); ++c) {   // half the columns each
                float o[32], x[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0.f;
                if (has_a) {
                    tmem_ld32(tmem + lanes + S::kO + c * 32, x);
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = fa * x[e];
                }
                if (has_b) {
                    tmem_ld32(tmem + lanes + S::kO + DH + c * 32, x);
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] += fb * x[e];
                }
                if (!live) continue;
                if (odd) {
                    // the values that were kept out of the product, for the keys that
                    // the row sees: they make the sum inf or NaN, whatever their weight
#pragma unroll 1
                    for (int key = max(w.ctx, w.t0 * kKeys); key < min(len, w.t1 * kKeys); ++key) {
                        const int rel = key - w.ctx;
                        if (!(seen_bits(p.trees, mask, node, rel) & 1)) continue;
                        const __nv_bfloat16 *v = value_row<DH>(p, w, key) + c * 32;
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float y = __bfloat162float(v[e]);
                            if (!isfinite(y)) o[e] += y;
                        }
                    }
                }
                if (w.part >= 0) {
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
            if (g == 0 && w.part >= 0 && live)
                *reinterpret_cast<float2 *>(p.ws_ml + ((int64_t)w.part * kRows + rt) * 2) =
                    make_float2(mm, ls);
            tc_fence_before();
            groups_sync();   // O and the exchange are free again
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
cudaError_t launch(const pk_token_kv *kv, const TreeParams &p, int ctas, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(tree_tc_kernel<DH>, TcShape<DH>::kSmem, done);
    if (e != cudaSuccess) return e;
    return launch_pdl(tree_tc_kernel<DH>, dim3(ctas), dim3(kTcThreads), TcShape<DH>::kSmem, s,
                      kv->kv_map, p);
}

}  // namespace

cudaError_t launch_tree_tc(const pk_token_kv *kv, const TreeParams &p, int ctas, cudaStream_t s) {
    return kv->d.head_dim == 64 ? launch<64>(kv, p, ctas, s) : launch<128>(kv, p, ctas, s);
}

}  // namespace pk
