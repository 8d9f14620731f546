// Attention of a step's token rows over a token pool: each row sees its
// request's context and, of the step's own tokens, its ancestors (or, in a
// chain, the rows before it) and itself.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j - m),  m = max_j
//
// One pass over the keys in tiles of 64 with a running maximum and sum (fp32).
// The rows of a K/V head are its group's query heads of every token, so a
// request's pages are read once for all of them that fit a row tile.  The step's
// work is a line of (row tile, key tile) pairs that is cut into equal shares, one a
// worker, whatever the lengths; a second launch joins the row tiles that a cut went
// through (two partial results a worker at most).
//
// bf16, row tiles of 16: every warp is a worker of its own, with a share of the line and
// two slots of shared memory, one for a tile of 64 keys and one for its V (TMA, a page a
// copy, 128B swizzle).  It requests the next K as soon as it has read one and the next
// V likewise, across its units, computes S = Q K^T and O += P V with mma.sync m16n8k16
// and waits for nobody: 12 such chains an SM for 64-wide heads, 6 for 128, hide each
// other's latencies.  Where every worker has the same, memory bounds it (160 requests of
// 505 tokens, 8 heads of 64, eight key tiles a warp: 36 us, 4.6 TB/s); where lengths differ
// and a worker has one row tile, the longest one's chain does (62 to 500 tokens: 27 us for
// 97 MB).  Warps that shared a row tile met in a barrier at its end and cost 5000 cycles a
// row tile, however short (the same: 41 us).
// P is rounded to bf16 for the product, by 2^-8 of each weight at most, as the bf16 V
// that it multiplies has been; the sum that normalises keeps fp32 weights.  Every wait is
// bounded: one that runs out sets PK_DEV_TIMEOUT, and the CTA's other waits return at once.
#include <math.h>

#include "pk_tree.cuh"

namespace pk {
namespace {

constexpr int kTile = kTokRowsBox;   // keys
// Workers (warps) of a CTA and CTAs an SM: what registers and shared memory hold.
template <int DH> struct TreeShape {
    static constexpr int kWarps = tok_warps(DH), kCtas = tok_workers(DH) / kWarps;
    static constexpr int kSlot = kTile * DH * 2;   // a tile of K or of V
    static constexpr int kSmem = kWarps * 2 * kSlot + 1024;
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Whether row `node` sees the step's token `rel` (>= 0) of its request.
__device__ __forceinline__ bool sees(int trees, uint64_t mask, int node, int rel) {
    return trees ? rel < PK_TOK_MAX_TREE && ((mask >> rel) & 1) : rel <= node;
}

// Bit j: whether a row sees key rel0 + j, counted from the step's first token.
__device__ __forceinline__ uint64_t seen_keys(int trees, uint64_t mask, int node, int rel0) {
    if (rel0 <= -64) return ~0ull;
    if (!trees) {
        const int n = node - rel0 + 1;   // keys up to the row's own
        return n <= 0 ? 0ull : (n >= 64 ? ~0ull : (1ull << n) - 1ull);
    }
    if (rel0 >= PK_TOK_MAX_TREE) return 0ull;
    return rel0 >= 0 ? mask >> rel0 : (mask << -rel0) | ((1ull << -rel0) - 1ull);
}

// V rows past the end hold what the page held before, and a token's values may be inf or
// NaN: zero in the product, where a weight of zero would not keep them from the rows
// that do not see them.  Returns whether there were any of the latter.  By one warp.
template <int DH>
__device__ __forceinline__ bool clean_values(uint8_t *vs, int k0, int ctx, int len) {
    bool odd = false;
    for (int c = max(ctx - k0, 0) * (DH / 8) + (threadIdx.x & 31); c < kTile * DH / 8; c += 32) {
        const int row = c / (DH / 8), ch = c % (DH / 8);
        uint4 *at = reinterpret_cast<uint4 *>(vs + tile_at<DH>(row, ch));
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (k0 + row < len) {
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
            odd = true;
        }
        *at = x;
    }
    fence_async_proxy();   // the slot's next TMA load comes after these writes
    const bool any = __any_sync(0xffffffffu, odd);   // (and the warp's writes before its reads)
    __syncwarp();
    return any;
}

template <int kWarps> struct TreeShared {
    uint64_t full[kWarps][2];   // K and V of each worker
    float2 ml[kWarps][16];
    int failed;
};

// One worker's share; or, kTeam, one warp's part of the CTA's row tile: every kWarps-th
// key tile, the warps meeting at the end.
template <int DH, bool kTeam>
__device__ __forceinline__ void attend(const CUtensorMap &kv_map, const TreeParams &p, uint8_t *smem,
                                       TreeShared<TreeShape<DH>::kWarps> &sh) {
    constexpr int kWarps = TreeShape<DH>::kWarps, kSlot = TreeShape<DH>::kSlot, kN = kTile / 8;
    constexpr int kStride = kTeam ? kWarps : 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t *ks = smem + warp * 2 * kSlot, *vs = ks + kSlot;
    const uint32_t kb = smem_u32(ks), vb = smem_u32(vs);
    uint64_t *full = sh.full[warp];
    volatile int *failed = &sh.failed;

    const int ps = 1 << p.ps_shift, rows_box = min(ps, kTile);
    int page = 0;   // of this lane's rows of the tile requested last
    // request V of tile t of a unit, whose K has been; K of one: a page a lane
    auto request_rows = [&](const Unit &w, int t, int v) {
        const int k0 = t * kTile;
        const int n = (min(kTile, w.ctx + w.count - k0) + rows_box - 1) / rows_box;
        const uint32_t bytes = rows_box * DH * 2;
        if (lane == 0) mbar_arrive_expect_tx(&full[v], n * bytes);
        __syncwarp();
        if (lane < n)
            tma_load_rows((v ? vs : ks) + lane * bytes, &kv_map, &full[v],
                          (k0 + lane * rows_box) & (ps - 1),
                          ((page * p.num_layers + p.layer) * 2 + v) * p.kv_heads + w.head);
    };
    auto request_keys = [&](const Unit &w, Pages &pages, int t) {
        const int k0 = t * kTile;
        const int last = (min(kTile, w.ctx + w.count - k0) - 1) / rows_box;
        // lanes without rows ask for the last page
        page = pages.get((k0 + min(lane, last) * rows_box) >> p.ps_shift);
        if (page < 0 || page >= p.num_pages) {
            raise(p.error, PK_DEV_BAD_PAGE);
            page = 0;
        }
        request_rows(w, t, 0);
    };

    const __nv_bfloat16 *q = static_cast<const __nv_bfloat16 *>(p.q);
    __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out);
    // neighbouring shares on different SMs
    Work work(p, kTeam ? blockIdx.x : warp * gridDim.x + blockIdx.x);
    // units that have tiles (a chain's rows may see none of a share's)
    auto advance = [&]() {
        while (work.next()) {
            if (kTeam) work.u.t0 += warp;
            if (work.u.t0 < work.u.t1 || kTeam) return true;
            if (work.u.part >= 0 && lane < 16)   // nothing seen: no weight in the join
                *reinterpret_cast<float2 *>(p.ws_ml + ((int64_t)work.u.part * 16 + lane) * 2) =
                    make_float2(-INFINITY, 0.f);
        }
        return false;
    };
    bool more = advance();
    Unit w = work.u;
    Pages pages, then;
    if (more && w.t0 < w.t1) {
        pages.open(p, w);
        request_keys(w, pages, w.t0);
        request_rows(w, w.t0, 1);
    }
    uint32_t phase = 0;   // of both barriers: one use a tile
    while (more) {
        const int m_rows = w.count * p.group, len = w.ctx + w.count;
        // this thread's two rows of the tile (fragment rows lane / 4 and + 8)
        uint32_t qf[DH / 16][4];
        uint64_t mask[2];
        int node[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = w.rt * 16 + (lane >> 2) + h * 8;
            node[h] = -1;
            mask[h] = 0;
            const __nv_bfloat16 *src = nullptr;
            if (r < m_rows) {
                node[h] = r / p.group;
                const int64_t row = w.row0 + node[h];
                if (p.trees)
                    mask[h] = reinterpret_cast<const uint64_t *>(p.step + p.l.mask)[row];
                src = q + row * p.q_rs +
                      (int64_t)(w.head * p.group + r - node[h] * p.group) * p.q_hs + (lane & 3) * 2;
            }
#pragma unroll
            for (int c = 0; c < DH / 16; ++c) {
                qf[c][h] = src ? *reinterpret_cast<const uint32_t *>(src + c * 16) : 0u;
                qf[c][h + 2] = src ? *reinterpret_cast<const uint32_t *>(src + c * 16 + 8) : 0u;
            }
        }
        // the next unit is known before this one is computed
        more = advance();
        if (more) then.open(p, work.u);
        float o[DH / 8][4];
#pragma unroll
        for (int i = 0; i < DH / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};   // maxima scaled

        for (int t = w.t0; t < w.t1; t += kStride, phase ^= 1) {
            const int k0 = t * kTile;
            const bool own = k0 + kTile > w.ctx;   // some of the step's own tokens, or the end
            // (a wait that gave up: nothing more is requested)
            if (!__all_sync(0xffffffffu, ring_wait(&full[0], phase, failed, p.error))) break;
            float s[kN][4];
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
            for (int c = 0; c < DH / 16; ++c) {
#pragma unroll
                for (int nb = 0; nb < kN / 2; ++nb) {
                    uint32_t b[4];
                    const uint32_t row = nb * 16 + ((lane >> 4) << 3) + (lane & 7);
                    ldsm4(kb + tile_at<DH>(row, c * 2 + ((lane >> 3) & 1)), b);
                    mma16816(s[2 * nb], qf[c], b[0], b[1]);
                    mma16816(s[2 * nb + 1], qf[c], b[2], b[3]);
                }
            }
            __syncwarp();
            const bool here = t + kStride < w.t1;   // the next tile is this unit's
            if (here) request_keys(w, pages, t + kStride);
            else if (more) request_keys(work.u, then, work.u.t0);
            if (own) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // bit j: key j of this thread's (no row sees a key past the end)
                    const uint64_t bits =
                        seen_keys(p.trees, mask[h], node[h], k0 - w.ctx) >> ((lane & 3) * 2);
#pragma unroll
                    for (int n = 0; n < kN; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (!(bits >> (n * 8 + e) & 1)) s[n][2 * h + e] = -INFINITY;
                }
            }
            float keep[2], base[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float top = fmaxf(s[0][2 * h], s[0][2 * h + 1]);
#pragma unroll
                for (int n = 1; n < kN; ++n)
                    top = fmaxf(top, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // (-inf stays so; a product rounded alike keeps an unchanged maximum's
                // factor at 1)
                top = fmaxf(m[h], top == -INFINITY ? top : __fmul_rn(top, p.scale_log2));
                // nothing seen yet: weights and factor are exp2(-inf) = 0
                base[h] = top == -INFINITY ? 0.f : top;
                keep[h] = ex2(m[h] - base[h]);
                m[h] = top;
                float sum = 0.f;
#pragma unroll
                for (int n = 0; n < kN; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float x = ex2(s[n][2 * h + e] * p.scale_log2 - base[h]);
                        s[n][2 * h + e] = x;
                        sum += x;
                    }
                l[h] = l[h] * keep[h] + sum;
            }
#pragma unroll
            for (int n = 0; n < DH / 8; ++n) {
                o[n][0] *= keep[0];
                o[n][1] *= keep[0];
                o[n][2] *= keep[1];
                o[n][3] *= keep[1];
            }
            if (!__all_sync(0xffffffffu, ring_wait(&full[1], phase, failed, p.error))) break;
            // values that are not finite among the step's own rows
            const bool odd = own && clean_values<DH>(vs, k0, w.ctx, len);
#pragma unroll
            for (int kk = 0; kk < kN / 2; ++kk) {
                const uint32_t a[4] = {
                    pack2(s[2 * kk][0], s[2 * kk][1]), pack2(s[2 * kk][2], s[2 * kk][3]),
                    pack2(s[2 * kk + 1][0], s[2 * kk + 1][1]),
                    pack2(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
                for (int nb = 0; nb < DH / 16; ++nb) {
                    uint32_t b[4];
                    ldsm4_t(vb + tile_at<DH>(kk * 16 + (lane & 15), nb * 2 + (lane >> 4)), b);
                    mma16816(o[2 * nb], a, b[0], b[1]);
                    mma16816(o[2 * nb + 1], a, b[2], b[3]);
                }
            }
            if (odd) {
                // the values kept out of the product, to the rows that see their keys:
                // they make the sum inf or NaN, whatever their weight
#pragma unroll 1
                for (int key = max(w.ctx, k0); key < min(len, k0 + kTile); ++key) {
                    const __nv_bfloat16 *v = value_row<DH>(p, w, key) + (lane & 3) * 2;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (!(seen_keys(p.trees, mask[h], node[h], key - w.ctx) & 1)) continue;
#pragma unroll
                        for (int n = 0; n < DH / 8; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float x = __bfloat162float(v[n * 8 + e]);
                                if (!isfinite(x)) o[n][2 * h + e] += x;
                            }
                    }
                }
            }
            __syncwarp();
            if (here) request_rows(w, t + kStride, 1);
            else if (more) request_rows(work.u, work.u.t0, 1);
        }
        // row sums over the quad's lanes
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        }
        if (kTeam) {
            // the warps' rows in their slots (all copies have been waited for)
            float *mine = reinterpret_cast<float *>(ks);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int rt = (lane >> 2) + h * 8;
#pragma unroll
                for (int n = 0; n < DH / 8; ++n)
                    *reinterpret_cast<float2 *>(mine + rt * DH + n * 8 + (lane & 3) * 2) =
                        make_float2(o[n][2 * h], o[n][2 * h + 1]);
                if ((lane & 3) == 0) sh.ml[warp][rt] = make_float2(m[h], l[h]);
            }
            __syncthreads();
            const float *all = reinterpret_cast<const float *>(smem);
            for (int c = threadIdx.x; c < 16 * DH / 2; c += kWarps * 32) {
                const int rt = c / (DH / 2), col = c % (DH / 2) * 2, r = w.rt * 16 + rt;
                if (r >= m_rows) continue;
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < kWarps; ++k) top = fmaxf(top, sh.ml[k][rt].x);
                const float ref = top == -INFINITY ? 0.f : top;
                float x = 0.f, y = 0.f, sum = 0.f;
#pragma unroll
                for (int k = 0; k < kWarps; ++k) {
                    const float f = ex2(sh.ml[k][rt].x - ref);
                    const float2 v = *reinterpret_cast<const float2 *>(
                        all + k * (2 * kSlot / 4) + rt * DH + col);
                    sum += f * sh.ml[k][rt].y;
                    x += f * v.x;
                    y += f * v.y;
                }
                const int nd = r / p.group;
                *reinterpret_cast<uint32_t *>(
                    out + (int64_t)(w.row0 + nd) * p.o_rs +
                    (int64_t)(w.head * p.group + r - nd * p.group) * p.o_hs + col) =
                    pack2(x / sum, y / sum);
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int rt = (lane >> 2) + h * 8, r = w.rt * 16 + rt;
                if (r >= m_rows) continue;
                if (w.part >= 0) {
                    const int64_t at = (int64_t)w.part * 16 + rt;
                    float *dst = p.ws_o + at * DH + (lane & 3) * 2;
#pragma unroll
                    for (int n = 0; n < DH / 8; ++n)
                        *reinterpret_cast<float2 *>(dst + n * 8) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
                    if ((lane & 3) == 0)
                        *reinterpret_cast<float2 *>(p.ws_ml + at * 2) = make_float2(m[h], l[h]);
                } else {
                    const float inv = 1.f / l[h];
                    __nv_bfloat16 *dst =
                        out + (int64_t)(w.row0 + node[h]) * p.o_rs +
                        (int64_t)(w.head * p.group + r - node[h] * p.group) * p.o_hs + (lane & 3) * 2;
#pragma unroll
                    for (int n = 0; n < DH / 8; ++n)
                        *reinterpret_cast<uint32_t *>(dst + n * 8) =
                            pack2(o[n][2 * h] * inv, o[n][2 * h + 1] * inv);
                }
            }
        }
        w = work.u;
        pages = then;
    }
    if (*failed) {   // leave no copy in flight: this tile's, or the next one's K
        mbar_wait_bounded(&full[0], phase, kWaitLimitNs);
        mbar_wait_bounded(&full[1], phase, kWaitLimitNs);
        mbar_wait_bounded(&full[0], phase ^ 1, kWaitLimitNs);
    }
}

template <int DH>
__global__ void __launch_bounds__(TreeShape<DH>::kWarps * 32, TreeShape<DH>::kCtas)
    tree_attn_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ TreeParams p) {
    extern __shared__ uint8_t tree_smem[];
    constexpr int kWarps = TreeShape<DH>::kWarps;
    __shared__ __align__(8) TreeShared<kWarps> sh;
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(tree_smem) + 1023) & ~uintptr_t(1023));
    if (threadIdx.x == 0) {
        for (int w = 0; w < kWarps; ++w) {
            mbar_init(&sh.full[w][0], 1);
            mbar_init(&sh.full[w][1], 1);
        }
        sh.failed = 0;
        fence_mbar_init();
        prefetch_tmap(&kv_map);
    }
    __syncthreads();
    grid_dep_wait();
    grid_dep_launch();
    // a CTA for every row tile (short requests, few of them): its warps are a team
    if (p.step[kTokShare] == 0 &&
        reinterpret_cast<const int64_t *>(p.step + p.l.work)[p.batch] <= gridDim.x)
        attend<DH, true>(kv_map, p, smem, sh);
    else
        attend<DH, false>(kv_map, p, smem, sh);
}

// ------------------------------------------------------------------ float32
// The parity mode: the same units, fp32 FMAs.  A CTA of four warps holds a
// 16-row tile; K rows are padded so that a lane per key reads without bank
// conflicts; a warp computes the scores of its four rows (two keys a lane), then
// their outputs (DH / 32 columns a lane).
constexpr int kRowsF32 = 16;
template <int DH>
__global__ void __launch_bounds__(128, 3) tree_attn_f32_kernel(const TreeParams p) {
    constexpr int kKp = DH + 4, NV = DH / 32;
    extern __shared__ uint8_t tree_smem[];
    float *sk = reinterpret_cast<float *>(tree_smem);   // [kTile][kKp]
    float *sv = sk + kTile * kKp;                       // [kTile][DH]
    float *sq = sv + kTile * DH;                        // [kRowsF32][DH]
    float *sp = sq + kRowsF32 * DH;                     // [kRowsF32][kTile]
    grid_dep_wait();
    grid_dep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float *q = static_cast<const float *>(p.q), *kv = static_cast<const float *>(p.kv);
    float *out = static_cast<float *>(p.out);
    Work work(p, blockIdx.x);
    while (work.next()) {
        const Unit &w = work.u;
        const int head = w.head, m_rows = w.count * p.group, len = w.ctx + w.count;
        __syncthreads();
        for (int c = threadIdx.x; c < kRowsF32 * DH / 4; c += 128) {
            const int rt = c / (DH / 4), e = c % (DH / 4), r = w.rt * kRowsF32 + rt;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < m_rows) {
                const int nd = r / p.group;
                x = *reinterpret_cast<const float4 *>(
                    q + (int64_t)(w.row0 + nd) * p.q_rs +
                    (int64_t)(head * p.group + r - nd * p.group) * p.q_hs + e * 4);
            }
            reinterpret_cast<float4 *>(sq)[c] = x;
        }
        float o[4][NV] = {}, m[4], l[4];
        // the warp's rows are warp, warp + 4, ..: as many as are live
        const int rows = (min(m_rows - w.rt * kRowsF32, kRowsF32) + 3 - warp) >> 2;
        uint64_t mask[4];
        int node[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = w.rt * kRowsF32 + i * 4 + warp;
            m[i] = -INFINITY;
            l[i] = 0.f;
            node[i] = r < m_rows ? r / p.group : -1;
            mask[i] = p.trees && r < m_rows
                          ? reinterpret_cast<const uint64_t *>(p.step + p.l.mask)[w.row0 + node[i]]
                          : 0;
        }
        for (int t = w.t0; t < w.t1; ++t) {
            const int k0 = t * kTile;
            __syncthreads();   // the previous tile is done with
            // eight chunks at a time, so that their table entries and then their rows are
            // requested together
            for (int c0 = threadIdx.x; c0 < kTile * DH / 4; c0 += 8 * 128) {
                int page[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int key = k0 + (c0 + i * 128) / (DH / 4);
                    page[i] = 0;
                    if (key < len)
                        page[i] = p.table[(int64_t)w.slot * p.table_width + (key >> p.ps_shift)];
                }
                float4 a[8], b[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int c = c0 + i * 128, e = c % (DH / 4), key = k0 + c / (DH / 4);
                    a[i] = b[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (page[i] < 0 || page[i] >= p.num_pages) {
                        raise(p.error, PK_DEV_BAD_PAGE);
                        page[i] = 0;
                    }
                    if (key < len) {
                        const int64_t ps = 1 << p.ps_shift, off = key & (ps - 1);
                        const int64_t plane =
                            (((int64_t)page[i] * p.num_layers + p.layer) * 2) * p.kv_heads + head;
                        const float *src = kv + (plane * ps + off) * DH + e * 4;
                        a[i] = *reinterpret_cast<const float4 *>(src);
                        b[i] = *reinterpret_cast<const float4 *>(src + p.kv_heads * ps * DH);
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int c = c0 + i * 128, row = c / (DH / 4), e = c % (DH / 4);
                    *reinterpret_cast<float4 *>(sk + row * kKp + e * 4) = a[i];
                    reinterpret_cast<float4 *>(sv)[c] = b[i];
                }
            }
            __syncthreads();
            float s[4][2] = {};
#pragma unroll 4
            for (int e = 0; e < DH / 4; ++e) {
                const float4 a = *reinterpret_cast<const float4 *>(sk + lane * kKp + e * 4);
                const float4 b = *reinterpret_cast<const float4 *>(sk + (lane + 32) * kKp + e * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (i >= rows) break;
                    const float4 x =
                        *reinterpret_cast<const float4 *>(sq + (i * 4 + warp) * DH + e * 4);
                    s[i][0] += x.x * a.x + x.y * a.y + x.z * a.z + x.w * a.w;
                    s[i][1] += x.x * b.x + x.y * b.y + x.z * b.z + x.w * b.w;
                }
            }
            const bool own = k0 + kTile > w.ctx;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i >= rows) break;
                float top = m[i];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int key = k0 + lane + 32 * h, rel = key - w.ctx;
                    if (own && (key >= len ||
                                (rel >= 0 && !sees(p.trees, mask[i], node[i], rel))))
                        s[i][h] = -INFINITY;
                    top = fmaxf(top, s[i][h]);
                }
#pragma unroll
                for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                // exp2 of the scaled difference, so that large scores lose nothing
                const float ref = top == -INFINITY ? 0.f : top;
                const float keep = exp2f((m[i] - ref) * p.scale_log2);
                const float a = exp2f((s[i][0] - ref) * p.scale_log2);
                const float b = exp2f((s[i][1] - ref) * p.scale_log2);
                m[i] = top;
                l[i] = l[i] * keep + a + b;
#pragma unroll
                for (int n = 0; n < NV; ++n) o[i][n] *= keep;
                // a key that the row does not see: -0, so that a weight too small for
                // fp32 keeps its value's inf or NaN
                sp[(i * 4 + warp) * kTile + lane] = s[i][0] == -INFINITY ? -0.f : a;
                sp[(i * 4 + warp) * kTile + lane + 32] = s[i][1] == -INFINITY ? -0.f : b;
            }
            __syncwarp();
            // (rows past the end were staged as zeros, their weights are zero)
#pragma unroll 2
            for (int j = 0; j < kTile; j += 4) {
                float v[4][NV];
                float4 x[4];   // the four rows' weights of the four keys
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int n = 0; n < NV; ++n) v[k][n] = sv[(j + k) * DH + n * 32 + lane];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (i >= rows) break;
                    x[i] = *reinterpret_cast<const float4 *>(sp + (i * 4 + warp) * kTile + j);
                    const float y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int n = 0; n < NV; ++n)   // an unseen key has no part, even inf
                            o[i][n] += __float_as_int(y[k]) >= 0 ? y[k] * v[k][n] : 0.f;
                }
            }
            __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int rt = i * 4 + warp, r = w.rt * kRowsF32 + rt;
            if (i >= rows) break;
            float sum = l[i];
#pragma unroll
            for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            if (w.part >= 0) {
                const int64_t part = (int64_t)w.part * kRowsF32 + rt;
#pragma unroll
                for (int n = 0; n < NV; ++n) p.ws_o[part * DH + n * 32 + lane] = o[i][n];
                if (lane == 0) {
                    p.ws_ml[part * 2] = m[i] * p.scale_log2;
                    p.ws_ml[part * 2 + 1] = sum;
                }
            } else {
                const float inv = 1.f / sum;
                float *dst = out + (int64_t)(w.row0 + node[i]) * p.o_rs +
                             (int64_t)(head * p.group + r - node[i] * p.group) * p.o_hs;
#pragma unroll
                for (int n = 0; n < NV; ++n) dst[n * 32 + lane] = o[i][n] * inv;
            }
        }
    }
}

// ------------------------------------------------------------------ the join
// For every (row, head) its row tile's partial results - of the workers whose shares
// cut the tile's keys - weighted by exp2(m - max m), in order of the keys, so that the
// result does not depend on which worker finished first.  A warp an entry, or, with few
// entries (kTeam), a block: each warp every eighth partial, then the warps' sums.
template <int DH, typename T, bool kTeam>
__global__ void __launch_bounds__(256) tree_join_kernel(const TreeParams p) {
    constexpr int NV = DH / 32;
    __shared__ float s_acc[8][DH], s_sum[8];
    grid_dep_launch();
    const int64_t share = p.step[kTokShare];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t n = (int64_t)p.rows * p.heads;
    const int bm = p.shape.rows;
    const int64_t *work = reinterpret_cast<const int64_t *>(p.step + p.l.work);
    // the workers of entry i, and where the first one's partial of its row lies
    auto find = [&](int64_t i, int &c0, int &c1, int &in_tile) {
        if (i >= n) return false;
        const int row = (int)(i / p.heads), qh = (int)(i - (int64_t)row * p.heads);
        const int b = p.step[p.l.request + row];
        if (b < 0) return false;
        const int ctx = p.step[p.l.context + b];
        if (ctx < 0) return false;
        const int r0 = p.step[p.l.row_start + b], cnt = p.step[p.l.row_start + b + 1] - r0;
        const int head = qh / p.group, r = (row - r0) * p.group + qh - head * p.group;
        const int nr = (cnt * p.group + bm - 1) / bm, rt = r / bm;
        const int kt = (ctx + cnt + p.shape.keys - 1) / p.shape.keys;
        in_tile = r - rt * bm;
        return shared_by(p, work[b] + ((int64_t)head * nr + rt) * (kt + p.shape.lead), kt, share, c0,
                         c1);
    };
    auto at = [&](int c, int c0, int in_tile) {   // the first worker's last unit, the others' first
        return ((int64_t)2 * c + (c == c0)) * bm + in_tile;
    };
    // sums workers c0 + w0, + step, ..: outputs and the sum, relative to exp2(top)
    auto add = [&](int c0, int c1, int in_tile, float top, int w0, int step, float (&acc)[NV]) {
        float sum = 0.f;
#pragma unroll 8
        for (int c = c0 + w0; c <= c1; c += step) {
            const int64_t k = at(c, c0, in_tile);
            const float2 ml = *reinterpret_cast<const float2 *>(p.ws_ml + k * 2);
            const bool saw = ml.x != -INFINITY;   // (a part that saw nothing wrote no outputs)
            const float f = saw ? exp2f(ml.x - top) : 0.f;
            sum += f * ml.y;
            const float *src = p.ws_o + k * DH + lane * NV;
#pragma unroll
            for (int e = 0; e < NV; ++e) {
                const float x = src[e];
                acc[e] += saw ? f * x : 0.f;
            }
        }
        return sum;
    };
    auto highest = [&](int c0, int c1, int in_tile) {
        float top = -INFINITY;
        for (int c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, p.ws_ml[at(c, c0, in_tile) * 2]);
#pragma unroll
        for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        return top == -INFINITY ? 0.f : top;
    };
    auto store = [&](int64_t i, const float (&acc)[NV], float sum) {
        const int64_t row = i / p.heads, qh = i - row * p.heads;
        T *dst = static_cast<T *>(p.out) + row * p.o_rs + qh * p.o_hs + lane * NV;
        const float inv = 1.f / sum;
#pragma unroll
        for (int e = 0; e < NV; ++e) dst[e] = Elem<T>::from_f(acc[e] * inv);
    };
    const int step = kTeam ? 8 : 1, first = kTeam ? warp : 0;
    const int64_t i0 = kTeam ? blockIdx.x : (int64_t)blockIdx.x * 8 + warp;
    int c0, c1, in_tile;
    // the step's tables are older than the kernel before, which has waited for them: the
    // first entry is found while that one ends
    bool cut = share > 0 && find(i0, c0, c1, in_tile);
    grid_dep_wait();
    if (share == 0) return;
    for (int64_t i = i0; i < n; i += (int64_t)gridDim.x * (kTeam ? 1 : 8)) {
        if (i != i0) cut = find(i, c0, c1, in_tile);
        if (!cut) continue;
        float acc[NV] = {};
        const float top = highest(c0, c1, in_tile);
        const float sum = add(c0, c1, in_tile, top, first, step, acc);
        if (kTeam) {
#pragma unroll
            for (int e = 0; e < NV; ++e) s_acc[warp][lane * NV + e] = acc[e];
            if (lane == 0) s_sum[warp] = sum;
            __syncthreads();
            if (warp == 0) {
                float total = 0.f;
#pragma unroll
                for (int e = 0; e < NV; ++e) acc[e] = 0.f;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    total += s_sum[x];
#pragma unroll
                    for (int e = 0; e < NV; ++e) acc[e] += s_acc[x][lane * NV + e];
                }
                store(i, acc, total);
            }
            __syncthreads();
        } else {
            store(i, acc, sum);
        }
    }
}

template <int DH>
cudaError_t launch_dim(const pk_token_kv *kv, const TreeParams &p, int workers, cudaStream_t s) {
    if (kv->d.dtype == PK_DTYPE_BF16) {
        static std::atomic<uint64_t> done{0};
        using S = TreeShape<DH>;
        constexpr int smem = S::kSmem;
        cudaError_t e = allow_smem(tree_attn_kernel<DH>, smem, done);
        if (e != cudaSuccess) return e;
        // few workers: one a CTA, on an SM of its own
        const int most = S::kCtas * kv->sms, ctas = workers < most ? workers : most;
        return launch_pdl(tree_attn_kernel<DH>, dim3(ctas), dim3(S::kWarps * 32), smem, s, kv->kv_map, p);
    }
    const int ctas = workers;
    static std::atomic<uint64_t> done{0};
    constexpr int smem = (kTile * (DH + 4) + kTile * DH + kRowsF32 * DH + kRowsF32 * kTile) * 4;
    cudaError_t e = allow_smem(tree_attn_f32_kernel<DH>, smem, done);
    if (e != cudaSuccess) return e;
    return launch_pdl(tree_attn_f32_kernel<DH>, dim3(ctas), dim3(128), smem, s, p);
}
template <int DH, typename T>
cudaError_t launch_join(const TreeParams &p, int sms, cudaStream_t s) {
    const int64_t n = (int64_t)p.rows * p.heads, most = 8 * (int64_t)sms;
    if (n <= most)
        return launch_pdl(tree_join_kernel<DH, T, true>, dim3((unsigned)n), dim3(256), 0, s, p);
    const int64_t ctas = (n + 7) / 8;
    return launch_pdl(tree_join_kernel<DH, T, false>, dim3((unsigned)(ctas < most ? ctas : most)),
                      dim3(256), 0, s, p);
}

// Most row tiles of a step.
int64_t max_items(const pk_token_kv *kv, int batch, int rows, const TokShape &sh) {
    return ((int64_t)rows * kv->group / sh.rows + batch) * kv->d.num_kv_heads;
}
// No row tile of such a step is shared by workers: as begin_plan decides, for the
// longest requests that the pool holds.
bool never_shared(const pk_token_kv *kv, int batch, int rows, const TokShape &sh) {
    const int64_t items = max_items(kv, batch, rows, sh), per = (items + sh.ctas - 1) / sh.ctas;
    const int64_t longest = (((int64_t)kv->d.table_width << kv->ps_shift) + sh.keys - 1) / sh.keys;
    return per * (longest + sh.lead) <= sh.least + sh.lead ||
           (items <= sh.team && longest <= sh.team_keys);
}

}  // namespace

int64_t tree_attn_workspace(const pk_token_kv *kv, int batch, int rows) {
    const TokShape sh = tok_shape(kv, batch, rows);
    return never_shared(kv, batch, rows, sh) ? 0
                                             : (int64_t)2 * sh.ctas * sh.rows * (kv->d.head_dim + 2) * 4;
}

int launch_tree_attention(const pk_token_kv *kv, const TreeAttnArgs &a, cudaStream_t s) {
    const pk_token_kv_desc &d = kv->d;
    TreeParams p;
    p.step = a.step;
    p.table = d.page_table;
    p.l = tok_layout(kv, a.batch, a.rows, a.trees);
    p.shape = tok_shape(kv, a.batch, a.rows);
    p.table_width = d.table_width;
    p.num_pages = d.num_pages;
    p.num_layers = d.num_layers;
    p.layer = a.layer;
    p.kv_heads = d.num_kv_heads;
    p.group = kv->group;
    p.ps_shift = kv->ps_shift;
    p.trees = a.trees;
    p.batch = a.batch;
    p.rows = a.rows;
    p.heads = d.num_heads;
    p.q = a.q;
    p.kv = d.kv;
    p.out = a.out;
    p.q_rs = a.q_rs;
    p.q_hs = a.q_hs;
    p.o_rs = a.o_rs;
    p.o_hs = a.o_hs;
    p.scale_log2 = a.scale * 1.44269504088896340736f;
    p.ws_o = a.ws;
    p.ws_ml = a.ws ? a.ws + (int64_t)2 * p.shape.ctas * p.shape.rows * d.head_dim : nullptr;
    p.error = d.error;
    const bool shared = !never_shared(kv, a.batch, a.rows, p.shape);
    // workers without a row tile are not started
    const int64_t items = max_items(kv, a.batch, a.rows, p.shape);
    const int ctas = shared || items > p.shape.ctas ? p.shape.ctas : (int)items;
    cudaError_t e = p.shape.rows == 128 ? launch_tree_tc(kv, p, ctas, s)
                    : d.head_dim == 64  ? launch_dim<64>(kv, p, ctas, s)
                                        : launch_dim<128>(kv, p, ctas, s);
    if (e != cudaSuccess) return cuda_status(e, "tree attention kernel");
    if (!shared) return PK_OK;
    if (d.dtype == PK_DTYPE_BF16)
        e = d.head_dim == 64 ? launch_join<64, __nv_bfloat16>(p, kv->sms, s)
                             : launch_join<128, __nv_bfloat16>(p, kv->sms, s);
    else
        e = d.head_dim == 64 ? launch_join<64, float>(p, kv->sms, s)
                             : launch_join<128, float>(p, kv->sms, s);
    return cuda_status(e, "tree_join_kernel");
}

}  // namespace pk
