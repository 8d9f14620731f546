// A projection shared by many requests, with each request's low-rank adapter:
//
//   acc[m] = x[m] W^T + S[m] up[a]^T,   S[m] = scale[a] * x[m] down[a]^T,  a = ids[m]
//   C[m]   = epilogue(acc[m])           (rows with ids[m] = -1: x[m] W^T alone)
//
// Three launches:
//  1. the plan (once per step: every projection of a model uses the same ids)
//     sorts the rows by adapter, so that a 128-row tile meets few adapters, and
//     lists each tile's (adapter, rows) pairs; an adapter's rows stay in their order, and
//     the rows of a single tile in theirs;
//  2. S in bf16 and the rows' sorted copy, bound by reading and writing them;
//  3. the product on the tcgen05 tensor cores, over the sorted rows; after the K
//     blocks of x W^T each pair of the tile adds one K block S up[a]^T into the same
//     accumulator, with the lanes of other rows disabled in the MMA: they get no zero
//     products, so one adapter's weights, whatever they hold, do not reach another's
//     rows.  The epilogue writes the rows back to their own places.  Rows that need no
//     sorted copy are read before launch 2 is done.
//
// S is rounded to bf16 because the tensor cores take it so: off by 2^-8 of each of
// its terms at most, as the bf16 result is of their sum.  Sums are
// fp32 throughout and in an order that the ids alone give.
#include "pk_common.cuh"
#include "pk_internal.h"
#include "pk_umma.cuh"

namespace pk {
namespace {

constexpr int kTileRows = 128;

// An adapter and its rows of a tile.
struct TilePair {
    int adapter;
    uint32_t rows[4];
};
__device__ __forceinline__ void store_pair(int32_t *at, int adapter, const uint32_t (&rows)[4]) {
    reinterpret_cast<int4 *>(at)[0] = make_int4((int)rows[0], (int)rows[1], (int)rows[2], (int)rows[3]);
    at[4] = adapter;
}
__device__ __forceinline__ void load_pair(const int32_t *at, TilePair &pr) {
    const int4 m = *reinterpret_cast<const int4 *>(at);
    pr.rows[0] = m.x;
    pr.rows[1] = m.y;
    pr.rows[2] = m.z;
    pr.rows[3] = m.w;
    pr.adapter = at[4];
}
__device__ __forceinline__ void load_pair(const int32_t *at, int &adapter) { adapter = at[4]; }

// ------------------------------------------------------------------ the plan
__device__ __forceinline__ uint32_t bits_below(int n) {
    return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u);
}

// Rows of one tile: they stay in their order, a thread a row.  The first row of each
// adapter has its pair (1.8 us; 3.9 sorted as below).
__global__ void __launch_bounds__(kTileRows)
    adapter_plan_tile_kernel(const int32_t *ids, int rows, int adapters, AdapterLayout l,
                             int32_t *plan, int32_t *error) {
    __shared__ __align__(16) int s_id[kTileRows];
    __shared__ int s_leads[4];
    grid_dep_wait();
    grid_dep_launch();
    const int r = threadIdx.x, warp = r >> 5, lane = r & 31;
    int a = r < rows ? ids[r] : -1;
    if (a < -1 || a >= adapters) {
        raise(error, PK_DEV_BAD_SLOT);
        a = -1;
    }
    s_id[r] = a;
    __syncthreads();
    uint32_t in[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < kTileRows; j += 4) {
        const int4 o = *reinterpret_cast<const int4 *>(s_id + j);
        in[j / 32] |= (uint32_t)(o.x == a) << (j & 31) | (uint32_t)(o.y == a) << ((j + 1) & 31) |
                      (uint32_t)(o.z == a) << ((j + 2) & 31) | (uint32_t)(o.w == a) << ((j + 3) & 31);
    }
    bool lead = a >= 0 && !(in[warp] & ((1u << lane) - 1u));
    for (int w = 0; w < warp; ++w) lead = lead && !in[w];
    const unsigned leads = __ballot_sync(0xffffffffu, lead);
    if (lane == 0) s_leads[warp] = __popc(leads);
    __syncthreads();
    int at = __popc(leads & ((1u << lane) - 1u));
    for (int w = 0; w < warp; ++w) at += s_leads[w];
    if (lead) store_pair(plan + l.pairs + kPairWords * at, a, in);
    plan[l.order + r] = min(r, rows);
    if (r == 0) {
        plan[l.tile_pair] = 0;
        plan[l.tile_pair + 1] = s_leads[0] + s_leads[1] + s_leads[2] + s_leads[3];
        plan[l.sorted] = 1;
    }
}

// More rows than a tile's: a counting sort.  The rows are cut into chunks of neighbouring
// ones, with counts of their own, and a row's place is its adapter's first one, the
// adapter's rows in the chunks before and its rank among those of the chunk, which one warp
// walks: rows of an adapter stay in their order.  (Places handed out by atomics go by which
// warp comes first, and a row near a tile's border with them from one tile to the other,
// where a split product adds its terms in another order.  They took 3.9 us for 320 rows of
// 32 adapters and 9.1 for 6720 of 64, this takes 5.0 and 10.9; 6720 of 8192 adapters, whose
// counts leave room for five chunks, 24 and 44.)
constexpr int kPlanCounts = 50 * 1024;   // words of shared memory
struct PlanCut {
    int chunks;   // as many as the counts leave room for, 32 at most
    int warps;    // that count the rows of each
    int steps;    // groups of 32 rows of each
};
PlanCut plan_cut(int rows, int adapters) {
    const int groups = (rows + 31) / 32, room = kPlanCounts / (adapters + 1) - 1;
    PlanCut c;
    c.chunks = room < 32 ? room : 32;
    c.warps = 32 / c.chunks;
    c.steps = (groups + c.chunks - 1) / c.chunks;
    return c;
}
__global__ void __launch_bounds__(1024) adapter_plan_kernel(const int32_t *ids, int rows,
                                                            int adapters, AdapterLayout l,
                                                            PlanCut cut, int32_t *plan,
                                                            int32_t *error) {
    // counts, then places [chunk][adapters + 1] (the last: rows without one); each
    // adapter's first place
    extern __shared__ int s_bins[];
    __shared__ int s_warp[2][33], s_moved;
    grid_dep_wait();
    grid_dep_launch();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bins = adapters + 1;
    const int tiles = (rows + kTileRows - 1) / kTileRows, steps = cut.steps;
    const int chunk = warp / cut.warps, sub = warp - chunk * cut.warps;
    const bool mine = chunk < cut.chunks;
    const int row0 = chunk * steps * 32 + lane;   // of the chunk
    const int of = chunk * bins, firsts = cut.chunks * bins;
    for (int i = tid; i < firsts; i += blockDim.x) s_bins[i] = 0;
    if (tid == 0) s_moved = 0;
    __syncthreads();
    // kHeld of the warp's steps of its chunk at a time, their ids requested together
    constexpr int kHeld = 8;
    bool bad = false;
    auto read = [&](int r) { return ids[min(r, rows - 1)]; };
    auto bin_of = [&](int r, int id) {   // -1 behind the last row
        const int a = id >= 0 && id < adapters ? id : adapters;
        bad |= id < -1 || id >= adapters;
        return r < rows ? a : -1;
    };
    int held[kHeld];
    bool moved = false;   // a row whose adapter is above the next one's
    if (mine)
        for (int s0 = sub; s0 < steps; s0 += kHeld * cut.warps) {
            int next[kHeld];   // the row behind each step
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                const int step = s0 + i * cut.warps;
                held[i] = next[i] = 0;
                if (step < steps) {
                    held[i] = read(row0 + step * 32);
                    next[i] = read(row0 - lane + step * 32 + 32);
                }
            }
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                const int step = s0 + i * cut.warps;
                if (step >= steps) break;
                const int a = held[i] = bin_of(row0 + step * 32, held[i]);
                // one atomic for a warp whose rows agree, one a row otherwise
                if (__all_sync(0xffffffffu, a == __shfl_sync(0xffffffffu, a, 0))) {
                    if (lane == 0 && a >= 0) atomicAdd(&s_bins[of + a], 32);
                } else if (a >= 0) {
                    atomicAdd(&s_bins[of + a], 1);
                }
                const int b = __shfl_down_sync(0xffffffffu, a, 1);
                const int after = lane == 31 ? bin_of(row0 + step * 32 + 1, next[i]) : b;
                moved |= after >= 0 && a > after;
            }
        }
    if (bad) raise(error, PK_DEV_BAD_SLOT);
    if (moved) s_moved = 1;
    // each adapter's first sorted row and first pair (it has one for each tile that
    // its rows touch), 1024 adapters at a time
    int32_t *pair = plan + l.pairs;
    for (int i = tid; i < tiles + 1; i += blockDim.x) plan[l.tile_pair + i] = 0x7fffffff;
    __syncthreads();
    int base = 0, pairs = 0;   // rows and pairs of the adapters before
    for (int a0 = 0; a0 < bins; a0 += blockDim.x) {
        const int a = a0 + tid;
        int n = 0;
        if (a < bins)
            for (int c0 = 0; c0 < cut.chunks; c0 += 8) {   // the chunks' places from first on
                int here[8];
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    here[c] = c0 + c < cut.chunks ? s_bins[(c0 + c) * bins + a] : 0;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    if (c0 + c < cut.chunks) s_bins[(c0 + c) * bins + a] = n;
                    n += here[c];
                }
            }
        auto scan = [&](int v, int &total, int (&sums)[33]) {
            int x = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            if (lane == 31) sums[warp] = x;
            __syncthreads();
            if (warp == 0) {
                int t = sums[lane];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, t, o);
                    if (lane >= o) t += y;
                }
                sums[lane] = t;
                if (lane == 31) sums[32] = t;
            }
            __syncthreads();
            total = sums[32];
            return (warp > 0 ? sums[warp - 1] : 0) + x - v;
        };
        int total;
        const int first = base + scan(n, total, s_warp[0]);
        base += total;
        const int t0 = first / kTileRows, t1 = n ? (first + n - 1) / kTileRows : t0 - 1;
        const int parts = a < adapters && n ? t1 - t0 + 1 : 0;
        // (the barriers of this scan part the other's uses of its sums, and the other way)
        const int p0 = pairs + scan(parts, total, s_warp[1]);
        pairs += total;
        if (a < bins) s_bins[firsts + a] = first;
        for (int i = 0; i < parts; ++i) {
            const int t = t0 + i, lo = max(first - t * kTileRows, 0);
            const int hi = min(first + n - t * kTileRows, kTileRows);
            uint32_t in[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) in[w] = bits_below(hi - w * 32) & ~bits_below(lo - w * 32);
            store_pair(pair + (int64_t)kPairWords * (p0 + i), a, in);
            if (lo == 0) plan[l.tile_pair + t] = p0 + i;
        }
    }
    __syncthreads();
    // tiles that no adapter's rows begin: past all of them
    for (int i = tid; i < tiles + 1; i += blockDim.x)
        if (plan[l.tile_pair + i] == 0x7fffffff) plan[l.tile_pair + i] = pairs;
    const bool resort = s_moved != 0;
    const int bits = 32 - __clz(adapters);
    const unsigned below = (1u << lane) - 1u;
    if (mine && sub == 0)
        for (int s0 = 0; s0 < steps; s0 += kHeld) {
            const bool others = steps > kHeld || cut.warps > 1;   // than were counted last
            if (others) {
#pragma unroll
                for (int i = 0; i < kHeld; ++i)
                    if (s0 + i < steps) held[i] = read(row0 + (s0 + i) * 32);
            }
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                if (s0 + i >= steps) break;
                const int r = row0 + (s0 + i) * 32, a = others ? bin_of(r, held[i]) : held[i];
                int at = r;
                if (resort) {
                    // the lanes of the same adapter, by a ballot for each of its bits
                    unsigned same = __ballot_sync(0xffffffffu, a >= 0);
                    if (!__all_sync(0xffffffffu, a == __shfl_sync(0xffffffffu, a, 0)))
#pragma unroll 4
                        for (int b = 0; b < bits; ++b) {
                            const unsigned has = __ballot_sync(0xffffffffu, a >> b & 1);
                            same &= a >> b & 1 ? has : ~has;
                        }
                    int before = 0;
                    if (a >= 0) before = s_bins[of + a] + __popc(same & below);
                    __syncwarp();   // read by all
                    if (a >= 0) {
                        if (same >> lane == 1) s_bins[of + a] = before + 1;   // the last
                        at = s_bins[firsts + a] + before;
                    }
                    __syncwarp();
                }
                if (a >= 0) plan[l.order + at] = r;
            }
        }
    if (tid == 0) plan[l.sorted] = !resort;
    for (int r = rows + tid; r < tiles * kTileRows; r += blockDim.x) plan[l.order + r] = rows;
}

// --------------------------------------------------------------------- S
// S[m] = scale[a] * x[m] down[a]^T for 16 sorted rows (one m16n8k16 row tile) a CTA,
// the K blocks of 64 dealt out to its eight warps.  Operands go from global memory to
// fragments directly: the contraction may take its terms in any order, so a lane's
// share of a row's 32 columns can be 8 neighbouring ones (16 bytes), for rows of x and
// of down alike, and needs no shared memory, no barrier and no ldmatrix.  Rows whose
// order is not the sorted one are written to their sorted copy on the way.
//
// A group of rows with several adapters takes a pass for each, and a pass keeps the
// sums of its own rows only, so no product of another adapter's weights reaches a row;
// with few groups the passes are CTAs of their own (blockIdx.y).
//
// Reading x and writing its copy bound it: 6720 x 4096, rank 32, 64 adapters, 126 MB,
// 34 us.  Tiles staged in shared memory with a barrier a stage took 46.
constexpr int kShWarps = 8, kShRows = 16;
// x a block ahead where the registers of two CTAs an SM hold it (rank 32: 34 us for 38 at
// three CTAs without; rank 16: level; rank 64, where it spills: 16 us slower)
constexpr bool shrink_ahead(int nt) { return nt == 4; }

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NT>   // 8-column tiles of S: rank <= 8 NT
__global__ void __launch_bounds__(kShWarps * 32, NT < 4 ? 3 : 2)
    adapter_shrink_kernel(const AdapterArgs p) {
    extern __shared__ float sh_part[];   // [warp][row][rank]
    __shared__ int2 s_pair[kShRows];     // the group's pairs: adapter, bits of its rows
    __shared__ int s_n;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
    grid_dep_wait();
    grid_dep_launch();
    const int32_t *plan = p.plan;
    const int tile = blockIdx.x / (kTileRows / kShRows);
    const int g0 = blockIdx.x % (kTileRows / kShRows) * kShRows;   // first row in the tile
    const int64_t m0 = (int64_t)tile * kTileRows + g0;
    // the pairs of the tile that have rows of the group
    if (warp == 0) {
        const int pair0 = plan[p.l.tile_pair + tile], pair1 = plan[p.l.tile_pair + tile + 1];
        int n = 0;
        for (int q = pair0; q < pair1; q += 32) {
            int2 pr = make_int2(0, 0);
            if (q + lane < pair1) {
                const int32_t *at = plan + p.l.pairs + (int64_t)kPairWords * (q + lane);
                pr = make_int2(at[4], (uint32_t)at[g0 >> 5] >> (g0 & 31) & 0xffffu);
            }
            const unsigned has = __ballot_sync(0xffffffffu, pr.y != 0);
            if (pr.y) s_pair[n + __popc(has & ((1u << lane) - 1u))] = pr;
            n += __popc(has);
        }
        if (lane == 0) s_n = n;
    }
    __syncthreads();
    const int n_pairs = s_n, r = p.rank, nk = p.K / 64;
    const int first = blockIdx.y, step = gridDim.y;
    if (first > 0 && first >= n_pairs) return;
    // this lane's rows of x: fragment rows lane / 4 and + 8
    const int fr = lane >> 2, fc = (lane & 3) * 8;
    const int r0 = plan[p.l.order + m0 + fr], r1 = plan[p.l.order + m0 + fr + 8];
    const bool in0 = r0 < p.M, in1 = r1 < p.M;
    const __nv_bfloat16 *x0 = static_cast<const __nv_bfloat16 *>(p.x) + (in0 ? (int64_t)r0 * p.ldx : 0) + fc;
    const __nv_bfloat16 *x1 = static_cast<const __nv_bfloat16 *>(p.x) + (in1 ? (int64_t)r1 * p.ldx : 0) + fc;
    const bool copying = first == 0 && !plan[p.l.sorted];
    __nv_bfloat16 *copy = static_cast<__nv_bfloat16 *>(p.xs) + (m0 + fr) * p.K + fc;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    const int warps = min(kShWarps, nk);

    for (int j = first; j < max(n_pairs, 1); j += step) {
        const bool any = j < n_pairs;
        const int2 pr = any ? s_pair[j] : make_int2(0, 0);
        const __nv_bfloat16 *down =
            static_cast<const __nv_bfloat16 *>(p.down) + ((int64_t)pr.x * r + fr) * p.K + fc;
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
        uint4 a[2][2], next[2][2];   // columns fc .. + 7 of both halves of the block
        auto fetch = [&](int kb, uint4 (&to)[2][2]) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                to[h][0] = in0 ? *reinterpret_cast<const uint4 *>(x0 + kb * 64 + h * 32) : zero;
                to[h][1] = in1 ? *reinterpret_cast<const uint4 *>(x1 + kb * 64 + h * 32) : zero;
            }
        };
        if (shrink_ahead(NT) && warp < nk) fetch(warp, next);
        for (int kb = warp; kb < nk; kb += kShWarps) {
            if (shrink_ahead(NT)) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 2; ++i) a[h][i] = next[h][i];
                if (kb + kShWarps < nk) fetch(kb + kShWarps, next);
            } else {
                fetch(kb, a);
            }
            constexpr int kAtOnce = NT < 8 ? NT : 8;   // tiles of S whose rows are in registers
#pragma unroll
            for (int n0 = 0; n0 < NT; n0 += kAtOnce) {
                uint4 b[kAtOnce][2];
#pragma unroll
                for (int n = 0; n < kAtOnce; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        b[n][h] = any && (n0 + n) * 8 < r
                                      ? __ldg(reinterpret_cast<const uint4 *>(
                                            down + (int64_t)(n0 + n) * 8 * p.K + kb * 64 + h * 32))
                                      : zero;
                if (copying && j == 0 && n0 == 0) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        *reinterpret_cast<uint4 *>(copy + kb * 64 + h * 32) = a[h][0];
                        *reinterpret_cast<uint4 *>(copy + (int64_t)8 * p.K + kb * 64 + h * 32) = a[h][1];
                    }
                }
                if (any) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int n = 0; n < kAtOnce; ++n) {
                            mma_16816(acc[n0 + n], a[h][0].x, a[h][1].x, a[h][0].y, a[h][1].y,
                                      b[n][h].x, b[n][h].y);
                            mma_16816(acc[n0 + n], a[h][0].z, a[h][1].z, a[h][0].w, a[h][1].w,
                                      b[n][h].z, b[n][h].w);
                        }
                }
            }
        }
        // the warps' sums, in order (rows without an adapter have no S: their lanes are
        // off in every product)
        if (warp < warps) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (n * 8 >= r) break;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<float2 *>(sh_part + (warp * kShRows + fr + 8 * h) * r + n * 8 +
                                                (lane & 3) * 2) =
                        make_float2(acc[n][2 * h], acc[n][2 * h + 1]);
            }
        }
        __syncthreads();
        const float scale = any && p.scale ? p.scale[pr.x] : 1.f;
        __nv_bfloat16 *s = static_cast<__nv_bfloat16 *>(p.s) + m0 * r;
        for (int c = tid; c < kShRows * r; c += kShWarps * 32) {
            const int row = c / r;
            if (!(pr.y >> row & 1)) continue;
            float v = 0.f;
            for (int w = 0; w < warps; ++w) v += sh_part[w * kShRows * r + c];
            s[c] = __float2bfloat16_rn(v * scale);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ the product
// umma_bf16 that leaves the accumulator lanes of `off`'s bits as they are
__device__ __forceinline__ void umma_bf16_lanes(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                                uint32_t idesc, const uint32_t (&off)[4]) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, 1, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%4, %5, %6, %7}, p;\n\t}" ::"r"(
            tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(off[0]), "r"(off[1]), "r"(off[2]), "r"(off[3])
        : "memory");
}

__device__ __forceinline__ void umma_bf16_pair_lanes(uint32_t tmem_d, uint64_t adesc,
                                                     uint64_t bdesc, uint32_t idesc,
                                                     const uint32_t (&off)[8]) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, 1, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%4, %5, %6, %7, %8, %9, %10, %11}, "
        "p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(off[0]), "r"(off[1]), "r"(off[2]), "r"(off[3]),
        "r"(off[4]), "r"(off[5]), "r"(off[6]), "r"(off[7])
        : "memory");
}
// The pairs p0 .. p1 of a tile (T: int, the adapters alone, or TilePair), read eight
// at a time: the first eight when the tile begins, so that the
// reads' latency (one a pair took 0.4 us of a pair's turn) is under the K blocks before
// them.
template <typename T> struct TilePairs {
    const int32_t *pairs;
    int p0, p1;
    T ahead[8];
    __device__ __forceinline__ TilePairs(const int32_t *all, int from, int to)
        : pairs(all), p0(from), p1(to) {
        fetch();
    }
    __device__ __forceinline__ bool any() const { return p0 < p1; }
    __device__ __forceinline__ void fetch() {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (p0 + i < p1) load_pair(pairs + (int64_t)kPairWords * (p0 + i), ahead[i]);
    }
    // fn(pair) for each, while it returns true
    template <typename F> __device__ __forceinline__ void each(F fn) {
        while (p0 < p1) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (p0 + i < p1 && !fn(ahead[i])) return;
            p0 += 8;
            fetch();
        }
    }
};

// A warp's rows of C and R in sorted order: the eight that this lane's pieces touch.
struct SortedRows {
    int row[8];
    __device__ __forceinline__ int operator()(int, int i) const { return row[i]; }
};

struct AdapterMaps {
    CUtensorMap x, xs, w, s, up;   // rows, sorted copy, weight, S, up
};

constexpr int kAdThreads = 192;   // TMA, MMA and 4 epilogue warps

// The persistent GEMM (pk_gemm.cu) over the sorted rows, with the pairs' K blocks.
// The rows come by TMA tile loads from their sorted copy (from x itself where its
// order is the sorted one).  Fetching them in place was slower at every size: TMA's
// gather4 (four 128-byte rows an instruction) takes 85 cycles each, six times what
// the MMAs of a stage last; 16-byte cp.async by four more warps costs its proxy
// fences, 0.5 us a stage (6720 x 1024 x 4096: 265 and 98 us against 67 for the
// plain tile loads).
template <int BN, int NS, int EPI>
__global__ void __launch_bounds__(kAdThreads, 1)
    adapter_gemm_kernel(const __grid_constant__ AdapterMaps tm, const AdapterArgs p) {
    constexpr int kBBytes = BN * kBK * 2;
    extern __shared__ uint8_t gemm_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(gemm_smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sA = smem, *sB = smem + NS * kABytes, *sS = sB + NS * kBBytes;
    __shared__ __align__(8) uint64_t full[NS], empty[NS], tmem_full[2], tmem_empty[2], s_full, s_empty;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int failed;

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int mtiles = (p.M + kBM - 1) / kBM, tiles = mtiles * (p.N / BN), nk = p.K / kBK;
    const int rblocks = (p.rank + kBK - 1) / kBK;
    uint8_t *stage = sS + rblocks * kABytes + (warp & 3) * kStageBytes;
    const int32_t *tile_pair = p.plan + p.l.tile_pair, *order = p.plan + p.l.order,
                  *sorted = p.plan + p.l.sorted;
    const int32_t *pairs = p.plan + p.l.pairs;
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tmem_full[a], 1);
            mbar_init(&tmem_empty[a], 4);
        }
        mbar_init(&s_full, 1);
        mbar_init(&s_empty, 1);
        failed = 0;
        fence_mbar_init();
        prefetch_tmap(&tm.w);
        prefetch_tmap(&tm.up);
        prefetch_tmap(&tm.s);
    }
    if (warp == 0) {
        tmem_alloc(&tmem_base, 2 * BN);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base;
    // (a lane that waits finds what another has found: the warp's answer is one)
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity)) return true;
        if (!failed && !mbar_wait_bounded(bar, parity, kWaitLimitNs)) {
            raise(p.error, PK_DEV_TIMEOUT);
            failed = 1;
        }
        return !failed;
    };
    // ring stage and its phase, a step a use
    int s = 0;
    uint32_t phase = 0;
    auto next = [&]() {
        if (++s == NS) {
            s = 0;
            phase ^= 1;
        }
    };
    // Producer and MMA warp: the whole warp walks along, so that indexes and descriptors
    // are uniform (one lane's walk took 270 cycles a stage beside its MMAs).
    if (warp == 0) {
        const bool one = elect_one();
        // The weights of the first stages do not depend on the kernel before: they are
        // requested ahead of the wait for it.
        const int pre = (int)blockIdx.x < tiles ? (nk < NS ? nk : NS) : 0;
        if (one)
            for (int kb = 0; kb < pre; ++kb) {
                mbar_arrive_expect_tx(&full[kb], kABytes + kBBytes);
                tma_load_2d(sB + kb * kBBytes, &tm.w, &full[kb], kb * kBK,
                            ((int)blockIdx.x / mtiles) * BN);
            }
        // (the plan, and rows in their own order, are older than the kernel before, which
        // has waited for them)
        const CUtensorMap *rows = *sorted ? &tm.x : &tm.xs;
        if (rows == &tm.xs) grid_dep_wait();
        int used = 0, with_s = 0;   // stages requested; tiles that had an S
        bool ok = true;
        for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
            const int mt = tile % mtiles, m0 = mt * kBM, n0 = (tile / mtiles) * BN;
            TilePairs<int> of_tile(pairs, tile_pair[mt], tile_pair[mt + 1]);
            for (int kb = 0; kb < nk; ++kb, ++used) {
                if (used >= NS && !(ok = __all_sync(0xffffffffu, wait(&empty[s], phase ^ 1)))) break;
                if (one) {
                    if (used >= pre) {
                        mbar_arrive_expect_tx(&full[s], kABytes + kBBytes);
                        tma_load_2d(sB + s * kBBytes, &tm.w, &full[s], kb * kBK, n0);
                    }
                    tma_load_2d(sA + s * kABytes, rows, &full[s], kb * kBK, m0);
                }
                __syncwarp();
                next();
            }
            if (!ok || !of_tile.any()) continue;
            grid_dep_wait();   // S
            // S once a tile (a copy for each pair made every CTA of a row tile ask for
            // the same few lines again and again: 0.65 us a pair)
            if (with_s >= 1 && !(ok = __all_sync(0xffffffffu, wait(&s_empty, (with_s - 1) & 1)))) break;
            ++with_s;
            if (one) {
                mbar_arrive_expect_tx(&s_full, rblocks * kABytes);
                for (int rb = 0; rb < rblocks; ++rb)
                    tma_load_2d(sS + rb * kABytes, &tm.s, &s_full, rb * kBK, m0);
            }
            of_tile.each([&](int adapter) {
                for (int rb = 0; rb < rblocks; ++rb, ++used) {
                    if (used >= NS && !(ok = __all_sync(0xffffffffu, wait(&empty[s], phase ^ 1))))
                        return false;
                    if (one) {
                        mbar_arrive_expect_tx(&full[s], kBBytes);
                        tma_load_3d(sB + s * kBBytes, &tm.up, &full[s], rb * kBK, n0, adapter);
                    }
                    __syncwarp();
                    next();
                }
                return true;
            });
        }
        if (!ok) {   // leave no copy in flight: the last NS stages' and the last S
            for (int i = 0; i < min(used, NS); ++i) {
                s = s == 0 ? NS - 1 : s - 1;
                if (s == NS - 1) phase ^= 1;
                mbar_wait_bounded(&full[s], phase, kWaitLimitNs);
            }
            if (with_s) mbar_wait_bounded(&s_full, (with_s - 1) & 1, kWaitLimitNs);
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_bf16(kBM, BN);
        const bool one = elect_one();
        const uint64_t a_desc = sw128_desc(smem_u32(sA)), b_desc = sw128_desc(smem_u32(sB)),
                       s_desc = sw128_desc(smem_u32(sS));
        int t = 0, with_s = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++t) {
            const int acc = t & 1, use = t >> 1, mt = tile % mtiles;
            if (use >= 1 && !(ok = __all_sync(0xffffffffu, wait(&tmem_empty[acc], (use - 1) & 1)))) break;
            tc_fence_after();
            const uint32_t d = tmem + acc * BN;
            TilePairs<TilePair> of_tile(pairs, tile_pair[mt], tile_pair[mt + 1]);
            for (int kb = 0; kb < nk; ++kb) {
                if (!(ok = __all_sync(0xffffffffu, wait(&full[s], phase)))) break;
                tc_fence_after();
                if (one) {
                    const uint64_t a0 = a_desc + s * (kABytes >> 4), b0 = b_desc + s * (kBBytes >> 4);
#pragma unroll
                    for (int kk = 0; kk < kBK / 16; ++kk)
                        umma_bf16(d, a0 + kk * 2, b0 + kk * 2, idesc, (kb | kk) != 0);
                    umma_commit(&empty[s]);
                }
                __syncwarp();
                next();
            }
            if (ok && of_tile.any()) {
                ok = __all_sync(0xffffffffu, wait(&s_full, with_s++ & 1));
                if (ok)
                    of_tile.each([&](const TilePair &pr) {
                        const uint32_t off[4] = {~pr.rows[0], ~pr.rows[1], ~pr.rows[2], ~pr.rows[3]};
                        for (int rb = 0; rb < rblocks; ++rb) {
                            if (!(ok = __all_sync(0xffffffffu, wait(&full[s], phase)))) return false;
                            tc_fence_after();
                            if (one) {
                                const uint64_t a0 = s_desc + rb * (kABytes >> 4),
                                               b0 = b_desc + s * (kBBytes >> 4);
                                const int steps = min(kBK, p.rank - rb * kBK);
                                for (int kk = 0; kk * 16 < steps; ++kk)
                                    umma_bf16_lanes(d, a0 + kk * 2, b0 + kk * 2, idesc, off);
                                umma_commit(&empty[s]);
                            }
                            __syncwarp();
                            next();
                        }
                        return true;
                    });
                if (one) umma_commit(&s_empty);
            }
            if (one) umma_commit(&tmem_full[acc]);
            __syncwarp();
        }
    } else {
        // epilogue warps 2..5
        grid_dep_wait();
        const int q = warp & 3;
        int t = 0;
        uint4 rv[8], rn[8];
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++t) {
            const int acc = t & 1, use = t >> 1;
            const int m0 = (tile % mtiles) * kBM, n0 = (tile / mtiles) * BN;
            SortedRows rows;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int m = order[m0 + q * 32 + i * 4 + (lane >> 3)];
                rows.row[i] = m < p.M ? m : -1;
            }
            __nv_bfloat16 *C = static_cast<__nv_bfloat16 *>(p.C);
            const __nv_bfloat16 *R = static_cast<const __nv_bfloat16 *>(p.R);
            if (is_residual(EPI)) load_residual64(rn, rows, n0, R, p.ldr);
            const bool ok = __all_sync(0xffffffffu,
                                       mbar_wait_bounded(&tmem_full[acc], use & 1, kWaitLimitNs));
            if (!ok) {
                if (lane == 0) raise(p.error, PK_DEV_TIMEOUT);
                failed = 1;
                break;
            }
            tc_fence_after();
            if (tile + (int)gridDim.x >= tiles) grid_dep_launch();
#pragma unroll 1
            for (int c = 0; c < BN / 64; ++c) {
#pragma unroll
                for (int i = 0; i < 8; ++i) rv[i] = rn[i];
                if (is_residual(EPI) && c + 1 < BN / 64)
                    load_residual64(rn, rows, n0 + (c + 1) * 64, R, p.ldr);
                epilogue_tile64<EPI>(tmem + acc * BN + ((uint32_t)(q * 32) << 16) + c * 64, rows,
                                     n0 + c * 64, C, p.ldc, rv,
                                     static_cast<const __nv_bfloat16 *>(p.bias), p.alpha, stage);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cta(&tmem_empty[acc]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 2 * BN);
    }
}

// Few tiles: a cluster for each, its CTAs with a part of K each and every c-th pair of the
// tile.  A tile is a chain of K blocks, some 0.2 us each whatever the depth of the ring,
// and most SMs have no tile: 4 rows, K 4096, N 512, rank 8 took 23 us on a CTA a tile and
// take 8.3 on eight; 16 rows, K and N 4096, 16 adapters: 29 and 21 on two.  The parts meet
// in shared memory: each CTA leaves its sums there, and all of them add up and write a
// share of the tile, in the order of the CTAs.
constexpr int kSplitBN = 64, kSplitStages = 6, kSplitRow = kSplitBN + 4;   // floats
template <int EPI>
__global__ void __launch_bounds__(kAdThreads, 1)
    adapter_gemm_split_kernel(const __grid_constant__ AdapterMaps tm, const AdapterArgs p) {
    constexpr int BN = kSplitBN, NS = kSplitStages, kBBytes = BN * kBK * 2;
    static_assert(kTileRows * kSplitRow * 4 <= NS * kABytes, "the sums take the ring's place");
    extern __shared__ uint8_t gemm_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(gemm_smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sA = smem, *sB = smem + NS * kABytes, *sS = sB + NS * kBBytes;
    float *sums = reinterpret_cast<float *>(sA);   // [row][kSplitRow]
    __shared__ __align__(8) uint64_t full[NS], empty[NS], tmem_full, s_full;
    __shared__ uint32_t tmem_base;
    __shared__ __align__(16) int32_t s_pairs[kTileRows * kPairWords];   // this CTA's
    __shared__ volatile int failed;

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int c = gridDim.x, part = (int)cluster_ctarank(), tile = blockIdx.y;
    const int mtiles = (p.M + kBM - 1) / kBM, mt = tile % mtiles;
    const int m0 = mt * kBM, n0 = tile / mtiles * BN, live = min(p.M - m0, kBM);
    const int nk = p.K / kBK, kb0 = (int)((int64_t)nk * part / c);
    const int n_kb = (int)((int64_t)nk * (part + 1) / c) - kb0;
    const int rblocks = (p.rank + kBK - 1) / kBK;
    const uint32_t a_bytes = p.box_rows * kBK * 2;
    const int pre = min(n_kb, NS);
    const int32_t *tile_pair = p.plan + p.l.tile_pair, *pairs = p.plan + p.l.pairs,
                  *order = p.plan + p.l.order, *sorted = p.plan + p.l.sorted;
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&tmem_full, 1);
        mbar_init(&s_full, 1);
        failed = 0;
        fence_mbar_init();
        // W first: it does not depend on the kernel before
        for (int g = 0; g < pre; ++g) {
            mbar_arrive_expect_tx(&full[g], a_bytes + kBBytes);
            tma_load_2d(sB + g * kBBytes, &tm.w, &full[g], (kb0 + g) * kBK, n0);
        }
        prefetch_tmap(&tm.up);
        prefetch_tmap(&tm.s);
    }
    if (warp == 0) {
        tmem_alloc(&tmem_base, BN);
        tmem_relinquish();
    }
    const int pair0 = tile_pair[mt], n_pairs = (tile_pair[mt + 1] - pair0 - part + c - 1) / c;
    const bool in_order = *sorted;
    for (int i = threadIdx.x; i < n_pairs * 2; i += kAdThreads)
        reinterpret_cast<int4 *>(s_pairs)[i] = reinterpret_cast<const int4 *>(
            pairs + (int64_t)kPairWords * (pair0 + part + (i >> 1) * c))[i & 1];
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base;
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity)) return true;
        if (!failed && !mbar_wait_bounded(bar, parity, kWaitLimitNs)) {
            raise(p.error, PK_DEV_TIMEOUT);
            failed = 1;
        }
        return !failed;
    };
    // ring stage and its phase, a step a use
    int s = 0;
    uint32_t phase = 0;
    auto next = [&]() {
        if (++s == NS) {
            s = 0;
            phase ^= 1;
        }
    };
    if (warp == 0) {
        const bool one = elect_one();
        // rows in their own order are older than the kernel before, which has waited for
        // them; their sorted copy is its work
        const CUtensorMap *rows = in_order ? &tm.x : &tm.xs;
        if (!in_order) grid_dep_wait();
        int used = 0;   // stages requested
        bool ok = true;
        for (int g = 0; g < n_kb; ++g, ++used) {
            if (g >= pre && !(ok = __all_sync(0xffffffffu, wait(&empty[s], phase ^ 1)))) break;
            if (one) {
                if (g >= pre) {
                    mbar_arrive_expect_tx(&full[s], a_bytes + kBBytes);
                    tma_load_2d(sB + s * kBBytes, &tm.w, &full[s], (kb0 + g) * kBK, n0);
                }
                tma_load_2d(sA + s * kABytes, rows, &full[s], (kb0 + g) * kBK, m0);
            }
            __syncwarp();
            next();
        }
        if (ok && n_pairs > 0) {
            grid_dep_wait();   // S
            if (one) {
                mbar_arrive_expect_tx(&s_full, rblocks * a_bytes);
                for (int rb = 0; rb < rblocks; ++rb)
                    tma_load_2d(sS + rb * kABytes, &tm.s, &s_full, rb * kBK, m0);
            }
            for (int i = 0; i < n_pairs && ok; ++i) {
                const int adapter = s_pairs[i * kPairWords + 4];
                for (int rb = 0; rb < rblocks; ++rb, ++used) {
                    if (used >= NS && !(ok = __all_sync(0xffffffffu, wait(&empty[s], phase ^ 1)))) break;
                    if (one) {
                        mbar_arrive_expect_tx(&full[s], kBBytes);
                        tma_load_3d(sB + s * kBBytes, &tm.up, &full[s], rb * kBK, n0, adapter);
                    }
                    __syncwarp();
                    next();
                }
            }
            if (!ok) mbar_wait_bounded(&s_full, 0, kWaitLimitNs);
        }
        if (!ok)   // leave no copy in flight: the last NS requests
            for (int i = 0; i < min(used, NS); ++i) {
                s = s == 0 ? NS - 1 : s - 1;
                if (s == NS - 1) phase ^= 1;
                mbar_wait_bounded(&full[s], phase, kWaitLimitNs);
            }
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_bf16(kBM, BN);
        const uint64_t a_desc = sw128_desc(smem_u32(sA)), b_desc = sw128_desc(smem_u32(sB)),
                       s_desc = sw128_desc(smem_u32(sS));
        const bool one = elect_one();
        bool ok = true;
        for (int g = 0; g < n_kb; ++g) {
            if (!(ok = __all_sync(0xffffffffu, wait(&full[s], phase)))) break;
            tc_fence_after();
            if (one) {
                const uint64_t a0 = a_desc + s * (kABytes >> 4), b0 = b_desc + s * (kBBytes >> 4);
#pragma unroll
                for (int kk = 0; kk < kBK / 16; ++kk)
                    umma_bf16(tmem, a0 + kk * 2, b0 + kk * 2, idesc, (g | kk) != 0);
                umma_commit(&empty[s]);
            }
            __syncwarp();
            next();
        }
        if (ok && n_pairs > 0) {
            ok = __all_sync(0xffffffffu, wait(&s_full, 0));
            for (int i = 0; i < n_pairs && ok; ++i) {
                const int4 in = reinterpret_cast<const int4 *>(s_pairs)[2 * i];
                const uint32_t off[4] = {~(uint32_t)in.x, ~(uint32_t)in.y, ~(uint32_t)in.z, ~(uint32_t)in.w};
                for (int rb = 0; rb < rblocks; ++rb) {
                    if (!(ok = __all_sync(0xffffffffu, wait(&full[s], phase)))) break;
                    tc_fence_after();
                    if (one) {
                        const uint64_t a0 = s_desc + rb * (kABytes >> 4), b0 = b_desc + s * (kBBytes >> 4);
                        const int steps = min(kBK, p.rank - rb * kBK);
                        for (int kk = 0; kk * 16 < steps; ++kk)
                            umma_bf16_lanes(tmem, a0 + kk * 2, b0 + kk * 2, idesc, off);
                        umma_commit(&empty[s]);
                    }
                    __syncwarp();
                    next();
                }
            }
        }
        if (one) umma_commit(&tmem_full);
    } else {
        // warps 2..5: this CTA's sums, a row a lane
        grid_dep_wait();
        const int row = (warp & 3) * 32 + lane;
        __all_sync(0xffffffffu, wait(&tmem_full, 0));
        tc_fence_after();
        if (row - lane < live) {
            float v[64];
            const uint32_t at = tmem + ((uint32_t)(row - lane) << 16);
            tmem_ld32(at, *reinterpret_cast<float(*)[32]>(v));
            tmem_ld32(at + 32, *reinterpret_cast<float(*)[32]>(v + 32));
            if (!failed && row < live)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    *reinterpret_cast<float4 *>(sums + row * kSplitRow + 4 * i) =
                        make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
        tc_fence_before();
    }
    grid_dep_launch();
    cluster_sync_all();   // every part's sums are there
    for (int i = part * kAdThreads + (int)threadIdx.x; i < live * (BN / 8); i += c * kAdThreads) {
        const int row = i / (BN / 8), col = i % (BN / 8) * 8, m = order[m0 + row];
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        const uint32_t mine = smem_u32(sums + row * kSplitRow + col);
        for (int r = 0; r < c; ++r) {
            const uint32_t at = mapa_rank(mine, r);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float4 x;
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                             : "r"(at + h * 16)
                             : "memory");
                v[4 * h] += x.x;
                v[4 * h + 1] += x.y;
                v[4 * h + 2] += x.z;
                v[4 * h + 3] += x.w;
            }
        }
        float f[8];
        if (is_residual(EPI))
            unpack16(*reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(p.R) +
                                                      (int64_t)m * p.ldr + n0 + col),
                     f, static_cast<const __nv_bfloat16 *>(nullptr));
        if (EPI == PK_GEMM_BIAS)
            unpack16(*reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(p.bias) + n0 + col),
                     f, static_cast<const __nv_bfloat16 *>(nullptr));
        uint4 o;
        __nv_bfloat162 *h = reinterpret_cast<__nv_bfloat162 *>(&o);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (EPI == PK_GEMM_SILU) v[e] = __fdividef(v[e], 1.f + __expf(-v[e]));
            if (is_residual(EPI)) v[e] = f[e] + p.alpha * v[e];
            if (EPI == PK_GEMM_RESIDUAL_RELU) v[e] = fmaxf(v[e], 0.f);
            if (EPI == PK_GEMM_BIAS) v[e] += f[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
        *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p.C) + (int64_t)m * p.ldc + n0 + col) = o;
    }
    cluster_sync_all();   // and no part is read any more
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, BN);
    }
}

// 3-D tile load into this CTA's shared memory, completion on an mbarrier of either
// CTA of the pair
__device__ __forceinline__ void tma_load_3d_pair(void *dst, const CUtensorMap *map, uint32_t bar,
                                                 int32_t c0, int32_t c1, int32_t c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}

// CTA-pair form (pk_gemm.cu's, 256 x BN tiles): CTA r loads sorted rows 128 r ..
// of the tile and rows (BN / 2) r .. of W.  The pairs of the tile's two
// 128-row halves are walked one half after the other, the other half's lanes off.
template <int BN, int NS, int EPI>
__global__ void __launch_bounds__(kAdThreads, 1)
    adapter_gemm_pair_kernel(const __grid_constant__ AdapterMaps tm, const AdapterArgs p) {
    constexpr int kHalfB = BN / 2;
    constexpr int kBBytes = kHalfB * kBK * 2;
    constexpr uint32_t kStageTx = 2 * (kABytes + kBBytes);   // both CTAs' loads
    extern __shared__ uint8_t gemm_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(gemm_smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sA = smem, *sB = smem + NS * kABytes, *sS = sB + NS * kBBytes;
    __shared__ __align__(8) uint64_t full[NS], empty[NS], tmem_full[2], tmem_empty[2], s_full, s_empty;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int failed;

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int pair = blockIdx.x / 2, npairs = gridDim.x / 2;
    const int halves = (p.M + kBM - 1) / kBM, mtiles = (halves + 1) / 2;
    const int tiles = mtiles * (p.N / BN), nk = p.K / kBK;
    const int rblocks = (p.rank + kBK - 1) / kBK;
    uint8_t *stage = sS + rblocks * kABytes + (warp & 3) * kStageBytes;
    const int32_t *tile_pair = p.plan + p.l.tile_pair, *order = p.plan + p.l.order,
                  *sorted = p.plan + p.l.sorted;
    const int32_t *pairs = p.plan + p.l.pairs;
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tmem_full[a], 1);
            mbar_init(&tmem_empty[a], 8);
        }
        mbar_init(&s_full, 1);
        mbar_init(&s_empty, 1);
        failed = 0;
        fence_mbar_init();
        prefetch_tmap(&tm.w);
        prefetch_tmap(&tm.up);
        prefetch_tmap(&tm.s);
    }
    if (warp == 0) {
        tmem_alloc_pair(&tmem_base, 2 * BN);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = tmem_base;
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (mbar_try_wait_cluster(bar, parity)) return true;
        if (!failed && !mbar_wait_cluster_bounded(bar, parity, kWaitLimitNs)) {
            raise(p.error, PK_DEV_TIMEOUT);
            failed = 1;
        }
        return !failed;
    };
    int s = 0;
    uint32_t phase = 0;
    auto next = [&]() {
        if (++s == NS) {
            s = 0;
            phase ^= 1;
        }
    };
    if (warp == 0) {
        const bool one = elect_one();
        const CUtensorMap *rows = *sorted ? &tm.x : &tm.xs;
        if (rows == &tm.xs) grid_dep_wait();
        int used = 0, with_s = 0;   // stages requested; tiles that had an S
        bool ok = true;
        const uint32_t f0 = mapa_rank(smem_u32(&full[0]), 0), sb = mapa_rank(smem_u32(&s_full), 0);
        for (int tile = pair; tile < tiles && ok; tile += npairs) {
            const int mt = tile % mtiles, m0 = mt * 2 * kBM + (int)rank * kBM;
            const int n0 = (tile / mtiles) * BN + (int)rank * kHalfB;
            TilePairs<int> of_tile(pairs, tile_pair[2 * mt], tile_pair[min(2 * mt + 2, halves)]);
            for (int kb = 0; kb < nk; ++kb, ++used) {
                if (used >= NS && !(ok = __all_sync(0xffffffffu, wait(&empty[s], phase ^ 1)))) break;
                if (one) {
                    if (leader) mbar_arrive_expect_tx(&full[s], kStageTx);
                    tma_load_2d_pair(sB + s * kBBytes, &tm.w, f0 + s * 8, kb * kBK, n0);
                    tma_load_2d_pair(sA + s * kABytes, rows, f0 + s * 8, kb * kBK, m0);
                }
                __syncwarp();
                next();
            }
            if (!ok || !of_tile.any()) continue;
            grid_dep_wait();   // S
            if (with_s >= 1 && !(ok = __all_sync(0xffffffffu, wait(&s_empty, (with_s - 1) & 1)))) break;
            ++with_s;
            if (one) {
                if (leader) mbar_arrive_expect_tx(&s_full, 2 * rblocks * kABytes);
                for (int rb = 0; rb < rblocks; ++rb)
                    tma_load_2d_pair(sS + rb * kABytes, &tm.s, sb, rb * kBK, m0);
            }
            of_tile.each([&](int adapter) {
                for (int rb = 0; rb < rblocks; ++rb, ++used) {
                    if (used >= NS && !(ok = __all_sync(0xffffffffu, wait(&empty[s], phase ^ 1))))
                        return false;
                    if (one) {
                        if (leader) mbar_arrive_expect_tx(&full[s], 2 * kBBytes);
                        tma_load_3d_pair(sB + s * kBBytes, &tm.up, f0 + s * 8, rb * kBK, n0, adapter);
                    }
                    __syncwarp();
                    next();
                }
                return true;
            });
        }
        if (leader) {   // leave none of the pair's loads in flight
            for (int i = 0; i < min(used, NS); ++i) {
                s = s == 0 ? NS - 1 : s - 1;
                if (s == NS - 1) phase ^= 1;
                mbar_wait_bounded(&full[s], phase, kWaitLimitNs);
            }
            if (with_s) mbar_wait_bounded(&s_full, (with_s - 1) & 1, kWaitLimitNs);
        }
    } else if (warp == 1) {
        if (leader) {
            constexpr uint32_t idesc = idesc_bf16(2 * kBM, BN);
            const bool one = elect_one();
            const uint64_t a_desc = sw128_desc(smem_u32(sA)), b_desc = sw128_desc(smem_u32(sB)),
                           s_desc = sw128_desc(smem_u32(sS));
            int t = 0, with_s = 0;
            bool ok = true;
            for (int tile = pair; tile < tiles && ok; tile += npairs, ++t) {
                const int acc = t & 1, use = t >> 1, mt = tile % mtiles;
                if (use >= 1 && !(ok = __all_sync(0xffffffffu, wait(&tmem_empty[acc], (use - 1) & 1)))) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * BN;
                const int border = tile_pair[min(2 * mt + 1, halves)];   // of the two halves
                TilePairs<TilePair> of_tile(pairs, tile_pair[2 * mt], tile_pair[min(2 * mt + 2, halves)]);
                for (int kb = 0; kb < nk; ++kb) {
                    if (!(ok = __all_sync(0xffffffffu, wait(&full[s], phase)))) break;
                    tc_fence_after();
                    if (one) {
                        const uint64_t a0 = a_desc + s * (kABytes >> 4), b0 = b_desc + s * (kBBytes >> 4);
#pragma unroll
                        for (int kk = 0; kk < kBK / 16; ++kk)
                            umma_bf16_pair(d, a0 + kk * 2, b0 + kk * 2, idesc, (kb | kk) != 0);
                        umma_commit_pair(&empty[s]);
                    }
                    __syncwarp();
                    next();
                }
                int pr_at = of_tile.p0;
                const bool any = of_tile.any();
                if (any && ok) ok = __all_sync(0xffffffffu, wait(&s_full, with_s++ & 1));
                if (ok)
                    of_tile.each([&](const TilePair &pr) {
                        const bool odd = pr_at++ >= border;   // the second half's
                        uint32_t off[8];
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            off[w] = odd ? ~0u : ~pr.rows[w];
                            off[w + 4] = odd ? ~pr.rows[w] : ~0u;
                        }
                        for (int rb = 0; rb < rblocks; ++rb) {
                            if (!(ok = __all_sync(0xffffffffu, wait(&full[s], phase)))) return false;
                            tc_fence_after();
                            if (one) {
                                const uint64_t a0 = s_desc + rb * (kABytes >> 4),
                                               b0 = b_desc + s * (kBBytes >> 4);
                                const int steps = min(kBK, p.rank - rb * kBK);
                                for (int kk = 0; kk * 16 < steps; ++kk)
                                    umma_bf16_pair_lanes(d, a0 + kk * 2, b0 + kk * 2, idesc, off);
                                umma_commit_pair(&empty[s]);
                            }
                            __syncwarp();
                            next();
                        }
                        return true;
                    });
                if (!ok) break;
                if (one) {
                    if (any) umma_commit_pair(&s_empty);
                    umma_commit_pair(&tmem_full[acc]);
                }
                __syncwarp();
            }
        }
    } else {
        // epilogue warps 2..5 of each CTA: its own 128 rows
        grid_dep_wait();
        const int q = warp & 3;
        const uint32_t empty0 = mapa_rank(smem_u32(&tmem_empty[0]), 0),
                       empty1 = mapa_rank(smem_u32(&tmem_empty[1]), 0);
        __nv_bfloat16 *C = static_cast<__nv_bfloat16 *>(p.C);
        const __nv_bfloat16 *R = static_cast<const __nv_bfloat16 *>(p.R);
        int t = 0;
        uint4 rv[8], rn[8];
        for (int tile = pair; tile < tiles; tile += npairs, ++t) {
            const int acc = t & 1, use = t >> 1;
            const int m0 = (tile % mtiles) * 2 * kBM + (int)rank * kBM, n0 = (tile / mtiles) * BN;
            SortedRows rows;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int m = m0 < p.M ? order[m0 + q * 32 + i * 4 + (lane >> 3)] : p.M;
                rows.row[i] = m < p.M ? m : -1;
            }
            if (is_residual(EPI)) load_residual64(rn, rows, n0, R, p.ldr);
            const bool ok = __all_sync(0xffffffffu,
                                       mbar_wait_bounded(&tmem_full[acc], use & 1, kWaitLimitNs));
            if (!ok) {
                if (lane == 0) raise(p.error, PK_DEV_TIMEOUT);
                failed = 1;
                break;
            }
            tc_fence_after();
            if (tile + npairs >= tiles) grid_dep_launch();
#pragma unroll 1
            for (int c = 0; c < BN / 64; ++c) {
#pragma unroll
                for (int i = 0; i < 8; ++i) rv[i] = rn[i];
                if (is_residual(EPI) && c + 1 < BN / 64)
                    load_residual64(rn, rows, n0 + (c + 1) * 64, R, p.ldr);
                epilogue_tile64<EPI>(tmem + acc * BN + ((uint32_t)(q * 32) << 16) + c * 64, rows,
                                     n0 + c * 64, C, p.ldc, rv,
                                     static_cast<const __nv_bfloat16 *>(p.bias), p.alpha, stage);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc ? empty1 : empty0);
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 2 * BN);
    }
}

template <int NT>
cudaError_t launch_shrink(const AdapterArgs &p, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(adapter_shrink_kernel<NT>, kShWarps * kShRows * NT * 8 * 4, done);
    if (e != cudaSuccess) return e;
    const int groups = (p.M + kTileRows - 1) / kTileRows * (kTileRows / kShRows);
    // a CTA for every adapter that a group can have while there is room for them on the
    // GPU; two otherwise, since a border between two adapters would take its group
    // twice as long
    const int room = 8 * current_sms() / groups;
    const int passes = room < 2 ? 2 : (room < kShRows ? room : kShRows);
    return launch_pdl(adapter_shrink_kernel<NT>, dim3(groups, passes), dim3(kShWarps * 32),
                      kShWarps * kShRows * p.rank * 4, s, p);
}

template <int BN, int NS, bool kPair, int EPI>
int launch_product_t(const AdapterArgs &p, const AdapterMaps &tm, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    auto k = kPair ? adapter_gemm_pair_kernel<kPair ? BN : 256, kPair ? NS : 5, EPI>
                   : adapter_gemm_kernel<kPair ? 64 : BN, kPair ? 6 : NS, EPI>;
    constexpr size_t ring =
        (size_t)NS * (kABytes + (kPair ? BN / 2 : BN) * kBK * 2) + 4 * kStageBytes + 1024;
    static_assert(ring + 2 * kABytes <= 226 * 1024, "shared memory");
    const size_t smem = ring + (p.rank + kBK - 1) / kBK * kABytes;   // and a tile's S
    cudaError_t e = allow_smem(k, ring + 2 * kABytes, done);
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(adapter gemm)");
    const int rows = kPair ? 2 * kBM : kBM, sms = current_sms();
    const int tiles = ((p.M + rows - 1) / rows) * (p.N / BN);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = kPair ? dim3(2 * (tiles < sms / 2 ? tiles : sms / 2)) : dim3(tiles < sms ? tiles : sms);
    cfg.blockDim = dim3(kAdThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = 2;
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = kPair ? 2 : 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, k, tm, p), "adapter_gemm_kernel");
}

template <int EPI>
int launch_split_t(const AdapterArgs &p, const AdapterMaps &tm, int c, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    auto k = adapter_gemm_split_kernel<EPI>;
    constexpr size_t ring = (size_t)kSplitStages * (kABytes + kSplitBN * kBK * 2) + 1024;
    cudaError_t e = allow_smem(k, ring + 2 * kABytes, done);
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(adapter gemm)");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c, (p.M + kBM - 1) / kBM * (p.N / kSplitBN));
    cfg.blockDim = dim3(kAdThreads);
    cfg.dynamicSmemBytes = ring + (p.rank + kBK - 1) / kBK * kABytes;
    cfg.stream = s;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = c;
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    return cuda_status(cudaLaunchKernelEx(&cfg, k, tm, p), "adapter_gemm_split_kernel");
}

// split: CTAs a tile (of 64 columns), 0: the other kernels
template <int BN, int NS, bool kPair = false>
int launch_product(const AdapterArgs &p, cudaStream_t s, int split = 0) {
    AdapterMaps tm;
    constexpr uint32_t box_n = kPair ? BN / 2 : BN;
    const uint64_t padded = (uint64_t)((p.M + kBM - 1) / kBM * kBM), rb = (uint64_t)p.rank * 2;
    const uint64_t xd[2] = {(uint64_t)p.K, (uint64_t)p.M}, xs[1] = {(uint64_t)p.ldx * 2};
    const uint64_t pd[2] = {(uint64_t)p.K, padded}, ps[1] = {(uint64_t)p.K * 2};
    const uint64_t wd[2] = {(uint64_t)p.K, (uint64_t)p.N}, ws[1] = {(uint64_t)p.ldw * 2};
    const uint64_t sd[2] = {(uint64_t)p.rank, padded}, ss[1] = {rb};
    const uint64_t ud[3] = {(uint64_t)p.rank, (uint64_t)p.N, (uint64_t)p.adapters};
    const uint64_t us[2] = {rb, rb * p.N};
    const uint32_t abox[2] = {kBK, (uint32_t)p.box_rows}, wbox[2] = {kBK, box_n}, ubox[3] = {kBK, box_n, 1};
    int st = encode_tmap(&tm.x, PK_DTYPE_BF16, p.x, 2, xd, xs, abox);
    if (st == PK_OK) st = encode_tmap(&tm.xs, PK_DTYPE_BF16, p.xs, 2, pd, ps, abox);
    if (st == PK_OK) st = encode_tmap(&tm.w, PK_DTYPE_BF16, p.W, 2, wd, ws, wbox);
    if (st == PK_OK) st = encode_tmap(&tm.s, PK_DTYPE_BF16, p.s, 2, sd, ss, abox);
    if (st == PK_OK) st = encode_tmap(&tm.up, PK_DTYPE_BF16, p.up, 3, ud, us, ubox);
    if (st != PK_OK) return st;
    if (split) switch (p.epilogue) {
            case PK_GEMM_SILU: return launch_split_t<PK_GEMM_SILU>(p, tm, split, s);
            case PK_GEMM_RESIDUAL: return launch_split_t<PK_GEMM_RESIDUAL>(p, tm, split, s);
            case PK_GEMM_RESIDUAL_RELU: return launch_split_t<PK_GEMM_RESIDUAL_RELU>(p, tm, split, s);
            case PK_GEMM_BIAS: return launch_split_t<PK_GEMM_BIAS>(p, tm, split, s);
            default: return launch_split_t<PK_GEMM_STORE>(p, tm, split, s);
        }
    switch (p.epilogue) {
        case PK_GEMM_SILU: return launch_product_t<BN, NS, kPair, PK_GEMM_SILU>(p, tm, s);
        case PK_GEMM_RESIDUAL: return launch_product_t<BN, NS, kPair, PK_GEMM_RESIDUAL>(p, tm, s);
        case PK_GEMM_RESIDUAL_RELU:
            return launch_product_t<BN, NS, kPair, PK_GEMM_RESIDUAL_RELU>(p, tm, s);
        case PK_GEMM_BIAS: return launch_product_t<BN, NS, kPair, PK_GEMM_BIAS>(p, tm, s);
        default: return launch_product_t<BN, NS, kPair, PK_GEMM_STORE>(p, tm, s);
    }
}

}  // namespace

int launch_adapter_plan(const int32_t *ids, int rows, int adapters, int32_t *plan, int32_t *error,
                        cudaStream_t s) {
    if (rows <= kTileRows)
        return cuda_status(launch_pdl(adapter_plan_tile_kernel, dim3(1), dim3(kTileRows), 0, s, ids, rows,
                                      adapters, adapter_layout(rows, adapters), plan, error),
                           "adapter_plan_kernel");
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(adapter_plan_kernel, kPlanCounts * 4, done);
    const PlanCut cut = plan_cut(rows, adapters);
    if (e == cudaSuccess)
        e = launch_pdl(adapter_plan_kernel, dim3(1), dim3(1024),
                       (size_t)(cut.chunks + 1) * (adapters + 1) * 4, s, ids, rows, adapters,
                       adapter_layout(rows, adapters), cut, plan, error);
    return cuda_status(e, "adapter_plan_kernel");
}

int launch_adapter_gemm(const AdapterArgs &a, cudaStream_t s) {
    AdapterArgs p = a;
    p.l = adapter_layout(p.M, p.adapters);
    p.box_rows = kBM;
    cudaError_t e = p.rank <= 8    ? launch_shrink<1>(p, s)
                    : p.rank <= 16 ? launch_shrink<2>(p, s)
                    : p.rank <= 32 ? launch_shrink<4>(p, s)
                    : p.rank <= 64 ? launch_shrink<8>(p, s)
                                   : launch_shrink<16>(p, s);
    if (e != cudaSuccess) return cuda_status(e, "adapter_shrink_kernel");
    // wide tiles where they still fill the GPU, narrow ones (more CTAs for the
    // weight stream) otherwise
    const int mtiles = (p.M + kBM - 1) / kBM, sms = current_sms();
    // CTA pairs as in pk_gemm.cu: their tiles fill a wave of pairs, and the waves are
    // at least 80 % full or K is long
    const int mt2 = (mtiles + 1) / 2, halves = sms / 2;
    const int t2 = p.N % 256 == 0 ? mt2 * (p.N / 256) : 0;
    if (t2 >= halves &&
        (p.K >= 2048 || 5 * t2 >= 4 * halves * ((t2 + halves - 1) / halves)))
        return launch_product<256, 5, true>(p, s);
    if (p.N % 256 == 0 && mtiles * (p.N / 256) >= 2 * sms) return launch_product<256, 3>(p, s);
    if (p.N % 128 == 0 && mtiles * (p.N / 128) >= sms) return launch_product<128, 5>(p, s);
    // two CTAs a tile while there are SMs for them, up to eight on half of the SMs: more
    // clusters of four or eight do not all find room in the GPCs at once (16 tiles of
    // K = 2048 on 1, 2, 4, 8 CTAs: 13.0, 9.2, 7.5, 13.0 us; 32: 13.9, 10.8, 10.4 us, with
    // an adapter 12.8 on two and 16.3 on four)
    const int tiles = mtiles * (p.N / kSplitBN), nk = p.K / kBK;
    const int split = 8 * tiles <= sms / 2 && nk >= 8   ? 8
                      : 4 * tiles <= sms / 2 && nk >= 4 ? 4
                      : 2 * tiles <= sms && nk >= 2     ? 2
                                                        : 1;
    if (split > 1) {
        // one row tile: no more of its rows than there are (8 a swizzle atom); the
        // others' sums are never read
        p.box_rows = mtiles > 1 ? kBM : (p.M + 7) / 8 * 8;
        return launch_product<64, 6>(p, s, split);
    }
    return launch_product<64, 6>(p, s);
}

}  // namespace pk
