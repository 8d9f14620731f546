// A projection shared by many requests, with each request's low-rank adapter:
//
//   acc[m] = x[m] W^T + S[m] up[a]^T,   S[m] = scale[a] * x[m] down[a]^T,  a = ids[m]
//   C[m]   = epilogue(acc[m])           (rows with ids[m] = -1: x[m] W^T alone)
//
// Three launches:
//  1. the plan (once per step: every projection of a model uses the same ids)
//     sorts the rows by adapter, so that a 128-row tile meets few adapters, and
//     lists each tile's (adapter, rows) pairs;
//  2. S in bf16 and the rows' sorted copy, bound by reading and writing them;
//  3. the product on the tcgen05 tensor cores, over the sorted rows; after the K
//     blocks of x W^T each pair of the tile adds one K block S up[a]^T into the same
//     accumulator, with the lanes of other rows disabled in the MMA: they get no zero
//     products, so one adapter's weights, whatever they hold, do not reach another's
//     rows.  The epilogue writes the rows back to their own places.
//
// S is rounded to bf16 because the tensor cores take it so: off by 2^-8 of each of
// its terms at most, as the bf16 result is of their sum.  Sums are
// fp32 throughout and in a fixed order.
#include "pk_common.cuh"
#include "pk_internal.h"
#include "pk_umma.cuh"

namespace pk {
namespace {

constexpr int kTileRows = 128;

// ------------------------------------------------------------------ the plan
__global__ void __launch_bounds__(1024) adapter_plan_kernel(const int32_t *ids, int rows,
                                                            int adapters, AdapterLayout l,
                                                            int32_t *plan, int32_t *error) {
    extern __shared__ int s_bin[];   // [adapters + 1] (the last: rows without one)
    __shared__ int s_warp[33], s_base, s_pairs, s_moved;
    grid_dep_wait();
    grid_dep_launch();
    const int tid = threadIdx.x, lane = tid & 31, bins = adapters + 1;
    const int tiles = (rows + kTileRows - 1) / kTileRows;
    for (int i = tid; i < bins; i += blockDim.x) s_bin[i] = 0;
    if (tid == 0) s_base = s_pairs = s_moved = 0;
    __syncthreads();
    // a thread's rows tid, tid + 1024, ...: the first kHeld of them are read once, all
    // at a time
    constexpr int kHeld = 8;
    const int padded = (rows + 31) / 32 * 32;
    auto bin_of = [&](int r) {   // -1 behind the last row
        if (r >= rows) return -1;
        const int a = ids[r];
        return a >= 0 && a < adapters ? a : adapters;
    };
    int held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = bin_of(tid + i * 1024);
    // one atomic for a warp whose rows agree, one a row otherwise (a match over the
    // warp's ids costs more than the conflicts that it saves)
    auto count = [&](int a) {
        if (__all_sync(0xffffffffu, a == __shfl_sync(0xffffffffu, a, 0))) {
            if (lane == 0 && a >= 0) atomicAdd(&s_bin[a], 32);
        } else if (a >= 0) {
            atomicAdd(&s_bin[a], 1);
        }
    };
    bool moved = false;   // a row whose adapter is above the next one's
    auto look = [&](int r, int a) {
        int next = __shfl_down_sync(0xffffffffu, a, 1);
        if (lane == 31) next = bin_of(r + 1);
        moved |= r + 1 < rows && a > next;
        if (r < rows && (ids[r] < -1 || ids[r] >= adapters)) raise(error, PK_DEV_BAD_SLOT);
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        if (i * 1024 < rows) {
            count(held[i]);
            look(tid + i * 1024, held[i]);
        }
    for (int r = tid + kHeld * 1024; r < padded; r += 1024) {
        const int a = bin_of(r);
        count(a);
        look(r, a);
    }
    if (moved) s_moved = 1;
    __syncthreads();
    // each adapter's first sorted row and first pair (it has one for each tile that
    // its rows touch), 1024 adapters at a time
    int32_t *pair = plan + l.pairs;
    for (int i = tid; i < tiles + 1; i += blockDim.x) plan[l.tile_pair + i] = 0x7fffffff;
    for (int a0 = 0; a0 < bins; a0 += blockDim.x) {
        const int a = a0 + tid, n = a < bins ? s_bin[a] : 0;
        auto scan = [&](int v, int &total) {
            int x = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            if (lane == 31) s_warp[tid >> 5] = x;
            __syncthreads();
            if (tid < 32) {
                int t = s_warp[tid];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, t, o);
                    if (lane >= o) t += y;
                }
                s_warp[tid] = t;
                if (tid == 31) s_warp[32] = t;
            }
            __syncthreads();
            total = s_warp[32];
            const int res = (tid >= 32 ? s_warp[(tid >> 5) - 1] : 0) + x - v;
            __syncthreads();
            return res;
        };
        int total;
        const int first = s_base + scan(n, total);
        __syncthreads();
        if (tid == 0) s_base += total;
        const int t0 = first / kTileRows, t1 = n ? (first + n - 1) / kTileRows : t0 - 1;
        const int mine = a < adapters && n ? t1 - t0 + 1 : 0;
        const int p0 = s_pairs + scan(mine, total);
        __syncthreads();
        if (tid == 0) s_pairs += total;
        if (a < bins) s_bin[a] = first;   // the sort's running position
        for (int i = 0; i < mine; ++i) {
            const int t = t0 + i, lo = max(first - t * kTileRows, 0);
            const int hi = min(first + n - t * kTileRows, kTileRows);
            pair[2 * (p0 + i)] = a;
            pair[2 * (p0 + i) + 1] = lo | hi << 16;
            if (lo == 0) plan[l.tile_pair + t] = p0 + i;
        }
        __syncthreads();
    }
    // tiles that no adapter's rows begin: past all of them
    for (int i = tid; i < tiles + 1; i += blockDim.x)
        if (plan[l.tile_pair + i] == 0x7fffffff) plan[l.tile_pair + i] = s_pairs;
    const bool resort = s_moved != 0;
    auto place = [&](int r, int a) {
        int at = r;
        if (resort) {
            if (__all_sync(0xffffffffu, a == __shfl_sync(0xffffffffu, a, 0))) {
                if (lane == 0 && a >= 0) at = atomicAdd(&s_bin[a], 32);
                at = __shfl_sync(0xffffffffu, at, 0) + lane;
            } else if (a >= 0) {
                at = atomicAdd(&s_bin[a], 1);
            }
        }
        if (a >= 0) plan[l.order + at] = r;
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        if (i * 1024 < rows) place(tid + i * 1024, held[i]);
    for (int r = tid + kHeld * 1024; r < padded; r += 1024) place(r, bin_of(r));
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
// Reading x and writing its copy bound it: 6720 x 4096, rank 32, 64 adapters, 110 MB.
// Tiles staged in shared memory with a barrier a stage took 46 us.
constexpr int kShWarps = 8, kShRows = 16;

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NT>   // 8-column tiles of S: rank <= 8 NT
__global__ void __launch_bounds__(kShWarps * 32, NT <= 4 ? 3 : 2)
    adapter_shrink_kernel(const AdapterArgs p) {
    extern __shared__ float sh_part[];   // [warp][row][rank]
    __shared__ int2 s_pair[kShRows];     // the group's pairs: adapter, first | end << 16
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
            if (q + lane < pair1) pr = reinterpret_cast<const int2 *>(plan + p.l.pairs)[q + lane];
            const int lo = max((pr.y & 0xffff) - g0, 0), hi = min((pr.y >> 16) - g0, kShRows);
            const unsigned has = __ballot_sync(0xffffffffu, lo < hi);
            if (lo < hi) s_pair[n + __popc(has & ((1u << lane) - 1u))] = make_int2(pr.x, lo | hi << 16);
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
        const int lo = pr.y & 0xffff, hi = pr.y >> 16;
        const __nv_bfloat16 *down =
            static_cast<const __nv_bfloat16 *>(p.down) + ((int64_t)pr.x * r + fr) * p.K + fc;
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
        for (int kb = warp; kb < nk; kb += kShWarps) {
            uint4 a[2][2];   // columns fc .. + 7 of both halves of the block
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                a[h][0] = in0 ? *reinterpret_cast<const uint4 *>(x0 + kb * 64 + h * 32) : zero;
                a[h][1] = in1 ? *reinterpret_cast<const uint4 *>(x1 + kb * 64 + h * 32) : zero;
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
            if (row < lo || row >= hi) continue;
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
// Lanes outside a pair's rows, 32 a word.
__device__ __forceinline__ void lanes_off(int range, uint32_t *off) {
    const int lo = range & 0xffff, hi = range >> 16;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int a = max(lo - w * 32, 0), b = min(hi - w * 32, 32);
        const uint32_t below = b >= 32 ? 0xffffffffu : (b > 0 ? (1u << b) - 1u : 0u);
        const uint32_t skip = a >= 32 ? 0xffffffffu : (1u << a) - 1u;
        off[w] = ~(below & ~skip);
    }
}

// The pairs p0 .. p1 of a tile, read eight at a time: the first eight when the tile
// begins, so that the reads' latency (one a pair took 0.4 us of a pair's turn) is
// under the K blocks before them.
struct TilePairs {
    const int2 *pairs;
    int p0, p1;
    int2 ahead[8];
    __device__ __forceinline__ TilePairs(const int2 *all, int from, int to)
        : pairs(all), p0(from), p1(to) {
        fetch();
    }
    __device__ __forceinline__ void fetch() {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            ahead[i] = p0 + i < p1 ? pairs[p0 + i] : make_int2(0, 0);
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
    const int2 *pairs = reinterpret_cast<const int2 *>(p.plan + p.l.pairs);
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
    // wait until stage g of the ring is free; false when a wait of the CTA gave up
    auto free_stage = [&](int g) {
        const int u = g / NS;
        if (u >= 1 && !failed && !mbar_wait_bounded(&empty[g % NS], (u - 1) & 1, kWaitLimitNs)) {
            raise(p.error, PK_DEV_TIMEOUT);
            failed = 1;
        }
        return !failed;
    };

    if (warp == 0) {
        if (lane == 0) {
            // producer.  The weights of the first stages do not depend on the kernel
            // before: they are requested ahead of the wait for it.
            const int pre = (int)blockIdx.x < tiles ? (nk < NS ? nk : NS) : 0;
            for (int kb = 0; kb < pre; ++kb) {
                mbar_arrive_expect_tx(&full[kb], kABytes + kBBytes);
                tma_load_2d(sB + kb * kBBytes, &tm.w, &full[kb], kb * kBK,
                            ((int)blockIdx.x / mtiles) * BN);
            }
            grid_dep_wait();
            const CUtensorMap *rows = *sorted ? &tm.x : &tm.xs;
            int g = 0, with_s = 0;   // ring uses; tiles that had an S
            bool ok = true;
            for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
                const int mt = tile % mtiles, m0 = mt * kBM, n0 = (tile / mtiles) * BN;
                TilePairs of_tile(pairs, tile_pair[mt], tile_pair[mt + 1]);
                for (int kb = 0; kb < nk; ++kb, ++g) {
                    const int s = g % NS;
                    if (g >= pre) {
                        if (!(ok = free_stage(g))) break;
                        mbar_arrive_expect_tx(&full[s], kABytes + kBBytes);
                        tma_load_2d(sB + s * kBBytes, &tm.w, &full[s], kb * kBK, n0);
                    }
                    tma_load_2d(sA + s * kABytes, rows, &full[s], kb * kBK, m0);
                }
                if (!ok || of_tile.p0 == of_tile.p1) continue;
                // S once a tile (a copy for each pair made every CTA of a row tile ask for
                // the same few lines again and again: 0.65 us a pair)
                if (with_s >= 1 && !mbar_wait_bounded(&s_empty, (with_s - 1) & 1, kWaitLimitNs)) {
                    raise(p.error, PK_DEV_TIMEOUT);
                    failed = 1;
                    ok = false;
                    break;
                }
                ++with_s;
                mbar_arrive_expect_tx(&s_full, rblocks * kABytes);
                for (int rb = 0; rb < rblocks; ++rb)
                    tma_load_2d(sS + rb * kABytes, &tm.s, &s_full, rb * kBK, m0);
                of_tile.each([&](int2 pr) {
                    for (int rb = 0; rb < rblocks; ++rb, ++g) {
                        const int s = g % NS;
                        if (!(ok = free_stage(g))) return false;
                        mbar_arrive_expect_tx(&full[s], kBBytes);
                        tma_load_3d(sB + s * kBBytes, &tm.up, &full[s], rb * kBK, n0, pr.x);
                    }
                    return true;
                });
            }
            if (!ok) {   // leave no copy in flight
                for (int s = 0; s < NS; ++s)
                    if (g > s) mbar_wait_bounded(&full[s], ((g - 1 - s) / NS) & 1, kWaitLimitNs);
                if (with_s) mbar_wait_bounded(&s_full, (with_s - 1) & 1, kWaitLimitNs);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = idesc_bf16(kBM, BN);
            grid_dep_wait();   // the plan
            int g = 0, t = 0, with_s = 0;
            auto done = [&](uint64_t *bar, uint32_t parity) {
                if (mbar_wait_bounded(bar, parity, kWaitLimitNs)) return true;
                raise(p.error, PK_DEV_TIMEOUT);
                failed = 1;
                return false;
            };
            auto ready = [&](int s) { return done(&full[s], (g / NS) & 1); };
            for (int tile = blockIdx.x; tile < tiles && !failed; tile += gridDim.x, ++t) {
                const int acc = t & 1, use = t >> 1, mt = tile % mtiles;
                if (use >= 1 && !mbar_wait_bounded(&tmem_empty[acc], (use - 1) & 1, kWaitLimitNs)) {
                    raise(p.error, PK_DEV_TIMEOUT);
                    failed = 1;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem + acc * BN;
                TilePairs of_tile(pairs, tile_pair[mt], tile_pair[mt + 1]);
                for (int kb = 0; kb < nk; ++kb, ++g) {
                    const int s = g % NS;
                    if (!ready(s)) break;
                    tc_fence_after();
                    const uint32_t a0 = smem_u32(sA + s * kABytes), b0 = smem_u32(sB + s * kBBytes);
#pragma unroll
                    for (int kk = 0; kk < kBK / 16; ++kk)
                        umma_bf16(d, sw128_desc(a0 + kk * 32), sw128_desc(b0 + kk * 32), idesc,
                                  (kb | kk) != 0);
                    umma_commit(&empty[s]);
                }
                const bool any = of_tile.p0 < of_tile.p1;
                if (any && !failed) done(&s_full, with_s++ & 1);
                of_tile.each([&](int2 pr) {
                    uint32_t off[4];
                    lanes_off(pr.y, off);
                    for (int rb = 0; rb < rblocks; ++rb, ++g) {
                        const int s = g % NS;
                        if (failed || !ready(s)) return false;
                        tc_fence_after();
                        const uint32_t a0 = smem_u32(sS + rb * kABytes),
                                       b0 = smem_u32(sB + s * kBBytes);
                        const int steps = min(kBK, p.rank - rb * kBK);
                        for (int kk = 0; kk * 16 < steps; ++kk)
                            umma_bf16_lanes(d, sw128_desc(a0 + kk * 32), sw128_desc(b0 + kk * 32),
                                            idesc, off);
                        umma_commit(&empty[s]);
                    }
                    return true;
                });
                if (any) umma_commit(&s_empty);
                umma_commit(&tmem_full[acc]);
            }
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
    const int2 *pairs = reinterpret_cast<const int2 *>(p.plan + p.l.pairs);
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
    auto free_stage = [&](int g) {
        const int u = g / NS;
        if (u >= 1 && !failed && !mbar_wait_bounded(&empty[g % NS], (u - 1) & 1, kWaitLimitNs)) {
            raise(p.error, PK_DEV_TIMEOUT);
            failed = 1;
        }
        return !failed;
    };

    if (warp == 0) {
        if (lane == 0) {
            grid_dep_wait();
            const CUtensorMap *rows = *sorted ? &tm.x : &tm.xs;
            int g = 0, with_s = 0;   // ring uses; tiles that had an S
            bool ok = true;
            const uint32_t sb = mapa_rank(smem_u32(&s_full), 0);
            for (int tile = pair; tile < tiles && ok; tile += npairs) {
                const int mt = tile % mtiles, m0 = mt * 2 * kBM + (int)rank * kBM;
                const int n0 = (tile / mtiles) * BN + (int)rank * kHalfB;
                TilePairs of_tile(pairs, tile_pair[2 * mt], tile_pair[min(2 * mt + 2, halves)]);
                for (int kb = 0; kb < nk; ++kb, ++g) {
                    if (!(ok = free_stage(g))) break;
                    const int s = g % NS;
                    const uint32_t fb = mapa_rank(smem_u32(&full[s]), 0);
                    if (leader) mbar_arrive_expect_tx(&full[s], kStageTx);
                    tma_load_2d_pair(sB + s * kBBytes, &tm.w, fb, kb * kBK, n0);
                    tma_load_2d_pair(sA + s * kABytes, rows, fb, kb * kBK, m0);
                }
                if (!ok || of_tile.p0 == of_tile.p1) continue;
                if (with_s >= 1 && !mbar_wait_bounded(&s_empty, (with_s - 1) & 1, kWaitLimitNs)) {
                    raise(p.error, PK_DEV_TIMEOUT);
                    failed = 1;
                    ok = false;
                    break;
                }
                ++with_s;
                if (leader) mbar_arrive_expect_tx(&s_full, 2 * rblocks * kABytes);
                for (int rb = 0; rb < rblocks; ++rb)
                    tma_load_2d_pair(sS + rb * kABytes, &tm.s, sb, rb * kBK, m0);
                of_tile.each([&](int2 pr) {
                    for (int rb = 0; rb < rblocks; ++rb, ++g) {
                        if (!(ok = free_stage(g))) return false;
                        const int s = g % NS;
                        const uint32_t fb = mapa_rank(smem_u32(&full[s]), 0);
                        if (leader) mbar_arrive_expect_tx(&full[s], 2 * kBBytes);
                        tma_load_3d_pair(sB + s * kBBytes, &tm.up, fb, rb * kBK, n0, pr.x);
                    }
                    return true;
                });
            }
            if (leader) {   // leave none of the pair's loads in flight
                for (int s = 0; s < NS; ++s)
                    if (g > s) mbar_wait_bounded(&full[s], ((g - 1 - s) / NS) & 1, kWaitLimitNs);
                if (with_s) mbar_wait_bounded(&s_full, (with_s - 1) & 1, kWaitLimitNs);
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            constexpr uint32_t idesc = idesc_bf16(2 * kBM, BN);
            grid_dep_wait();
            int g = 0, t = 0, with_s = 0;
            auto done = [&](uint64_t *bar, uint32_t parity) {
                if (mbar_wait_cluster_bounded(bar, parity, kWaitLimitNs)) return true;
                raise(p.error, PK_DEV_TIMEOUT);
                failed = 1;
                return false;
            };
            auto ready = [&](int s) { return done(&full[s], (g / NS) & 1); };
            for (int tile = pair; tile < tiles && !failed; tile += npairs, ++t) {
                const int acc = t & 1, use = t >> 1, mt = tile % mtiles;
                if (use >= 1 &&
                    !mbar_wait_cluster_bounded(&tmem_empty[acc], (use - 1) & 1, kWaitLimitNs)) {
                    raise(p.error, PK_DEV_TIMEOUT);
                    failed = 1;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem + acc * BN;
                const int border = tile_pair[min(2 * mt + 1, halves)];   // of the two halves
                TilePairs of_tile(pairs, tile_pair[2 * mt], tile_pair[min(2 * mt + 2, halves)]);
                for (int kb = 0; kb < nk; ++kb, ++g) {
                    const int s = g % NS;
                    if (!ready(s)) break;
                    tc_fence_after();
                    const uint32_t a0 = smem_u32(sA + s * kABytes), b0 = smem_u32(sB + s * kBBytes);
#pragma unroll
                    for (int kk = 0; kk < kBK / 16; ++kk)
                        umma_bf16_pair(d, sw128_desc(a0 + kk * 32), sw128_desc(b0 + kk * 32), idesc,
                                       (kb | kk) != 0);
                    umma_commit_pair(&empty[s]);
                }
                int pr_at = of_tile.p0;
                const bool any = of_tile.p0 < of_tile.p1;
                if (any && !failed) done(&s_full, with_s++ & 1);
                of_tile.each([&](int2 pr) {
                    const bool odd = pr_at++ >= border;   // the second half's
                    uint32_t off[8];
                    lanes_off(odd ? 0 : pr.y, off);
                    lanes_off(odd ? pr.y : 0, off + 4);
                    for (int rb = 0; rb < rblocks; ++rb, ++g) {
                        const int s = g % NS;
                        if (failed || !ready(s)) return false;
                        tc_fence_after();
                        const uint32_t a0 = smem_u32(sS + rb * kABytes), b0 = smem_u32(sB + s * kBBytes);
                        const int steps = min(kBK, p.rank - rb * kBK);
                        for (int kk = 0; kk * 16 < steps; ++kk)
                            umma_bf16_pair_lanes(d, sw128_desc(a0 + kk * 32),
                                                 sw128_desc(b0 + kk * 32), idesc, off);
                        umma_commit_pair(&empty[s]);
                    }
                    return true;
                });
                if (failed) break;
                if (any) umma_commit_pair(&s_empty);
                umma_commit_pair(&tmem_full[acc]);
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

template <int BN, int NS, bool kPair = false>
int launch_product(const AdapterArgs &p, cudaStream_t s) {
    AdapterMaps tm;
    constexpr uint32_t box_n = kPair ? BN / 2 : BN;
    const uint64_t padded = (uint64_t)((p.M + kBM - 1) / kBM * kBM), rb = (uint64_t)p.rank * 2;
    const uint64_t xd[2] = {(uint64_t)p.K, (uint64_t)p.M}, xs[1] = {(uint64_t)p.ldx * 2};
    const uint64_t pd[2] = {(uint64_t)p.K, padded}, ps[1] = {(uint64_t)p.K * 2};
    const uint64_t wd[2] = {(uint64_t)p.K, (uint64_t)p.N}, ws[1] = {(uint64_t)p.ldw * 2};
    const uint64_t sd[2] = {(uint64_t)p.rank, padded}, ss[1] = {rb};
    const uint64_t ud[3] = {(uint64_t)p.rank, (uint64_t)p.N, (uint64_t)p.adapters};
    const uint64_t us[2] = {rb, rb * p.N};
    const uint32_t abox[2] = {kBK, kBM}, wbox[2] = {kBK, box_n}, ubox[3] = {kBK, box_n, 1};
    int st = encode_tmap(&tm.x, PK_DTYPE_BF16, p.x, 2, xd, xs, abox);
    if (st == PK_OK) st = encode_tmap(&tm.xs, PK_DTYPE_BF16, p.xs, 2, pd, ps, abox);
    if (st == PK_OK) st = encode_tmap(&tm.w, PK_DTYPE_BF16, p.W, 2, wd, ws, wbox);
    if (st == PK_OK) st = encode_tmap(&tm.s, PK_DTYPE_BF16, p.s, 2, sd, ss, abox);
    if (st == PK_OK) st = encode_tmap(&tm.up, PK_DTYPE_BF16, p.up, 3, ud, us, ubox);
    if (st != PK_OK) return st;
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
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(adapter_plan_kernel, (PK_ADAPTER_MAX + 1) * 4, done);
    if (e == cudaSuccess)
        e = launch_pdl(adapter_plan_kernel, dim3(1), dim3(1024), (size_t)(adapters + 1) * 4, s, ids,
                       rows, adapters, adapter_layout(rows, adapters), plan, error);
    return cuda_status(e, "adapter_plan_kernel");
}

int launch_adapter_gemm(const AdapterArgs &a, cudaStream_t s) {
    AdapterArgs p = a;
    p.l = adapter_layout(p.M, p.adapters);
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
    return launch_product<64, 6>(p, s);
}

}  // namespace pk
