// What the tree-attention kernels (pk_tree_attn.cu, pk_tree_attn_tc.cu) share: the
// walk over a CTA's part of the step's work, and small device helpers.
#pragma once

#include "pk_common.cuh"
#include "pk_internal.h"

namespace pk {
namespace {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&v);
}
__device__ __forceinline__ void fence_async_proxy() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// Bounded wait that gives up (false) at once when another wait of the CTA already has.
__device__ __forceinline__ bool ring_wait(uint64_t *bar, uint32_t parity, volatile int *failed,
                                          int32_t *error) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*failed) return false;
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (*failed) return false;
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
            *failed = 1;
            raise(error, PK_DEV_TIMEOUT);
            return false;
        }
    }
    return true;
}

// kv_map's copy of a page's rows from `row` on (a multiple of 8): groups of 8 rows, in
// each the 64-column blocks, 1024 bytes a block.
__device__ __forceinline__ void tma_load_rows(void *dst, const CUtensorMap *map, uint64_t *bar,
                                              int32_t row, int32_t plane) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(0), "r"(0), "r"(row >> 3), "r"(plane),
        "r"(smem_u32(bar))
        : "memory");
}
// Byte of a tile laid out so: row, 16-byte chunk of the row (8 a column block).
template <int DH>
__device__ __forceinline__ uint32_t tile_at(uint32_t row, uint32_t chunk) {
    return (row >> 3) * (DH / 64 * 1024) + (chunk >> 3) * 1024 + (row & 7) * 128 +
           (((chunk ^ row) & 7) << 4);
}

// A row tile of one request and K/V head over key tiles [t0, t1).
struct Unit {
    int slot, row0, count, ctx;   // the request: table row, first row, tokens, context
    int head, rt, t0, t1;
    int part;                     // where its partial result goes, -1: it has all keys
};

// The units of one CTA, in order: a walk over its share of the line of tiles.
struct Work {
    const TreeParams &p;
    int cta, b, nr, kt;   // request, its row tiles and key tiles
    int head, rt, at;     // the next unit's K/V head, row tile and place in it
    int left;             // places (or row tiles) left to this worker
    bool whole;
    Unit u;

    __device__ __forceinline__ Work(const TreeParams &params, int c) : p(params), cta(c) {
        b = p.step[p.l.first + c];
        const int share = p.step[kTokShare];
        whole = share == 0;
        left = 0;
        if (b < 0) return;
        load();
        const int64_t *work = reinterpret_cast<const int64_t *>(p.step + p.l.work);
        const int64_t each = whole ? p.step[kTokPer] : share, from = c * each, local = from - work[b];
        left = (int)min(each, work[p.batch] - from);
        int64_t item = local;
        at = 0;
        if (!whole) {
            const int places = kt + p.shape.lead;
            item = local / places;
            at = (int)(local - item * places);
        }
        head = (int)(item / nr);
        rt = (int)(item - (int64_t)head * nr);
    }
    __device__ __forceinline__ void load() {
        u.ctx = p.step[p.l.context + b];
        u.slot = p.step[p.l.slot + b];
        u.row0 = p.step[p.l.row_start + b];
        u.count = p.step[p.l.row_start + b + 1] - u.row0;
        nr = u.ctx < 0 ? 0 : (int)(((int64_t)u.count * p.group + p.shape.rows - 1) / p.shape.rows);
        kt = (u.ctx + u.count + p.shape.keys - 1) / p.shape.keys;
    }
    __device__ __forceinline__ bool next() {
        do {
            if (left <= 0) return false;
            if (head == p.kv_heads) {   // the next request that has rows
                do {
                    if (++b >= p.batch) return false;
                    load();
                } while (nr == 0);
                head = 0;
            }
            u.head = head;
            u.rt = rt;
            if (whole) {
                u.t0 = 0;
                u.t1 = kt;
                u.part = -1;
                --left;
                at = 0;
            } else {
                const int lead = p.shape.lead, n = min(kt + lead - at, left);
                u.t0 = max(at - lead, 0);
                u.t1 = max(at + n - lead, 0);
                u.part = u.t1 - u.t0 == kt ? -1 : (u.t0 == 0 ? 2 * cta + 1 : 2 * cta);
                left -= n;
                at = at + n == kt + lead ? 0 : at + n;
            }
            if (at == 0 && ++rt == nr) {
                rt = 0;
                ++head;
            }
        } while (u.t0 == u.t1);   // empty places alone
        if (!p.trees) {   // a chain's rows see no key past their own
            const int64_t last = ((int64_t)(u.rt + 1) * p.shape.rows + p.group - 1) / p.group;
            const int seen = u.ctx + (int)min(last, (int64_t)u.count);
            u.t1 = min(u.t1, (seen + p.shape.keys - 1) / p.shape.keys);
        }
        return true;
    }
};

// Whether a row tile whose places begin at `from` is shared by CTAs c0 .. c1.
__device__ __forceinline__ bool shared_by(const TreeParams &p, int64_t from, int kt, int64_t share,
                                          int &c0, int &c1) {
    c0 = (int)((from + p.shape.lead) / share);
    c1 = (int)((from + p.shape.lead + kt - 1) / share);
    return c0 != c1;
}

// Page ids of a unit's tiles, for the warp that issues their loads: 32 table entries
// at a time, one in a lane, the next 32 requested ahead.  (A load of its own for each
// tile puts its latency, as long as a tile's share of the memory rate, between the
// tiles.)  The pages of a tile never cross a multiple of 32: a tile has a power of
// two of them, or one.
struct Pages {
    const int32_t *table;
    int width, block, ids, ahead;

    __device__ __forceinline__ int fetch(int at) const {
        const int i = at + (threadIdx.x & 31);
        return i < width ? table[i] : -1;
    }
    // the first entries of a unit; used a unit before it begins
    __device__ __forceinline__ void open(const TreeParams &p, const Unit &w) {
        table = p.table + (int64_t)w.slot * p.table_width;
        width = p.table_width;
        block = ((w.t0 * p.shape.keys) >> p.ps_shift) & ~31;
        ids = fetch(block);
        ahead = fetch(block + 32);
    }
    // entry `at` of the caller's lane; uniform in at / 32
    __device__ __forceinline__ int get(int at) {
        while (at >= block + 32) {
            ids = ahead;
            block += 32;
            ahead = fetch(block + 32);
        }
        return __shfl_sync(0xffffffffu, ids, at & 31);
    }
};

// The V row of a unit's key in its page (bf16).
template <int DH>
__device__ __forceinline__ const __nv_bfloat16 *value_row(const TreeParams &p, const Unit &w,
                                                          int key) {
    int64_t page = p.table[(int64_t)w.slot * p.table_width + (key >> p.ps_shift)];
    if (page < 0 || page >= p.num_pages) page = 0;   // (the loads have reported it)
    const int64_t plane = ((page * p.num_layers + p.layer) * 2 + 1) * p.kv_heads + w.head;
    const int64_t row = (plane << p.ps_shift) + (key & ((1 << p.ps_shift) - 1));
    return static_cast<const __nv_bfloat16 *>(p.kv) + row * DH;
}

}  // namespace
}  // namespace pk
