// Token pools: page tables, slot maps and tree masks from request lengths, and
// the cache traffic of a step (append, keep the accepted path, cut).
//
// For request b with len tokens kept, held pages and n new tokens:
//   take(b)  = max(ceil((len + n) / page_size) - held, 0)
//   page i of the step's new pages = free_pages[free_count - 1 - i], batch order
//   node j's cache row = table[(len + j) / page_size] * page_size + (len + j) % page_size
//   mask(j) = bit j | mask(parent(j)),  position(j) = len + |ancestors of j|
//
// The prefix sums over the batch (rows, pages, attention tiles) need every
// request, so one CTA makes them; what they place (rows, table entries, where each
// attention CTA begins) is written by that CTA too while there is little of it, and by a grid
// otherwise.  Masks come by doubling over the ancestors (mask |= mask[jump],
// jump = jump[jump]): 6 rounds of warp shuffles for 64 nodes, whatever the depth.
// Everything is integer work bound by latency: a few thousand rows are written
// faster than a second launch starts.  The pages go back in the order that
// restores the stack exactly, so a step that is cut back leaves no trace.
#include "pk_common.cuh"
#include "pk_internal.h"

namespace pk {
namespace {

constexpr int kPlanThreads = 1024;
// Rows (and twice the table entries) that the planning CTA writes itself: above
// it a second launch over the whole GPU is faster.
constexpr int kOneCtaRows = 2048;

struct TokParams {
    pk_token_kv_desc d;
    TokLayout l;
    TokShape shape;
    int ps_shift, row_shift, key_shift, group, kv_heads, batch, rows;
    const int32_t *slots, *counts, *parents;
    int32_t *step;
};

__device__ int64_t block_exclusive_sum64(int64_t v, int64_t &total, int64_t *s_warp) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s_warp[wid] = x;
    __syncthreads();
    if (wid == 0) {
        int64_t t = lane < nw ? s_warp[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += y;
        }
        if (lane < nw) s_warp[lane] = t;
        if (lane == 31) s_warp[32] = t;
    }
    __syncthreads();
    total = s_warp[32];
    const int64_t res = (wid > 0 ? s_warp[wid - 1] : 0) + x - v;
    __syncthreads();
    return res;
}

// The requests of one thread of the planning CTA, b0 .. b0 + NK - 1: contiguous, so
// that each prefix sum over the batch is one scan over the threads' sums, and in
// registers, so that their loads overlap.
//
// A slot may be named once.  Every slot of the batch is marked with the first
// request that names it; a slot out of range is nobody's.  The marks, one a slot of
// the pool, are in shared memory where they fit (kSharedMarks: a step and a truncation
// of 2048 requests took 24.9 us with the marks in global memory and take 21.3), in
// scratch[0 .. num_slots) otherwise.
// `state(slot, k)` is called for slots in range before the marks are settled, so that
// its loads run under them.
constexpr int kSharedMarks = 8192;
__host__ __device__ __forceinline__ size_t mark_bytes(int num_slots) {
    return num_slots <= kSharedMarks ? (size_t)num_slots * 4 : 0;
}
template <int NK, typename F>
__device__ __forceinline__ void own_slots(const pk_token_kv_desc &d, const int32_t *slots, int batch,
                                          int b0, int (&slot)[NK], bool (&own)[NK], F state) {
    extern __shared__ int32_t s_marks[];
    int32_t *marks = d.num_slots <= kSharedMarks ? s_marks : d.scratch;
#pragma unroll
    for (int k = 0; k < NK; ++k) slot[k] = b0 + k < batch ? slots[b0 + k] : -1;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
        own[k] = slot[k] >= 0 && slot[k] < d.num_slots;
        if (own[k]) {
            marks[slot[k]] = 0x7fffffff;
            state(slot[k], k);
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NK; ++k)
        if (own[k]) atomicMin(&marks[slot[k]], b0 + k);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NK; ++k) own[k] = own[k] && marks[slot[k]] == b0 + k;
}

__device__ __forceinline__ int ceil_shift(int64_t n, int shift) {
    return (int)((n + (1 << shift) - 1) >> shift);
}

// The cache row of a request's token: in a held page, or one of the step's (free stack, top
// first).  -1, and an error bit, where the table or the stack names no page of the pool.
__device__ __forceinline__ int row_of(const TokParams &p, int slot, int held, int first, int free_n,
                                      int tok) {
    const int i = tok >> p.ps_shift;
    const int page = i < held ? p.d.page_table[(int64_t)slot * p.d.table_width + i]
                              : p.d.free_pages[free_n - 1 - (first + i - held)];
    if ((unsigned)page >= (unsigned)p.d.num_pages) {
        raise(p.d.error, PK_DEV_BAD_PAGE);
        return -1;
    }
    return (page << p.ps_shift) | (tok & ((1 << p.ps_shift) - 1));
}

template <int NK>
__device__ void begin_plan(const TokParams &p) {
    __shared__ int64_t s_scan[33];
    __shared__ int s_taken, s_longest;
    const pk_token_kv_desc &d = p.d;
    int32_t *st = p.step;
    const int b0 = threadIdx.x * NK;
    const int free_n = *d.free_count;
    if (threadIdx.x == 0) {
        s_taken = free_n;
        s_longest = 0;
    }
    int slot[NK], count[NK], ctx[NK], held[NK], take[NK];
    bool own[NK];
#pragma unroll
    for (int k = 0; k < NK; ++k) count[k] = b0 + k < p.batch ? p.counts[b0 + k] : 0;
#pragma unroll
    for (int k = 0; k < NK; ++k) ctx[k] = held[k] = 0;
    own_slots<NK>(d, p.slots, p.batch, b0, slot, own, [&](int s, int k) {
        ctx[k] = d.lengths[s];
        held[k] = d.held[s];
    });
#pragma unroll
    for (int k = 0; k < NK; ++k)
        if (!own[k]) ctx[k] = -1;

    // rows; which requests can be served but for their pages
    int64_t sum = 0, total;
#pragma unroll
    for (int k = 0; k < NK; ++k) sum += max(count[k], 0);
    int64_t at = block_exclusive_sum64(sum, total, s_scan);
    int64_t takes = 0;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
        const int b = b0 + k, n = max(count[k], 0);
        take[k] = 0;
        if (b >= p.batch) continue;
        const int64_t len = (int64_t)ctx[k] + n;
        if (!own[k]) {
            raise(d.error, PK_DEV_BAD_SLOT);
        } else if (count[k] < 0 || at + n > p.rows || (p.parents && n > PK_TOK_MAX_TREE) ||
                   len > (int64_t)d.table_width << p.ps_shift) {
            raise(d.error, PK_DEV_BAD_COUNT);
            ctx[k] = -1;
        } else {
            take[k] = max(ceil_shift(len, p.ps_shift) - held[k], 0);
        }
        st[p.l.row_start + b] = (int)min(at, (int64_t)p.rows);
        st[p.l.slot + b] = slot[k];
        st[p.l.held + b] = held[k];
        takes += take[k];
        at += n;
    }
    if (threadIdx.x == 0) {
        const int used = (int)min(total, (int64_t)p.rows);
        st[p.l.row_start + p.batch] = used;
        st[kTokRows] = used;
        st[kTokFree] = free_n;
    }

    // pages, in batch order: from the first request that finds too few on, those that need
    // any are left out (nobody overtakes, and one prefix sum decides)
    int64_t first = block_exclusive_sum64(takes, total, s_scan);
    const int64_t all_takes = total;
    int64_t tiles = 0;
    int items = 0, longest = 0, nr[NK], kt[NK];   // row tiles and key tiles
#pragma unroll
    for (int k = 0; k < NK; ++k) {
        const int b = b0 + k;
        nr[k] = kt[k] = 0;
        if (b >= p.batch) continue;
        st[p.l.take + b] = (int)min(first, (int64_t)0x7fffffff);
        if (take[k] > 0 && first + take[k] > free_n) {
            raise(d.error, PK_DEV_POOL_EXHAUSTED);
            atomicMin(&s_taken, (int)min(first, (int64_t)free_n));   // the pages before it
            ctx[k] = -1;
        } else if (take[k] > 0) {
            d.held[slot[k]] = held[k] + take[k];
        }
        first += take[k];
        st[p.l.context + b] = ctx[k];
        if (ctx[k] >= 0 && count[k] > 0) {
            nr[k] = ceil_shift((int64_t)count[k] * p.group, p.row_shift);
            kt[k] = ceil_shift((int64_t)ctx[k] + count[k], p.key_shift);
        }
        tiles += (int64_t)nr[k] * (kt[k] + p.shape.lead);
        items += nr[k];
        longest = max(longest, kt[k]);
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    if ((threadIdx.x & 31) == 0 && longest) atomicMax(&s_longest, longest);

    // the attention's line of tiles: an equal share of it a worker, but the shape's least
    // at least (and two, while few workers have any); whole row tiles where the most of
    // them that a worker gets are no longer than that, or where a CTA takes one (167
    // requests of 14 rows and a few tokens, 8 heads: 33 us in shares, 15 whole)
    const int64_t items_before = block_exclusive_sum64(items, total, s_scan);
    const int64_t all_items = total * p.kv_heads;
    int64_t before = block_exclusive_sum64(tiles, total, s_scan);
    int64_t all = total * p.kv_heads;
    // (divisions, 0.3 us each, only where their results are not the bounds)
    const int least = all >= (int64_t)p.shape.least * p.shape.busy ? p.shape.least
                      : all < 3 * (int64_t)p.shape.busy            ? min(p.shape.least, 2)
                                                                   : (int)(all / p.shape.busy);
    int64_t share = least + p.shape.lead;
    if (all > share * p.shape.ctas) share = (all + p.shape.ctas - 1) / p.shape.ctas;
    const int64_t per = all_items <= p.shape.ctas ? 1 : (all_items + p.shape.ctas - 1) / p.shape.ctas;
    const bool whole = per * (s_longest + p.shape.lead) <=
                           max(share, (int64_t)(p.shape.least + p.shape.lead)) ||
                       (all_items <= p.shape.team && s_longest <= p.shape.team_keys);
    if (whole) {
        share = 0;
        before = items_before;
        all = all_items;
    }
    int64_t *work = reinterpret_cast<int64_t *>(st + p.l.work);
#pragma unroll
    for (int k = 0; k < NK; ++k) {
        if (b0 + k < p.batch) work[b0 + k] = before * p.kv_heads;
        before += whole ? nr[k] : (int64_t)nr[k] * (kt[k] + p.shape.lead);
    }
    if (threadIdx.x == 0) {
        work[p.batch] = all;
        st[kTokShare] = (int)min(share, (int64_t)0x7fffffff);
        st[kTokPer] = (int)per;
        *d.free_count = free_n - (int)min(all_takes, (int64_t)s_taken);
    }
    // CTAs behind the last tile
    const int64_t each = whole ? per : share, used = each == 1 ? all : (all + each - 1) / each;
    for (int64_t c = used + threadIdx.x; c < p.shape.ctas; c += blockDim.x) st[p.l.first + c] = -1;
}

// One value of a 64-entry array held two entries a lane (j, j + 32).
template <typename T>
__device__ __forceinline__ T shfl64(T lo, T hi, int j) {
    const T a = __shfl_sync(0xffffffffu, lo, j & 31), b = __shfl_sync(0xffffffffu, hi, j & 31);
    return j & 32 ? b : a;
}

// A tree's rows, by one warp: nodes lane and lane + 32.
__device__ void tree_rows(const TokParams &p, int b, int lane) {
    int32_t *st = p.step;
    const int r0 = st[p.l.row_start + b], n = st[p.l.row_start + b + 1] - r0;
    const int ctx = st[p.l.context + b], slot = st[p.l.slot + b], held = st[p.l.held + b];
    const int first = st[p.l.take + b], free_n = st[kTokFree];
    int64_t *mask = reinterpret_cast<int64_t *>(st + p.l.mask);
    if (ctx < 0) {   // left out: its rows may be more than a tree's
        for (int j = lane; j < n; j += 32) {
            st[p.l.request + r0 + j] = b;
            st[p.l.position + r0 + j] = 0;
            st[p.l.slot_map + r0 + j] = -1;
            mask[r0 + j] = 0;
        }
        return;
    }
    unsigned long long m[2];
    int jump[2], depth[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int j = lane + 32 * h;
        int par = -1;
        if (j < n) {
            par = p.parents[r0 + j];
            if (par < -1 || par >= j) {
                raise(p.d.error, PK_DEV_BAD_COUNT);
                par = -1;
            }
        }
        m[h] = 1ull << j;
        jump[h] = par;
        depth[h] = par >= 0;
    }
#pragma unroll 1
    for (int round = 0; round < 6; ++round) {
        unsigned long long nm[2];
        int nj[2], nd[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int j = max(jump[h], 0);
            const unsigned long long am = shfl64(m[0], m[1], j);
            const int aj = shfl64(jump[0], jump[1], j), ad = shfl64(depth[0], depth[1], j);
            const bool live = jump[h] >= 0;
            nm[h] = live ? m[h] | am : m[h];
            nd[h] = live ? depth[h] + ad : depth[h];
            nj[h] = live ? aj : -1;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            m[h] = nm[h];
            jump[h] = nj[h];
            depth[h] = nd[h];
        }
        if (__all_sync(0xffffffffu, jump[0] < 0 && jump[1] < 0)) break;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int j = lane + 32 * h;
        if (j < n) {
            st[p.l.request + r0 + j] = b;
            st[p.l.position + r0 + j] = ctx + depth[h];
            st[p.l.slot_map + r0 + j] = row_of(p, slot, held, first, free_n, ctx + j);
            mask[r0 + j] = (int64_t)m[h];
        }
    }
}

// What the prefix sums place, by warps w of nw: the requests' new table entries,
// CTAs and tree rows a request at a time; chain rows and the rows behind
// the last request a row at a time.
__device__ void begin_fill(const TokParams &p, int w, int nw) {
    int32_t *st = p.step;
    const int lane = threadIdx.x & 31;
    const int free_n = st[kTokFree];
    const int64_t share = st[kTokShare] > 0 ? st[kTokShare] : st[kTokPer];
    const int64_t *work = reinterpret_cast<const int64_t *>(st + p.l.work);
    for (int b = w; b < p.batch; b += nw) {
        const int ctx = st[p.l.context + b];
        if (ctx >= 0) {
            const int r0 = st[p.l.row_start + b], n = st[p.l.row_start + b + 1] - r0;
            const int slot = st[p.l.slot + b], held = st[p.l.held + b], first = st[p.l.take + b];
            const int need = ceil_shift((int64_t)ctx + n, p.ps_shift);
            for (int i = held + lane; i < need; i += 32)
                p.d.page_table[(int64_t)slot * p.d.table_width + i] =
                    p.d.free_pages[free_n - 1 - (first + i - held)];
            // the CTAs that begin in this request
            const int64_t w0 = work[b], w1 = work[b + 1];
            for (int64_t c = (w0 + share - 1) / share + lane; c * share < w1; c += 32)
                st[p.l.first + c] = b;
        }
        if (p.parents) tree_rows(p, b, lane);
    }
    const int used = st[kTokRows];
    for (int r = (p.parents ? used : 0) + w * 32 + lane; r < p.rows; r += nw * 32) {
        int req = -1, pos = 0, map = -1;
        if (r < used) {
            int lo = 0, hi = p.batch;   // the last request that starts at or before row r
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (st[p.l.row_start + mid] <= r) lo = mid;
                else hi = mid;
            }
            req = lo;
            const int ctx = st[p.l.context + lo];
            if (ctx >= 0) {
                pos = ctx + r - st[p.l.row_start + lo];
                map = row_of(p, st[p.l.slot + lo], st[p.l.held + lo], st[p.l.take + lo], free_n, pos);
            }
        }
        st[p.l.request + r] = req;
        st[p.l.position + r] = pos;
        st[p.l.slot_map + r] = map;
        if (p.parents) reinterpret_cast<int64_t *>(st + p.l.mask)[r] = 0;
    }
}

template <int NK, bool kFill>
__global__ void __launch_bounds__(kPlanThreads) token_begin_kernel(const TokParams p) {
    grid_dep_wait();
    grid_dep_launch();
    begin_plan<NK>(p);
    if (kFill) {
        __syncthreads();
        begin_fill(p, threadIdx.x >> 5, blockDim.x >> 5);
    }
}

__global__ void __launch_bounds__(256) token_fill_kernel(const TokParams p) {
    grid_dep_wait();
    grid_dep_launch();
    begin_fill(p, (blockIdx.x * blockDim.x + threadIdx.x) >> 5, (gridDim.x * blockDim.x) >> 5);
}

__global__ void token_reset_kernel(pk_token_kv_desc d, const int32_t *order) {
    grid_dep_wait();
    grid_dep_launch();
    const int64_t tid = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t n = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = tid; i < d.num_pages; i += n) d.free_pages[i] = order ? order[i] : (int)i;
    for (int64_t i = tid; i < (int64_t)d.num_slots * d.table_width; i += n) d.page_table[i] = -1;
    for (int64_t i = tid; i < d.num_slots; i += n) {
        d.lengths[i] = 0;
        d.held[i] = 0;
    }
    if (tid == 0) {
        *d.free_count = d.num_pages;
        *d.error = 0;
    }
}

// ------------------------------------------------------------------ append
// 16 bytes a thread: a row's K and V of one layer, head by head.
__global__ void __launch_bounds__(256)
    token_append_kernel(pk_token_kv_desc d, TokAppendArgs a, int64_t slot_map, int ps_shift,
                        int esize) {
    grid_dep_wait();
    grid_dep_launch();
    const int per_head = d.head_dim * esize / 16, per_row = per_head * d.num_kv_heads;
    const int64_t n = (int64_t)a.rows * per_row;
    const int layer = blockIdx.y;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / per_row;
        const int c = (int)(i - r * per_row), h = c / per_head, e = c - h * per_head;
        const int map = a.step[slot_map + r];
        if (map < 0) continue;
        if (map >> ps_shift >= d.num_pages) {   // a step block that was written to
            raise(d.error, PK_DEV_BAD_PAGE);
            continue;
        }
        const int64_t src = (layer * a.ls + r * a.rs + h * a.hs) * esize + e * 16;
        const uint4 k = *reinterpret_cast<const uint4 *>(static_cast<const char *>(a.key) + src);
        const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const char *>(a.value) + src);
        const int64_t page = map >> ps_shift, off = map & (d.page_size - 1);
        const int64_t plane = ((page * d.num_layers + a.layer0 + layer) * 2) * d.num_kv_heads + h;
        char *kv = static_cast<char *>(d.kv) + (plane * d.page_size + off) * d.head_dim * esize +
                   e * 16;
        *reinterpret_cast<uint4 *>(kv) = k;
        *reinterpret_cast<uint4 *>(kv + (int64_t)d.num_kv_heads * d.page_size * d.head_dim *
                                            esize) = v;
    }
}

// --------------------------------------------------------------- acceptance
// One CTA per (request, layer).  The path's nodes p_0 < p_1 < ... go to rows
// len, len + 1, ...: p_i >= i, so in ascending order no row is overwritten before
// it has been read, and kAhead rows are read before the first of them is written.
constexpr int kAhead = 8;
__global__ void __launch_bounds__(256)
    token_end_kernel(pk_token_kv_desc d, TokLayout l, const int32_t *last, int trees,
                     const int32_t *step, int ps_shift, int esize) {
    __shared__ int s_src[PK_TOK_MAX_TREE], s_dst[PK_TOK_MAX_TREE], s_n;
    grid_dep_wait();
    grid_dep_launch();
    const int b = blockIdx.x, layer = blockIdx.y;
    const int ctx = step[l.context + b];
    if (ctx < 0) return;
    const int r0 = step[l.row_start + b], n = step[l.row_start + b + 1] - r0;
    const int slot = step[l.slot + b];
    int keep = last[b];
    // pages given back since the step began: the request has been cut (or the pool
    // reset), and a length past its pages would read what others write there
    if (((int64_t)d.held[slot] << ps_shift) < (int64_t)ctx + n) {
        if (layer == 0 && threadIdx.x == 0) raise(d.error, PK_DEV_BAD_COUNT);
        return;
    }
    if (keep < -1 || keep >= n) {
        if (layer == 0 && threadIdx.x == 0) raise(d.error, PK_DEV_BAD_COUNT);
        keep = -1;
    }
    unsigned long long path = 0;
    if (trees && keep >= 0)
        path = (unsigned long long)reinterpret_cast<const int64_t *>(step + l.mask)[r0 + keep];
    const int kept = trees ? __popcll(path) : keep + 1;
    if (layer == 0 && threadIdx.x == 0) d.lengths[slot] = ctx + kept;
    // a path of nodes 0, 1, ... is in place already (every chain)
    if (!trees || path == (kept >= 64 ? ~0ull : (1ull << kept) - 1ull)) return;
    const int in_place = __ffsll(~path) - 1;   // nodes 0 .. in_place - 1 stay
    if (threadIdx.x < PK_TOK_MAX_TREE && (path >> threadIdx.x & 1) &&
        (int)threadIdx.x >= in_place) {
        const int rank = __popcll(path & ((1ull << threadIdx.x) - 1ull));
        int src = step[l.slot_map + r0 + threadIdx.x];
        const int dst = step[l.slot_map + r0 + rank];
        if ((unsigned)src >> ps_shift >= (unsigned)d.num_pages ||
            (unsigned)dst >> ps_shift >= (unsigned)d.num_pages) {
            raise(d.error, PK_DEV_BAD_PAGE);
            src = -1;   // not moved
        }
        s_src[rank - in_place] = src;
        s_dst[rank - in_place] = dst;
    }
    if (threadIdx.x == 0) s_n = kept - in_place;
    __syncthreads();
    const int moves = s_n;
    const int per_head = d.head_dim * esize / 16;
    const int64_t row_bytes = (int64_t)d.head_dim * esize;
    for (int c = threadIdx.x; c < 2 * d.num_kv_heads * per_head; c += blockDim.x) {
        const int plane = c / per_head, e = c - plane * per_head;   // (K|V, head)
        auto at = [&](int map) {
            const int64_t page = map >> ps_shift, off = map & (d.page_size - 1);
            return static_cast<char *>(d.kv) +
                   (((page * d.num_layers + layer) * 2 * d.num_kv_heads + plane) * d.page_size +
                    off) * row_bytes + e * 16;
        };
        for (int i = 0; i < moves; i += kAhead) {
            uint4 v[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (i + k < moves && s_src[i + k] >= 0)
                    v[k] = *reinterpret_cast<const uint4 *>(at(s_src[i + k]));
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (i + k < moves && s_src[i + k] >= 0)
                    *reinterpret_cast<uint4 *>(at(s_dst[i + k])) = v[k];
        }
    }
}

// -------------------------------------------------------------------- cutting
// scratch: the slots' marks, then per request give's prefix, pages kept and given.
struct TokCut {
    pk_token_kv_desc d;
    const int32_t *slots, *lengths;
    int batch, ps_shift;
};
template <int NK>
__device__ void cut_plan(const TokCut &p) {
    __shared__ int64_t s_scan[33];
    const pk_token_kv_desc &d = p.d;
    int32_t *head = d.scratch + d.num_slots, *tmp = head + 16;
    const int free_n = *d.free_count;
    const int b0 = threadIdx.x * NK;
    int slot[NK], len[NK], have[NK], held[NK], give[NK];
    bool own[NK];
#pragma unroll
    for (int k = 0; k < NK; ++k) len[k] = b0 + k < p.batch ? p.lengths[b0 + k] : 0;
#pragma unroll
    for (int k = 0; k < NK; ++k) have[k] = held[k] = 0;
    own_slots<NK>(d, p.slots, p.batch, b0, slot, own, [&](int s, int k) {
        have[k] = d.lengths[s];
        held[k] = d.held[s];
    });
    int64_t sum = 0, total;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
        const int b = b0 + k;
        give[k] = 0;
        if (b >= p.batch) continue;
        int keep = 0;
        if (!own[k]) {
            raise(d.error, PK_DEV_BAD_SLOT);
        } else if (len[k] < 0 || len[k] > have[k]) {
            raise(d.error, PK_DEV_BAD_COUNT);
        } else {
            keep = min(ceil_shift(len[k], p.ps_shift), held[k]);
            give[k] = held[k] - keep;
            d.held[slot[k]] = keep;
            d.lengths[slot[k]] = len[k];
        }
        tmp[3 * b + 1] = keep;
        tmp[3 * b + 2] = give[k];
        sum += give[k];
    }
    int64_t first = block_exclusive_sum64(sum, total, s_scan);
#pragma unroll
    for (int k = 0; k < NK; ++k) {
        if (b0 + k < p.batch) tmp[3 * (b0 + k)] = (int)first;
        first += give[k];
    }
    if (threadIdx.x == 0) {
        head[0] = free_n + (int)total;
        *d.free_count = free_n + (int)total;
    }
}
__device__ void cut_fill(const TokCut &p, int w, int nw) {
    const pk_token_kv_desc &d = p.d;
    const int32_t *head = d.scratch + d.num_slots, *tmp = head + 16;
    const int top = head[0], lane = threadIdx.x & 31;
    for (int b = w; b < p.batch; b += nw) {
        const int first = tmp[3 * b], keep = tmp[3 * b + 1], give = tmp[3 * b + 2];
        if (!give) continue;
        int32_t *row = d.page_table + (int64_t)p.slots[b] * d.table_width + keep;
        for (int i = lane; i < give; i += 32) {
            d.free_pages[top - 1 - (first + i)] = row[i];
            row[i] = -1;
        }
    }
}
template <int NK, bool kFill>
__global__ void __launch_bounds__(kPlanThreads) token_cut_kernel(const TokCut p) {
    grid_dep_wait();
    grid_dep_launch();
    cut_plan<NK>(p);
    if (kFill) {
        __syncthreads();
        cut_fill(p, threadIdx.x >> 5, blockDim.x >> 5);
    }
}
__global__ void __launch_bounds__(256) token_cut_fill_kernel(const TokCut p) {
    grid_dep_wait();
    grid_dep_launch();
    cut_fill(p, (blockIdx.x * blockDim.x + threadIdx.x) >> 5, (gridDim.x * blockDim.x) >> 5);
}

// Threads of the planning CTA for a batch at NK requests each.
int plan_threads(int batch, int nk) {
    const int n = ((batch + nk - 1) / nk + 31) / 32 * 32;
    return n < kPlanThreads ? n : kPlanThreads;
}

int grid_for(int64_t threads, int block) {
    const int64_t n = (threads + block - 1) / block, most = (int64_t)current_sms() * (2048 / block);
    return (int)(n < 1 ? 1 : (n < most ? n : most));
}

}  // namespace

int current_sms() {
    static std::atomic<int> sms[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    int n = sms[dev & 63].load(std::memory_order_relaxed);
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
        sms[dev & 63].store(n, std::memory_order_relaxed);
    }
    return n;
}

int launch_token_reset(const pk_token_kv *kv, const int32_t *init_order, cudaStream_t s) {
    const pk_token_kv_desc &d = kv->d;
    const int64_t n = (int64_t)d.num_slots * d.table_width;
    return cuda_status(launch_pdl(token_reset_kernel,
                                  dim3(grid_for(n > d.num_pages ? n : d.num_pages, 256)), dim3(256),
                                  0, s, d, init_order),
                       "token_reset_kernel");
}

int launch_token_begin(const pk_token_kv *kv, const int32_t *slots, const int32_t *counts,
                       int batch, const int32_t *parents, int rows, int32_t *step,
                       cudaStream_t s) {
    TokParams p = {};
    p.d = kv->d;
    p.l = tok_layout(kv, batch, rows, parents != nullptr);
    p.ps_shift = kv->ps_shift;
    p.group = kv->group;
    p.shape = tok_shape(kv, batch, rows);
    p.kv_heads = kv->d.num_kv_heads;
    while ((1 << p.row_shift) < p.shape.rows) ++p.row_shift;
    while ((1 << p.key_shift) < p.shape.keys) ++p.key_shift;
    p.batch = batch;
    p.rows = rows;
    p.slots = slots;
    p.counts = counts;
    p.parents = parents;
    p.step = step;
    const size_t marks = mark_bytes(kv->d.num_slots);
    if (batch <= 64 && rows <= kOneCtaRows)
        return cuda_status(launch_pdl(token_begin_kernel<1, true>, dim3(1), dim3(kPlanThreads), marks, s, p),
                           "token_begin_kernel");
    // requests a thread: the fewest of 1, 2, 8 and 64 that the batch needs
    cudaError_t e =
        batch <= kPlanThreads
            ? launch_pdl(token_begin_kernel<1, false>, dim3(1), dim3(plan_threads(batch, 1)), marks, s, p)
        : batch <= 2 * kPlanThreads
            ? launch_pdl(token_begin_kernel<2, false>, dim3(1), dim3(plan_threads(batch, 2)), marks, s, p)
        : batch <= 8 * kPlanThreads
            ? launch_pdl(token_begin_kernel<8, false>, dim3(1), dim3(plan_threads(batch, 8)), marks, s, p)
            : launch_pdl(token_begin_kernel<64, false>, dim3(1), dim3(plan_threads(batch, 64)), marks, s, p);
    if (e != cudaSuccess) return cuda_status(e, "token_begin_kernel");
    const int64_t warps = parents ? (int64_t)batch : ((int64_t)rows + 31) / 32;
    return cuda_status(launch_pdl(token_fill_kernel,
                                  dim3(grid_for((warps > batch ? warps : batch) * 32, 256)),
                                  dim3(256), 0, s, p),
                       "token_fill_kernel");
}

int launch_token_append(const pk_token_kv *kv, const TokAppendArgs &a, cudaStream_t s) {
    const pk_token_kv_desc &d = kv->d;
    const TokLayout l = tok_layout(kv, a.batch, a.rows, a.trees);
    const int64_t n = (int64_t)a.rows * d.num_kv_heads * d.head_dim * kv->esize / 16;
    return cuda_status(launch_pdl(token_append_kernel, dim3(grid_for(n, 256), a.nlayers), dim3(256),
                                  0, s, d, a, l.slot_map, kv->ps_shift, kv->esize),
                       "token_append_kernel");
}

int launch_token_end(const pk_token_kv *kv, const int32_t *last, int batch, int rows, int trees,
                     const int32_t *step, cudaStream_t s) {
    const pk_token_kv_desc &d = kv->d;
    return cuda_status(launch_pdl(token_end_kernel, dim3(batch, trees ? d.num_layers : 1), dim3(256),
                                  0, s, d, tok_layout(kv, batch, rows, trees), last, trees, step,
                                  kv->ps_shift, kv->esize),
                       "token_end_kernel");
}

int launch_token_truncate(const pk_token_kv *kv, const int32_t *slots, const int32_t *lengths,
                          int batch, cudaStream_t s) {
    TokCut p;
    p.d = kv->d;
    p.slots = slots;
    p.lengths = lengths;
    p.batch = batch;
    p.ps_shift = kv->ps_shift;
    const size_t marks = mark_bytes(kv->d.num_slots);
    if (batch <= 64 && (int64_t)batch * kv->d.table_width <= 2 * kOneCtaRows)
        return cuda_status(launch_pdl(token_cut_kernel<1, true>, dim3(1), dim3(kPlanThreads), marks, s, p),
                           "token_cut_kernel");
    cudaError_t e =
        batch <= kPlanThreads
            ? launch_pdl(token_cut_kernel<1, false>, dim3(1), dim3(plan_threads(batch, 1)), marks, s, p)
        : batch <= 2 * kPlanThreads
            ? launch_pdl(token_cut_kernel<2, false>, dim3(1), dim3(plan_threads(batch, 2)), marks, s, p)
        : batch <= 8 * kPlanThreads
            ? launch_pdl(token_cut_kernel<8, false>, dim3(1), dim3(plan_threads(batch, 8)), marks, s, p)
            : launch_pdl(token_cut_kernel<64, false>, dim3(1), dim3(plan_threads(batch, 64)), marks, s, p);
    if (e != cudaSuccess) return cuda_status(e, "token_cut_kernel");
    return cuda_status(launch_pdl(token_cut_fill_kernel, dim3(grid_for((int64_t)batch * 32, 256)),
                                  dim3(256), 0, s, p),
                       "token_cut_fill_kernel");
}

}  // namespace pk
