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
// Bounded wait that gives up at once when another wait of the CTA already has.
__device__ __forceinline__ void ring_wait(uint64_t *bar, uint32_t parity, volatile int *failed,
                                          int32_t *error) {
    if (mbar_try_wait(bar, parity)) return;
    if (*failed) return;
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (*failed) return;
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
            *failed = 1;
            raise(error, PK_DEV_TIMEOUT);
            return;
        }
    }
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
    int cta, b, nr, kt;
    int64_t at, end, base, next_base;
    bool whole;
    Unit u;

    __device__ __forceinline__ Work(const TreeParams &params, int c) : p(params), cta(c) {
        b = p.step[p.l.first + c];
        const int64_t share = p.step[kTokShare];
        whole = share == 0;
        at = whole ? c : c * share;
        end = b < 0 ? at : at + (whole ? 1 : share);
        if (b >= 0) load();
    }
    __device__ __forceinline__ void load() {
        const int64_t *work = reinterpret_cast<const int64_t *>(p.step + p.l.work);
        base = work[b];
        next_base = work[b + 1];
        u.ctx = p.step[p.l.context + b];
        u.slot = p.step[p.l.slot + b];
        u.row0 = p.step[p.l.row_start + b];
        u.count = p.step[p.l.row_start + b + 1] - u.row0;
        nr = (int)(((int64_t)u.count * p.group + p.shape.rows - 1) / p.shape.rows);
        kt = (u.ctx + u.count + p.shape.keys - 1) / p.shape.keys;
    }
    __device__ __forceinline__ bool next() {
        if (at >= end) return false;
        while (at >= next_base) {   // requests without work have no tiles
            if (++b >= p.batch) return false;
            load();
        }
        const int64_t local = at - base;
        int item;
        if (whole) {
            item = (int)local;
            u.t0 = 0;
            u.t1 = kt;
            u.part = -1;
            ++at;
        } else {
            item = (int)(local / kt);
            u.t0 = (int)(local - (int64_t)item * kt);
            const int n = (int)min((int64_t)(kt - u.t0), end - at);
            u.t1 = u.t0 + n;
            u.part = n == kt ? -1 : (u.t0 == 0 ? 2 * cta + 1 : 2 * cta);
            at += n;
        }
        u.head = item / nr;
        u.rt = item - u.head * nr;
        if (!p.trees) {   // a chain's rows see no key past their own
            const int64_t last = ((int64_t)(u.rt + 1) * p.shape.rows + p.group - 1) / p.group;
            const int seen = u.ctx + (int)min(last, (int64_t)u.count);
            u.t1 = min(u.t1, (seen + p.shape.keys - 1) / p.shape.keys);
        }
        return true;
    }
};

}  // namespace
}  // namespace pk
