// Internal interfaces between the C-ABI layer (pk_api.cu) and the kernel
// translation units.  Nothing here is exported.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "pk.h"

struct pk_paged_kv {
    pk_paged_kv_desc d;
    CUtensorMap kv_map;  // 3-D view {dim, page_size, pages*layers*2}, 128B-swizzled boxes
    int head_dim;
    int esize;
};

namespace pk {

void set_error(const char *fmt, ...);
int cuda_status(cudaError_t e, const char *what);
// pk_selftest.cu: one CTA waits on an mbarrier with the shared bounded wait
int launch_selftest_wait(int32_t *error, int32_t arrive, uint64_t limit_ns, int64_t *waited_ns,
                         cudaStream_t stream);
// Encode a tiled TMA descriptor (driver entry point fetched once via cudart).
int encode_tmap(CUtensorMap *map, int dtype, const void *base, int rank, const uint64_t *dims,
                const uint64_t *strides_bytes, const uint32_t *box);
int encode_tmap_3d(CUtensorMap *map, int dtype, const void *base, uint64_t d0, uint64_t d1,
                   uint64_t d2, uint64_t stride1_bytes, uint64_t stride2_bytes, uint32_t box0,
                   uint32_t box1, uint32_t box2);

// Launch with programmatic stream serialization: the kernel may be scheduled
// while the previous kernel of the stream finishes, and must call
// grid_dep_wait() before it reads anything that kernel could have written.
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                       cudaStream_t s, Args &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Args &&>(args)...);
}

// pk_pages.cu
int launch_pages_reset(const pk_paged_kv *kv, const int32_t *init_order, cudaStream_t s);
int launch_pages_begin(const pk_paged_kv *kv, const int32_t *slots, const int32_t *lengths,
                       int batch, const int32_t *released, int num_released, cudaStream_t s);
int launch_pages_end(const pk_paged_kv *kv, const int32_t *slots, const int32_t *lengths,
                     int batch, cudaStream_t s);


// pk_kv.cu
int launch_append(const pk_paged_kv *kv, int layer0, int nlayers, const void *key,
                  const void *value, int64_t ls, int64_t bs, int64_t rs, const int32_t *slots,
                  int batch, cudaStream_t s);
int launch_gather(const pk_paged_kv *kv, int layer0, int nlayers, const int32_t *slots, int batch,
                  void *k_out, void *v_out, int64_t out_layer_stride, cudaStream_t s);

// pk_attn.cu
struct AttnArgs {
    const void *q;
    int64_t q_ls, q_bs, q_rs;
    const void *k_new, *v_new;   // optional: this step's K/V rows (q's strides) to append
    const void *bias_u, *bias_v;
    int64_t bias_ls;
    const void *pos;             // pos_proj rows (l, p, c) at l * pos_ls + p * dim + c
    int64_t pos_ls;
    int pos_rows;                // 2 * (left + chunk) - 1
    const float *bd;             // optional: rel-pos term from launch_relpos_bd (replaces pos)
    const int32_t *slots, *lengths;
    int batch;
    void *out;
    int64_t o_ls, o_bs, o_rs;
    int layer0, nlayers;
};
int launch_attention(const pk_paged_kv *kv, const CUtensorMap &pos_map, const AttnArgs &a,
                     cudaStream_t s);
// pk_attn_bf16.cu
int launch_attention_bf16(const pk_paged_kv *kv, const CUtensorMap &pos_map, const AttnArgs &a,
                          cudaStream_t s);
// pk_attn_stacked.cu: all heads of a (stream, layer) per CTA, when heads * chunk <= 16;
// returns PK_ENOTSUP for other shapes.  pos_map16 has 16-row boxes.
int launch_attention_stacked(const pk_paged_kv *kv, const CUtensorMap &pos_map16,
                             const AttnArgs &a, cudaStream_t s);
// pk_attn_stacked.cu: the rel-pos term of every (layer, stream, head, query) of a
// step, bd[l][b][h][t][relpos_bd_cols], for the shapes launch_attention_stacked
// handles (PK_ENOTSUP otherwise); reads a.q, a.bias_v, a.pos.
int relpos_bd_cols(const pk_paged_kv *kv);
int launch_relpos_bd(const pk_paged_kv *kv, const AttnArgs &a, float *bd, cudaStream_t s);
// pk_pages.cu: launch_pages_begin and launch_relpos_bd in one launch (batch <= 256,
// shapes with the pre-pass; PK_ENOTSUP otherwise)
int launch_pages_begin_relpos(const pk_paged_kv *kv, const int32_t *slots,
                              const int32_t *lengths, int batch, const int32_t *released,
                              int num_released, const AttnArgs &a, float *bd, cudaStream_t s);
// pk_attn_heads.cu: head_dim 128, chunks of 8..16 frames, K/V appended before;
// returns PK_ENOTSUP for other shapes.  pos_map16 has 16-row boxes of 64 columns.
int launch_attention_heads(const pk_paged_kv *kv, const CUtensorMap &pos_map16,
                           const AttnArgs &a, cudaStream_t s);

// pk_conv.cu
struct ConvArgs {
    void *state;
    int num_slots, num_layers, layer, dim, kernel, chunk, dtype;
    const void *x;
    int64_t x_bs, x_rs;
    const void *w, *ln_w, *ln_b;
    float eps;
    const int32_t *slots, *lengths;
    int batch;
    void *y;
    int32_t *error;
    int x_vec;   // x rows 16-byte aligned (base, row and batch strides): vector staging
};
int launch_conv(const ConvArgs &a, cudaStream_t s);

// pk_pre_encode.cu
int launch_pre_encode_window(void *cache, const void *feats, const int32_t *slots, int batch,
                             int feat_in, int frames, int csize, int prefix, void *out,
                             int dtype, int32_t *error, int num_slots, cudaStream_t s);

// pk_rnnt.cu
int launch_rnnt_pick(const void *logits, int64_t ld, int dtype, int batch, int nclass, int blank,
                     const int32_t *lengths, int frame, int symbol, int max_symbols, int frames,
                     int32_t *done, int32_t *emit, int64_t *ids, int32_t *tokens, int32_t *counts,
                     cudaStream_t s);
int launch_lstm_cell(const void *gates, int64_t gld, const void *xtab, int64_t xld,
                     const int64_t *ids, void *h, void *c, int64_t sld, const int32_t *emit,
                     int batch, int hidden, int dtype, cudaStream_t s);

// pk_norm.cu
struct LnArgs {
    const void *x;
    int64_t x_ld;
    int rows, dim, dtype;
    const void *g1, *b1;
    float eps1;
    void *y1;
    int64_t y1_ld;
    const void *g2, *b2;   // optional second LayerNorm of y1 (g2 == nullptr: none)
    float eps2;
    void *y2;
    int64_t y2_ld;
};
int launch_layer_norm(const LnArgs &a, cudaStream_t s);

// pk_gemm.cu
struct GemmArgs {
    const void *A, *W;
    int64_t lda, ldw;
    int M, N, K, epilogue;
    void *C;
    int64_t ldc;
    const void *R;
    int64_t ldr;
    const void *bias;
    float alpha;
    int32_t *error;
};
int launch_gemm(const GemmArgs &g, cudaStream_t s);

// pk_subsample.cu
struct SubsampleArgs {
    const void *x;
    int64_t xb, xf, xt;      // stage12: x[b][f][t] strides (elements)
    int batch, frames, feat, channels, dtype;
    const void *w1, *b1, *w2, *b2;   // dw: w2 / b2 are the depthwise conv's
    int first, first_out;
    void *y;
};
int launch_subsample_stage12(const SubsampleArgs &a, cudaStream_t s);
int launch_subsample_dw(const SubsampleArgs &a, cudaStream_t s);

// pk_features.cu.  Table block: int32 header[kFeHeader], then float2
// twiddle[n_fft] (exp(-2 pi i u / n_fft)), float window[n_fft], int32 lo[n_mels],
// cnt[n_mels], off[n_mels] (first bin, length and offset of each filter's
// nonzero run), float weight[nnz].
constexpr int kFeHeader = 16;
enum FeHeaderField { kFeMagic = 0, kFeNfft, kFeNmels, kFeNnz, kFeWin, kFeRate };
constexpr int32_t kFeMagicValue = 0x45464b50;  // "PKFE"
int build_feature_tables(int sample_rate, int n_fft, int win_length, int n_mels, double fmin,
                         double fmax, int norm, int32_t *words, int64_t *nwords, int32_t *nnz);
struct FeArgs {
    const int32_t *tables;
    float *hist;
    int64_t *meta;
    int32_t *error;
    int num_slots, hop, n_mels, nnz;
    float preemph, dither, mag_power, guard, pad;
    uint32_t seed_lo, seed_hi;
    const float *samples;
    int64_t ld;
    const int32_t *nsamp, *flags, *slots;
    int batch;
    void *out;
    int out_dtype, max_frames;
    int32_t *nframes;
};
int launch_features(const FeArgs &a, cudaStream_t s);

// pk_tokens.cu / pk_tree_attn.cu: token pools
}  // namespace pk

struct pk_token_kv {
    pk_token_kv_desc d;
    CUtensorMap kv_map;  // bf16 pools: {64, 8, head_dim / 64, page_size / 8, pages*layers*2*
                         // kv_heads}, boxes of min(page_size, kTokRowsBox) rows, 128B-swizzled
    int ps_shift, esize, group;
    int sms;
};

namespace pk {

// How a step's rows are attended.  A row tile is up to `rows` query rows (token x
// group) of one request and K/V head, a key tile `keys` of its keys; `ctas` workers
// (CTAs, or warps) share the work.
struct TokShape {
    int rows, keys;
    int ctas;    // workers: CTAs, or warps of the 16-row bf16 kernel
    int least;   // key tiles that a worker takes before a request's are split over several
    int lead;    // what beginning a row tile costs, in key tiles
    // so many row tiles of so many key tiles at most: a CTA each, its warps sharing it (24
    // requests of up to 553 tokens, 4 heads of 128: 27 us in shares, 11 so)
    int team, team_keys;
    // workers that get a share of their own before shares grow from two key tiles to
    // `least` (two requests of up to 5908 tokens, one head of 128: 24 us at 8 tiles, 14 at
    // two; 160 of up to 500, 8 heads of 64: 27 at 8, 34 at 4)
    int busy;
};
// Most rows of a page that one TMA copy brings, and keys of a tile of the 16-row
// kernel; its workers an SM, with two tiles of shared memory each (8 KB, or 16 for
// 128-wide heads).
constexpr int kTokRowsBox = 64;
constexpr int tok_workers(int head_dim) { return head_dim == 64 ? 12 : 6; }
constexpr int tok_warps(int head_dim) { return head_dim == 64 ? 4 : 6; }   // of a CTA
// bf16: row tiles of 16 by mma.sync, a warp a worker, where they hold an average
// request (its K/V is read once per row tile); of 128 by tcgen05, two workers a CTA,
// otherwise (160 requests of 21 rows, 8 heads of 64: 500 tokens 54 us by the former, 64
// by the latter, 2000 tokens 138 and 128; one request of 24 rows and 20,000 tokens 30
// and 23; 32 x 8 heads of 128 with 28 rows, 8000 tokens 203 and 113; the lengths, which
// also tell them apart, are known on the device only).  float32: 16.
inline TokShape tok_shape(const pk_token_kv *kv, int batch, int rows) {
    const int64_t mean = ((int64_t)rows + batch - 1) / (batch > 0 ? batch : 1) * kv->group;
    if (kv->d.dtype == PK_DTYPE_F32) return {16, 64, (kv->d.head_dim == 64 ? 3 : 2) * kv->sms, 1, 1, 0, 0, 1};
    if (mean <= 16) {
        const int workers = tok_workers(kv->d.head_dim), warps = tok_warps(kv->d.head_dim);
        return {16, kTokRowsBox, workers * kv->sms, 8, 1, workers / warps * kv->sms, 4 * warps, 4 * kv->sms};
    }
    return {128, 64, 2 * kv->sms, 6, 4, 0, 0, 2 * kv->sms};   // a row tile's ends: 5 to 7 us, four tiles
}

// Step block, int32 words: header, then arrays at these offsets.  The step's work
// is a line of key tiles, request by request, K/V head by head, row tile by row
// tile; worker c takes tiles [c * share, (c + 1) * share), whatever they belong to, so
// that every worker has the same number however the lengths are spread (share 0: kTokPer
// whole row tiles each).
enum TokHeader { kTokShare = 0, kTokRows, kTokFree, kTokPer, kTokHeaderWords = 16 };
struct TokLayout {
    // work: int64 first place (share 0: row tile) of each request; first: the request
    // that each worker begins in (-1: no work); take: first new page; held: pages before
    int64_t row_start, context, slot, work, first, take, held, request, position, slot_map, mask,
        words;
};
inline TokLayout tok_layout(const pk_token_kv *kv, int batch, int rows, int trees) {
    TokLayout l;
    int64_t o = kTokHeaderWords;
    auto take = [&](int64_t n) {
        const int64_t at = o;
        o += n;
        return at;
    };
    l.work = take(2 * ((int64_t)batch + 1));
    l.mask = take(trees ? 2 * (int64_t)rows : 0);
    l.row_start = take(batch + 1);
    l.context = take(batch);
    l.slot = take(batch);
    l.first = take(tok_workers(64) * kv->sms);
    l.take = take(batch + 1);
    l.held = take(batch);
    l.request = take(rows);
    l.position = take(rows);
    l.slot_map = take(rows);
    l.words = o;
    return l;
}
int launch_token_reset(const pk_token_kv *kv, const int32_t *init_order, cudaStream_t s);
int launch_token_begin(const pk_token_kv *kv, const int32_t *slots, const int32_t *counts,
                       int batch, const int32_t *parents, int rows, int32_t *step, cudaStream_t s);
struct TokAppendArgs {
    const void *key, *value;
    int64_t ls, rs, hs;
    int layer0, nlayers, batch, rows, trees;
    const int32_t *step;
};
int launch_token_append(const pk_token_kv *kv, const TokAppendArgs &a, cudaStream_t s);
int launch_token_end(const pk_token_kv *kv, const int32_t *last, int batch, int rows, int trees,
                     const int32_t *step, cudaStream_t s);
int launch_token_truncate(const pk_token_kv *kv, const int32_t *slots, const int32_t *lengths,
                          int batch, cudaStream_t s);
struct TreeAttnArgs {
    const void *q;
    int64_t q_rs, q_hs, o_rs, o_hs;
    void *out;
    float scale;
    int layer, batch, rows, trees;
    const int32_t *step;
    float *ws;
};
struct TreeParams {
    const int32_t *step, *table;
    TokLayout l;
    TokShape shape;
    int table_width, num_pages, num_layers, layer, kv_heads, group, ps_shift, trees;
    int batch, rows, heads;
    const void *q, *kv;
    void *out;
    int64_t q_rs, q_hs, o_rs, o_hs;
    float scale_log2;
    // partial results of row tiles that CTAs share, two a CTA: outputs [part][row][dim],
    // (maximum, sum) pairs
    float *ws_o, *ws_ml;
    int32_t *error;
};
// pk_tree_attn_tc.cu: row tiles of 128
cudaError_t launch_tree_tc(const pk_token_kv *kv, const TreeParams &p, int workers, cudaStream_t s);
int64_t tree_attn_workspace(const pk_token_kv *kv, int batch, int rows);
int launch_tree_attention(const pk_token_kv *kv, const TreeAttnArgs &a, cudaStream_t s);

// pk_adapter.cu: plan block, int32 words
constexpr int kPairWords = 8;
struct AdapterLayout {
    int64_t tile_pair, order, sorted, pairs, words;
};
inline AdapterLayout adapter_layout(int rows, int adapters) {
    AdapterLayout l;
    const int64_t tiles = ((int64_t)rows + 127) / 128;
    l.order = 0;                         // sorted row -> row; `rows` past the last
    l.tile_pair = l.order + tiles * 128; // first pair of each tile
    l.sorted = l.tile_pair + tiles + 1;  // 1: the rows' own order is sorted
    l.pairs = (l.sorted + 1 + 3) / 4 * 4;   // adapter, 128 bits: its rows of the tile
    l.words = l.pairs + kPairWords * (tiles + (adapters < rows ? adapters : rows));
    return l;
}
struct AdapterArgs {
    const void *x, *W, *R, *bias, *down, *up;
    int64_t ldx, ldw, ldc, ldr;
    void *C, *s, *xs;   // output; S and the rows' copy, sorted and padded to 128
    int M, N, K, epilogue, rank, adapters;
    int box_rows;       // rows of a TMA copy of x, its sorted copy and S
    float alpha;
    const float *scale;
    const int32_t *plan;
    int32_t *error;
    AdapterLayout l;
};
int launch_adapter_plan(const int32_t *ids, int rows, int adapters, int32_t *plan, int32_t *error,
                        cudaStream_t s);
int launch_adapter_gemm(const AdapterArgs &a, cudaStream_t s);

// Allow `bytes` of dynamic shared memory for `kernel` on the current device, once
// per device (`done`: a bit per device, of the kernel's own).
template <typename K>
cudaError_t allow_smem(K kernel, size_t bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}
int current_sms();   // multiprocessors of the current device

}  // namespace pk
