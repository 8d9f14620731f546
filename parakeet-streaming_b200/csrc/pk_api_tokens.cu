// C-ABI entry points of the token pools and the adapters (include/pk.h): argument
// checks on the host, the pool's TMA descriptor, dispatch.
#include <math.h>
#include <stdlib.h>

#include "pk_internal.h"

using namespace pk;

#define PK_CHECK(cond, ...)             \
    do {                                \
        if (!(cond)) {                  \
            pk::set_error(__VA_ARGS__); \
            return PK_EINVAL;           \
        }                               \
    } while (0)

static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What every call on a step block needs.
#define PK_CHECK_STEP(kv, batch, rows, step)                                                   \
    PK_CHECK(kv, "null pool");                                                                 \
    PK_CHECK((batch) >= 0 && (batch) <= PK_TOK_MAX_BATCH && (batch) <= (kv)->d.num_slots,       \
             "batch %d outside [0, min(num_slots, %d)]", (batch), PK_TOK_MAX_BATCH);           \
    PK_CHECK((rows) >= 0 && (int64_t)(rows) * (kv)->d.num_heads <= 0x7fffffff,                 \
             "rows %d: negative or too many", (rows));                                         \
    PK_CHECK((batch) == 0 || ((step) && aligned16(step)), "step block null or not 16-byte aligned")

extern "C" {

int pk_token_kv_create(const pk_token_kv_desc *desc, pk_token_kv **out) {
    PK_CHECK(desc && out, "null argument");
    const pk_token_kv_desc &d = *desc;
    PK_CHECK(d.kv && d.page_table && d.free_pages && d.free_count && d.lengths && d.held &&
                 d.scratch && d.error,
             "null device buffer in descriptor");
    PK_CHECK(d.dtype == PK_DTYPE_F32 || d.dtype == PK_DTYPE_BF16, "bad dtype %d", d.dtype);
    PK_CHECK(d.num_pages > 0 && d.num_slots > 0 && d.num_layers > 0 && d.table_width > 0,
             "empty pool");
    PK_CHECK(d.num_kv_heads > 0 && d.num_heads > 0 && d.num_heads % d.num_kv_heads == 0,
             "num_heads (%d) must be a multiple of num_kv_heads (%d)", d.num_heads, d.num_kv_heads);
    PK_CHECK(d.head_dim == 64 || d.head_dim == 128, "head_dim %d: 64 or 128", d.head_dim);
    PK_CHECK(d.page_size >= 8 && d.page_size <= 256 && (d.page_size & (d.page_size - 1)) == 0,
             "page_size must be a power of two in [8, 256]");
    PK_CHECK((int64_t)d.num_pages * d.page_size <= 0x7fffffff &&
                 (int64_t)d.table_width * d.page_size <= 0x7fffffff - 65536,
             "more tokens than 32 bits count");
    const int64_t planes = (int64_t)d.num_pages * d.num_layers * 2 * d.num_kv_heads;
    PK_CHECK(planes <= 0x7fffffff, "more (page, layer, head) planes than 32 bits count");
    PK_CHECK(aligned16(d.kv), "kv pool not 16-byte aligned");
    pk_token_kv *kv = static_cast<pk_token_kv *>(calloc(1, sizeof(pk_token_kv)));
    PK_CHECK(kv, "out of host memory");
    kv->d = d;
    kv->esize = d.dtype == PK_DTYPE_BF16 ? 2 : 4;
    kv->group = d.num_heads / d.num_kv_heads;
    while ((1 << kv->ps_shift) < d.page_size) ++kv->ps_shift;
    kv->sms = current_sms();
    if (d.dtype == PK_DTYPE_BF16) {
        // a page's rows of one head in one copy, laid out in groups of 8 rows of 128
        // bytes (a swizzle atom), the 64-column blocks of a group beside each other
        const uint64_t row = (uint64_t)d.head_dim * 2, blocks = d.head_dim / 64;
        const uint64_t dims[5] = {64, 8, blocks, (uint64_t)d.page_size / 8, (uint64_t)planes};
        const uint64_t strides[4] = {row, 128, 8 * row, row * d.page_size};
        const uint32_t groups = (d.page_size < kTokRowsBox ? d.page_size : kTokRowsBox) / 8;
        const uint32_t box[5] = {64, 8, (uint32_t)blocks, groups, 1};
        int st = encode_tmap(&kv->kv_map, d.dtype, d.kv, 5, dims, strides, box);
        if (st != PK_OK) {
            free(kv);
            return st;
        }
    }
    *out = kv;
    return PK_OK;
}

int pk_token_kv_destroy(pk_token_kv *kv) {
    free(kv);
    return PK_OK;
}

int pk_token_reset(pk_token_kv *kv, const int32_t *init_order, void *stream) {
    PK_CHECK(kv, "null pool");
    return launch_token_reset(kv, init_order, static_cast<cudaStream_t>(stream));
}

int64_t pk_token_step_words(const pk_token_kv *kv, int32_t batch, int32_t rows, int32_t trees,
                            int64_t *offsets) {
    if (!kv || batch < 0 || rows < 0) return -1;
    const TokLayout l = tok_layout(kv, batch, rows, trees);
    if (offsets) {
        offsets[PK_TOK_ROW_START] = l.row_start;
        offsets[PK_TOK_CONTEXT] = l.context;
        offsets[PK_TOK_REQUEST] = l.request;
        offsets[PK_TOK_POSITION] = l.position;
        offsets[PK_TOK_SLOT_MAP] = l.slot_map;
        offsets[PK_TOK_MASK] = l.mask;
    }
    return l.words;
}

int pk_token_begin_step(pk_token_kv *kv, const int32_t *slots, const int32_t *counts,
                        int32_t batch, const int32_t *parents, int32_t rows, int32_t *step,
                        void *stream) {
    PK_CHECK_STEP(kv, batch, rows, step);
    if (batch == 0) return PK_OK;
    PK_CHECK(slots && counts, "null slots/counts");
    return launch_token_begin(kv, slots, counts, batch, parents, rows, step,
                              static_cast<cudaStream_t>(stream));
}

int pk_token_append(pk_token_kv *kv, int32_t layer0, int32_t num_layers, const void *key,
                    const void *value, int64_t layer_stride, int64_t row_stride,
                    int64_t head_stride, int32_t batch, int32_t rows, int32_t trees,
                    const int32_t *step, void *stream) {
    PK_CHECK_STEP(kv, batch, rows, step);
    PK_CHECK(layer0 >= 0 && num_layers >= 0 && num_layers <= kv->d.num_layers - layer0,
             "layers [%d, +%d) outside [0, %d)", layer0, num_layers, kv->d.num_layers);
    PK_CHECK(num_layers <= 65535, "more than 65535 layers in one call");
    if (batch == 0 || rows == 0 || num_layers == 0) return PK_OK;
    PK_CHECK(key && value && aligned16(key) && aligned16(value),
             "key/value null or not 16-byte aligned");
    const int es = kv->esize;
    PK_CHECK((layer_stride * es) % 16 == 0 && (row_stride * es) % 16 == 0 &&
                 (head_stride * es) % 16 == 0,
             "strides must be multiples of 16 bytes");
    TokAppendArgs a;
    a.key = key;
    a.value = value;
    a.ls = layer_stride;
    a.rs = row_stride;
    a.hs = head_stride;
    a.layer0 = layer0;
    a.nlayers = num_layers;
    a.batch = batch;
    a.rows = rows;
    a.trees = trees;
    a.step = step;
    return launch_token_append(kv, a, static_cast<cudaStream_t>(stream));
}

int64_t pk_token_attention_workspace(const pk_token_kv *kv, int32_t batch, int32_t rows) {
    return kv && batch >= 0 && rows >= 0 ? tree_attn_workspace(kv, batch, rows) : -1;
}

int pk_token_attention(pk_token_kv *kv, int32_t layer, const void *query, int64_t q_row_stride,
                       int64_t q_head_stride, float scale, int32_t batch, int32_t rows,
                       int32_t trees, const int32_t *step, void *out, int64_t o_row_stride,
                       int64_t o_head_stride, void *workspace, void *stream) {
    PK_CHECK_STEP(kv, batch, rows, step);
    PK_CHECK(layer >= 0 && layer < kv->d.num_layers, "layer out of range");
    PK_CHECK(scale > 0.f && isfinite(scale), "scale must be positive and finite");
    if (batch == 0 || rows == 0) return PK_OK;
    PK_CHECK(query && out && aligned16(query) && aligned16(out),
             "query/out null or not 16-byte aligned");
    const int es = kv->esize;
    PK_CHECK((q_row_stride * es) % 16 == 0 && (q_head_stride * es) % 16 == 0 &&
                 (o_row_stride * es) % 16 == 0 && (o_head_stride * es) % 16 == 0,
             "strides must be multiples of 16 bytes");
    PK_CHECK((workspace && aligned16(workspace)) || tree_attn_workspace(kv, batch, rows) == 0,
             "workspace null or not 16-byte aligned");
    TreeAttnArgs a;
    a.q = query;
    a.q_rs = q_row_stride;
    a.q_hs = q_head_stride;
    a.out = out;
    a.o_rs = o_row_stride;
    a.o_hs = o_head_stride;
    a.scale = scale;
    a.layer = layer;
    a.batch = batch;
    a.rows = rows;
    a.trees = trees != 0;
    a.step = step;
    a.ws = static_cast<float *>(workspace);
    return launch_tree_attention(kv, a, static_cast<cudaStream_t>(stream));
}

int pk_token_end_step(pk_token_kv *kv, const int32_t *last, int32_t batch, int32_t rows,
                      int32_t trees, const int32_t *step, void *stream) {
    PK_CHECK_STEP(kv, batch, rows, step);
    if (batch == 0) return PK_OK;
    PK_CHECK(last, "null last");
    PK_CHECK(kv->d.num_layers <= 65535, "more than 65535 layers");
    return launch_token_end(kv, last, batch, rows, trees, step, static_cast<cudaStream_t>(stream));
}

int pk_token_truncate(pk_token_kv *kv, const int32_t *slots, const int32_t *lengths,
                      int32_t batch, void *stream) {
    PK_CHECK(kv, "null pool");
    PK_CHECK(batch >= 0 && batch <= kv->d.num_slots && batch <= PK_TOK_MAX_BATCH,
             "batch %d outside [0, min(num_slots, %d)]", batch, PK_TOK_MAX_BATCH);
    if (batch == 0) return PK_OK;
    PK_CHECK(slots && lengths, "null slots/lengths");
    return launch_token_truncate(kv, slots, lengths, batch, static_cast<cudaStream_t>(stream));
}

int64_t pk_adapter_plan_words(int32_t rows, int32_t num_adapters) {
    if (rows < 0 || rows > PK_ADAPTER_MAX_ROWS || num_adapters <= 0 || num_adapters > PK_ADAPTER_MAX)
        return -1;
    return adapter_layout(rows, num_adapters).words;
}

int pk_adapter_plan(const int32_t *ids, int32_t rows, int32_t num_adapters, int32_t *plan,
                    int32_t *error, void *stream) {
    PK_CHECK(rows >= 0 && rows <= PK_ADAPTER_MAX_ROWS, "rows %d outside [0, %d]", rows,
             PK_ADAPTER_MAX_ROWS);
    PK_CHECK(num_adapters > 0 && num_adapters <= PK_ADAPTER_MAX, "num_adapters %d outside [1, %d]",
             num_adapters, PK_ADAPTER_MAX);
    if (rows == 0) return PK_OK;
    PK_CHECK(ids && plan && error, "null pointer");
    PK_CHECK(aligned16(plan), "plan not 16-byte aligned");
    return launch_adapter_plan(ids, rows, num_adapters, plan, error,
                               static_cast<cudaStream_t>(stream));
}

int64_t pk_adapter_workspace(int32_t rows, int32_t K, int32_t rank) {
    if (rows < 0 || rows > PK_ADAPTER_MAX_ROWS || K <= 0 || rank <= 0 || rank > PK_ADAPTER_MAX_RANK)
        return -1;
    return ((int64_t)rows + 127) / 128 * 128 * ((int64_t)K + rank) * 2;
}

int pk_adapter_gemm(const void *A, int64_t lda, const void *W, int64_t ldw, int32_t M, int32_t N,
                    int32_t K, void *C, int64_t ldc, int32_t epilogue, const void *R, int64_t ldr,
                    const void *bias, float alpha, const void *down, const void *up, int32_t rank,
                    int32_t num_adapters, const float *scale, const int32_t *plan,
                    void *workspace, int32_t *error, void *stream) {
    PK_CHECK(M >= 0 && M <= PK_ADAPTER_MAX_ROWS && N > 0 && K > 0, "bad shape %d x %d x %d", M, N, K);
    PK_CHECK(num_adapters > 0 && num_adapters <= PK_ADAPTER_MAX, "num_adapters %d outside [1, %d]",
             num_adapters, PK_ADAPTER_MAX);
    PK_CHECK(rank > 0 && rank % 8 == 0 && rank <= PK_ADAPTER_MAX_RANK,
             "rank %d: a multiple of 8 up to %d", rank, PK_ADAPTER_MAX_RANK);
    if (M == 0) return PK_OK;
    PK_CHECK(K % 64 == 0 && N % 64 == 0, "K (%d) and N (%d) must be multiples of 64", K, N);
    PK_CHECK(epilogue >= PK_GEMM_STORE && epilogue <= PK_GEMM_BIAS, "bad epilogue %d", epilogue);
    PK_CHECK(A && W && C && down && up && plan && workspace && error, "null pointer");
    PK_CHECK(aligned16(A) && aligned16(W) && aligned16(C) && aligned16(down) && aligned16(up) &&
                 aligned16(plan) && aligned16(workspace),
             "operands must be 16-byte aligned");
    PK_CHECK(lda >= K && ldw >= K && ldc >= N && lda % 8 == 0 && ldw % 8 == 0 && ldc % 8 == 0,
             "row strides must cover the rows and be multiples of 8 elements");
    if (epilogue == PK_GEMM_RESIDUAL || epilogue == PK_GEMM_RESIDUAL_RELU)
        PK_CHECK(R && aligned16(R) && ldr >= N && ldr % 8 == 0, "bad residual operand");
    if (epilogue == PK_GEMM_BIAS) PK_CHECK(bias && aligned16(bias), "bad bias operand");
    AdapterArgs a;
    a.x = A;
    a.W = W;
    a.R = R;
    a.bias = bias;
    a.down = down;
    a.up = up;
    a.ldx = lda;
    a.ldw = ldw;
    a.ldc = ldc;
    a.ldr = ldr;
    a.C = C;
    a.xs = workspace;   // padded rows of K, then of rank
    a.s = static_cast<char *>(workspace) + ((int64_t)M + 127) / 128 * 128 * K * 2;
    a.M = M;
    a.N = N;
    a.K = K;
    a.epilogue = epilogue;
    a.rank = rank;
    a.adapters = num_adapters;
    a.alpha = alpha;
    a.scale = scale;
    a.plan = plan;
    a.error = error;
    return launch_adapter_gemm(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
