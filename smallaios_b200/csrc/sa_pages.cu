// C entry points of paged serving: the page pool, appending to pages,
// attention over pages, and beam search (argument checks; the kernels are in
// kv_pages_append.cu, gqa_pages.cu, beam_select.cu and kv_pages_reorder.cu).
#include <stdlib.h>
#include <string.h>

#include <new>

#include "sa_pages.cuh"

using namespace sa;

namespace {

bool dtype_ok(int32_t dt) { return dt == SA_DTYPE_FLOAT || dt == SA_DTYPE_FLOAT16 || dt == SA_DTYPE_BFLOAT16; }

kv_pages_impl *impl(sa_kv_pages *p) { return reinterpret_cast<kv_pages_impl *>(p); }
const kv_pages_impl *impl(const sa_kv_pages *p) { return reinterpret_cast<const kv_pages_impl *>(p); }

// Makes the pool's device current while a call launches on it.
struct OnDevice {
    int before = -1;
    explicit OnDevice(int device) {
        if (cudaGetDevice(&before) != cudaSuccess) before = -1;
        if (before == device) before = -1;
        else cudaSetDevice(device);
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// Checks shared by the calls over rows of new tokens.
int check_rows(const char *op, const kv_pages_impl *k, int32_t layer, int32_t dtype, int32_t batch, int32_t seq_len,
               int64_t batch_stride, int64_t token_stride, int64_t width, const int32_t *page_table,
               int64_t table_stride, int32_t max_pages, const int32_t *seq_lens) {
    if (layer < 0 || layer >= k->cfg.num_layers)
        return set_error(SA_ERR_INVALID_ARGUMENT, "%s: layer_idx %d", op, layer);
    if (!dtype_ok(dtype)) return set_error(SA_ERR_UNSUPPORTED, "%s: dtype %d not supported", op, dtype);
    if (batch < 0 || seq_len < 0) return set_error(SA_ERR_SHAPE_MISMATCH, "%s: batch %d, seq_len %d", op, batch, seq_len);
    if (max_pages < 0 || max_pages > INT32_MAX / kPageTokens || table_stride < max_pages)
        return set_error(SA_ERR_SHAPE_MISMATCH, "%s: table rows of %d pages, %lld apart", op, max_pages,
                         (long long)table_stride);
    if ((int64_t)batch * seq_len > INT32_MAX)
        return set_error(SA_ERR_UNSUPPORTED, "%s: %d x %d tokens", op, batch, seq_len);
    if (batch == 0 || seq_len == 0) return SA_OK;
    if ((seq_len > 1 && token_stride < width) || (batch > 1 && batch_stride < width))
        return set_error(SA_ERR_SHAPE_MISMATCH, "%s: strides %lld, %lld below the width %lld", op,
                         (long long)batch_stride, (long long)token_stride, (long long)width);
    if (!seq_lens || (!page_table && max_pages > 0))
        return set_error(SA_ERR_INVALID_ARGUMENT, "%s: NULL page_table/seq_lens", op);
    return SA_OK;
}

// As check_rope of the contiguous cache; the positions themselves are on the device.
int check_tables(const char *op, int32_t do_rotary, const float *cos_cache, const float *sin_cache, int32_t rows) {
    if (!do_rotary) return SA_OK;
    if (!cos_cache || !sin_cache || rows <= 0)
        return set_error(SA_ERR_SHAPE_MISMATCH, "%s: do_rotary=1 requires cos_cache and sin_cache (tables of %d rows)", op, rows);
    return SA_OK;
}

PageRows page_rows(const kv_pages_impl *k, const int32_t *page_table, int64_t table_stride, int32_t max_pages,
                   const int32_t *seq_lens, const int32_t *counts) {
    return PageRows{page_table, table_stride, max_pages, seq_lens, counts, k->cfg.num_pages, k->dev_status};
}

RopeArgs rope_args(const float *cos_cache, const float *sin_cache, int32_t rows, int32_t on, int32_t interleaved) {
    const int aligned = ((reinterpret_cast<uintptr_t>(cos_cache) | reinterpret_cast<uintptr_t>(sin_cache)) & 15) == 0;
    return RopeArgs{cos_cache, sin_cache, rows, on != 0, interleaved != 0, aligned};
}

bool vectors_aligned(const void *p, int64_t batch_stride, int64_t token_stride, int32_t dtype, int batch, int seq_len) {
    const int64_t width = dtype == SA_DTYPE_FLOAT ? 4 : 2;
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (batch <= 1 || batch_stride * width % 16 == 0) &&
           (seq_len <= 1 || token_stride * width % 16 == 0);
}

// Whether two tables of `rows` rows of `width` pages share an element.  Column slices of one table lie between each
// other's rows and share none.
bool tables_overlap(const int32_t *x, int64_t x_stride, const int32_t *y, int64_t y_stride, int64_t rows, int64_t width) {
    const int64_t bytes = width * 4, step = y_stride * 4;
    const int64_t first = (int64_t)(reinterpret_cast<uintptr_t>(y) - reinterpret_cast<uintptr_t>(x));  // of y, from x on
    if (first >= (rows - 1) * x_stride * 4 + bytes || first + (rows - 1) * step + bytes <= 0) return false;
    for (int64_t i = 0; i < rows; i++) {
        // the last row of y that begins before row i of x ends
        const int64_t before = i * x_stride * 4 + bytes - 1 - first;
        if (before < 0) continue;
        const int64_t j = before / step < rows - 1 ? before / step : rows - 1;
        if (first + j * step + bytes > i * x_stride * 4) return true;
    }
    return false;
}

}  // namespace

extern "C" {

int sa_kv_pages_create(const sa_kv_pages_config *config, sa_kv_pages **out) {
    if (!config || !out) return set_error(SA_ERR_INVALID_ARGUMENT, "kv_pages_create: NULL argument");
    *out = nullptr;
    const sa_kv_pages_config c = *config;
    if (c.num_layers <= 0 || c.num_pages <= 0 || c.num_kv_heads <= 0)
        return set_error(SA_ERR_INVALID_ARGUMENT, "kv_pages_create: zero dimension");
    if (c.bits != 4 && c.bits != 8) return set_error(SA_ERR_UNSUPPORTED, "kv_pages_create: bits must be 4 or 8");
    if (c.head_dim != 64 && c.head_dim != 128)
        return set_error(SA_ERR_UNSUPPORTED, "kv_pages_create: head_dim %d, not 64 or 128", c.head_dim);
    if (c.num_heads <= 0 || c.num_heads % c.num_kv_heads != 0)
        return set_error(SA_ERR_INVALID_ATTRIBUTE, "num_heads must be a positive multiple of num_kv_heads");
    if (c.kv_head_count <= 0 || c.kv_head_begin < 0 || c.kv_head_count > c.num_kv_heads - c.kv_head_begin)
        return set_error(SA_ERR_INVALID_ATTRIBUTE, "kv head range [%d, +%d) outside [0, %d)", c.kv_head_begin,
                         c.kv_head_count, c.num_kv_heads);
    // more than any B200 holds, and the products below fit in 64 bits
    if ((double)c.num_layers * c.num_pages * c.kv_head_count * page_record(c.head_dim * c.bits / 8) > 0x1p38)
        return set_error(SA_ERR_OUT_OF_MEMORY, "kv_pages_create: %d layers of %d pages for %d heads need more than 256 GiB",
                         c.num_layers, c.num_pages, c.kv_head_count);
    kv_pages_impl *k = new (std::nothrow) kv_pages_impl();
    if (!k) return set_error(SA_ERR_OUT_OF_MEMORY, "kv_pages_create: no host memory");
    memset(k, 0, sizeof(*k));
    k->cfg = c;
    k->code_bytes = c.head_dim * c.bits / 8;
    k->group = c.num_heads / c.num_kv_heads;
    k->wht_scale = 1.0f / host_sqrt_approx((float)c.head_dim);
    const size_t H = c.kv_head_count, L = c.num_layers, D = c.head_dim;
    float *signs = static_cast<float *>(malloc(L * H * D * sizeof(float)));
    int rc = signs ? check_cuda(cudaGetDevice(&k->device), "cudaGetDevice")
                   : set_error(SA_ERR_OUT_OF_MEMORY, "kv_pages_create: no host memory");
    if (rc == SA_OK) {
        for (size_t l = 0; l < L; l++)
            for (size_t h = 0; h < H; h++)
                make_signs(head_seed(c.seed, (int)l, c.num_kv_heads, c.kv_head_begin + (int)h), (int)D, signs + (l * H + h) * D);
        cudaDeviceGetAttribute(&k->sm_count, cudaDevAttrMultiProcessorCount, k->device);
        if (k->sm_count <= 0) k->sm_count = 148;
        const size_t sign_bytes = (L * H * D * sizeof(float) + 255) / 256 * 256;
        k->layer_bytes = (size_t)c.num_pages * H * page_record(k->code_bytes);
        const size_t bytes = L * k->layer_bytes + sign_bytes + 256;
        cudaError_t e = cudaMalloc(&k->base, bytes);
        if (e != cudaSuccess) {
            cudaGetLastError();
            rc = set_error(SA_ERR_OUT_OF_MEMORY, "kv_pages_create: cudaMalloc(%zu bytes) failed: %s", bytes,
                           cudaGetErrorString(e));
        } else {
            k->records = static_cast<uint8_t *>(k->base);
            k->signs = reinterpret_cast<float *>(k->records + L * k->layer_bytes);
            k->dev_status = reinterpret_cast<int *>(k->records + L * k->layer_bytes + sign_bytes);
            e = cudaMemset(k->base, 0, bytes);
            if (e == cudaSuccess) e = cudaMemcpy(k->signs, signs, L * H * D * sizeof(float), cudaMemcpyHostToDevice);
            if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);  // both are over when the call returns
            rc = check_cuda(e, "kv_pages_create init");
            if (rc != SA_OK) cudaFree(k->base);
        }
    }
    free(signs);
    if (rc != SA_OK) {
        delete k;
        return rc;
    }
    *out = reinterpret_cast<sa_kv_pages *>(k);
    return SA_OK;
}

int sa_kv_pages_destroy(sa_kv_pages *pages) {
    if (!pages) return SA_OK;
    kv_pages_impl *k = impl(pages);
    cudaError_t e;
    {
        OnDevice on(k->device);
        e = cudaFree(k->base);
    }
    delete k;
    return check_cuda(e, "kv_pages_destroy cudaFree");
}

int sa_kv_pages_get_config(const sa_kv_pages *pages, sa_kv_pages_config *config) {
    if (!pages || !config) return set_error(SA_ERR_INVALID_ARGUMENT, "kv_pages_get_config: NULL argument");
    *config = impl(pages)->cfg;
    return SA_OK;
}

int sa_kv_pages_layer_view(const sa_kv_pages *pages, int32_t layer, sa_kv_pages_view *view) {
    if (!pages || !view) return set_error(SA_ERR_INVALID_ARGUMENT, "kv_pages_layer_view: NULL argument");
    const kv_pages_impl *k = impl(pages);
    if (layer < 0 || layer >= k->cfg.num_layers)
        return set_error(SA_ERR_INVALID_ARGUMENT, "kv_pages_layer_view: layer_idx %d", layer);
    view->records = k->records + (size_t)layer * k->layer_bytes;
    view->signs = k->signs + (size_t)layer * k->cfg.kv_head_count * k->cfg.head_dim;
    view->num_pages = k->cfg.num_pages;
    view->kv_heads = k->cfg.kv_head_count;
    view->head_dim = k->cfg.head_dim;
    view->bits = k->cfg.bits;
    view->code_bytes = k->code_bytes;
    view->record_bytes = page_record(k->code_bytes);
    view->k_meta_offset = page_k_meta(k->code_bytes);
    view->v_meta_offset = page_v_meta(k->code_bytes);
    view->v_codes_offset = page_v_codes(k->code_bytes);
    view->wht_scale = k->wht_scale;
    return SA_OK;
}

int sa_kv_pages_device_status(sa_kv_pages *pages, int32_t *status, int32_t clear) {
    if (!pages || !status) return set_error(SA_ERR_INVALID_ARGUMENT, "kv_pages_device_status: NULL argument");
    kv_pages_impl *k = impl(pages);
    OnDevice on(k->device);
    int v = 0;
    int rc = check_cuda(cudaDeviceSynchronize(), "kv_pages_device_status");
    if (rc == SA_OK)
        rc = check_cuda(cudaMemcpy(&v, k->dev_status, sizeof(int), cudaMemcpyDeviceToHost), "kv_pages_device_status read");
    if (rc != SA_OK) return rc;
    *status = v;
    if (clear && v) rc = check_cuda(cudaMemset(k->dev_status, 0, sizeof(int)), "kv_pages_device_status clear");
    return rc;
}

int sa_kv_pages_append(sa_kv_pages *pages, int32_t layer, const void *key, const void *value, int64_t batch_stride,
                       int64_t token_stride, int32_t dtype, int32_t batch, int32_t seq_len, const int32_t *page_table,
                       int64_t table_stride, int32_t max_pages, const int32_t *seq_lens, const int32_t *counts,
                       const float *cos_cache, const float *sin_cache, int32_t cache_rows, int32_t do_rotary,
                       int32_t rotary_interleaved, sa_stream_t stream) {
    if (!pages) return set_error(SA_ERR_INVALID_ARGUMENT, "kv_pages_append: NULL pages");
    const kv_pages_impl *k = impl(pages);
    const int64_t width = (int64_t)k->cfg.kv_head_count * k->cfg.head_dim;
    int rc = check_rows("kv_pages_append", k, layer, dtype, batch, seq_len, batch_stride, token_stride, width, page_table,
                        table_stride, max_pages, seq_lens);
    if (rc == SA_OK) rc = check_tables("kv_pages_append", do_rotary, cos_cache, sin_cache, cache_rows);
    if (rc != SA_OK || batch == 0 || seq_len == 0) return rc;
    if (!key || !value) return set_error(SA_ERR_INVALID_ARGUMENT, "kv_pages_append: NULL key/value");
    if ((int64_t)batch * k->cfg.kv_head_count > INT32_MAX)
        return set_error(SA_ERR_UNSUPPORTED, "kv_pages_append: %d rows of %d heads", batch, k->cfg.kv_head_count);
    PagesAppendArgs a{};
    a.key = key;
    a.value = value;
    a.batch_stride = batch_stride;
    a.token_stride = token_stride;
    a.aligned = vectors_aligned(key, batch_stride, token_stride, dtype, batch, seq_len) &&
                vectors_aligned(value, batch_stride, token_stride, dtype, batch, seq_len);
    a.dtype = dtype;
    a.batch = batch;
    a.seq_len = seq_len;
    a.heads = k->cfg.kv_head_count;
    a.head_dim = k->cfg.head_dim;
    a.bits = k->cfg.bits;
    a.records = k->records + (size_t)layer * k->layer_bytes;
    a.signs = k->signs + (size_t)layer * width;
    a.wht_scale = k->wht_scale;
    a.rows = page_rows(k, page_table, table_stride, max_pages, seq_lens, counts);
    a.rope = rope_args(cos_cache, sin_cache, cache_rows, do_rotary, rotary_interleaved);
    OnDevice on(k->device);
    return launch_pages_append(a, static_cast<cudaStream_t>(stream));
}

int sa_kv_pages_set_precision(sa_kv_pages *pages, int32_t full) {
    if (!pages) return set_error(SA_ERR_INVALID_ARGUMENT, "kv_pages_set_precision: NULL pages");
    impl(pages)->full = full != 0;
    return SA_OK;
}

int64_t sa_gqa_paged_workspace_bytes(const sa_kv_pages *pages, int32_t batch, int32_t seq_len, int32_t dtype) {
    if (!pages || batch <= 0 || seq_len <= 0 || !dtype_ok(dtype) || (int64_t)batch * seq_len > INT32_MAX) return 0;
    return (int64_t)pages_attend_workspace(impl(pages), batch, seq_len, dtype);
}

int sa_gqa_paged_attend(sa_kv_pages *pages, int32_t layer, const void *query, int64_t batch_stride,
                        int64_t token_stride, void *attn_out, int32_t dtype, int32_t batch, int32_t seq_len,
                        int64_t num_heads, int32_t has_scale, float scale, const int32_t *page_table,
                        int64_t table_stride, int32_t max_pages, const int32_t *seq_lens, const int32_t *counts,
                        const float *cos_cache, const float *sin_cache, int32_t cache_rows, int32_t do_rotary,
                        int32_t rotary_interleaved, void *workspace, int64_t workspace_bytes, sa_stream_t stream) {
    if (!pages) return set_error(SA_ERR_INVALID_ARGUMENT, "gqa_paged_attend: NULL pages");
    const kv_pages_impl *k = impl(pages);
    const int64_t width = (int64_t)k->cfg.kv_head_count * k->group * k->cfg.head_dim;
    int rc = check_rows("gqa_paged_attend", k, layer, dtype, batch, seq_len, batch_stride, token_stride, width, page_table,
                        table_stride, max_pages, seq_lens);
    if (rc == SA_OK) rc = check_tables("gqa_paged_attend", do_rotary, cos_cache, sin_cache, cache_rows);
    if (rc != SA_OK) return rc;
    if (num_heads != k->cfg.num_heads)
        return set_error(SA_ERR_SHAPE_MISMATCH, "gqa_paged_attend: num_heads %lld != %d", (long long)num_heads,
                         k->cfg.num_heads);
    if (batch == 0 || seq_len == 0) return SA_OK;
    if (!query || !attn_out) return set_error(SA_ERR_INVALID_ARGUMENT, "gqa_paged_attend: NULL query/attn_out");
    const int64_t need = sa_gqa_paged_workspace_bytes(pages, batch, seq_len, dtype);
    if (!workspace || workspace_bytes < need)
        return set_error(SA_ERR_INVALID_ARGUMENT, "gqa_paged_attend: workspace of %lld bytes, needs %lld",
                         workspace ? (long long)workspace_bytes : 0ll, (long long)need);
    if (reinterpret_cast<uintptr_t>(workspace) & 255)
        return set_error(SA_ERR_INVALID_ARGUMENT, "gqa_paged_attend: workspace must be 256-byte aligned");
    PagesAttendArgs a{};
    a.query = query;
    a.batch_stride = batch_stride;
    a.token_stride = token_stride;
    a.out = attn_out;
    a.dtype = dtype;
    a.batch = batch;
    a.seq_len = seq_len;
    a.heads = k->cfg.kv_head_count;
    a.group = k->group;
    a.head_dim = k->cfg.head_dim;
    a.bits = k->cfg.bits;
    a.full = k->full;
    a.records = k->records + (size_t)layer * k->layer_bytes;
    a.signs = k->signs + (size_t)layer * k->cfg.kv_head_count * k->cfg.head_dim;
    a.wht_scale = k->wht_scale;
    a.scale = has_scale ? scale : 1.0f / host_sqrt_f32((float)k->cfg.head_dim);
    a.sm_count = k->sm_count;
    a.rows = page_rows(k, page_table, table_stride, max_pages, seq_lens, counts);
    a.rope = rope_args(cos_cache, sin_cache, cache_rows, do_rotary, rotary_interleaved);
    OnDevice on(k->device);
    return launch_pages_attend(a, workspace, static_cast<cudaStream_t>(stream));
}

int64_t sa_beam_select_workspace_bytes(int32_t batch, int32_t num_beams, int64_t vocab) {
    if (batch <= 0 || num_beams <= 0 || num_beams > SA_MAX_BEAMS || vocab <= 0 || vocab * num_beams > INT32_MAX) return 0;
    return beam_select_workspace((int64_t)batch * num_beams, vocab);
}

int sa_beam_select(const void *logits, int64_t row_stride, int32_t dtype, const float *scores, const uint8_t *finished,
                   int32_t batch, int32_t num_beams, int64_t vocab, int32_t end_token, int32_t keep, int32_t *parents,
                   int32_t *tokens, float *out_scores, void *workspace, int64_t workspace_bytes, sa_stream_t stream) {
    if (!dtype_ok(dtype)) return set_error(SA_ERR_UNSUPPORTED, "beam_select: dtype %d not supported", dtype);
    if (batch < 0) return set_error(SA_ERR_SHAPE_MISMATCH, "beam_select: negative batch");
    if (num_beams < 1 || num_beams > SA_MAX_BEAMS)
        return set_error(SA_ERR_INVALID_ATTRIBUTE, "beam_select: %d beams (1..%d)", num_beams, SA_MAX_BEAMS);
    if (keep < 1 || keep > SA_MAX_BEAM_KEEP)
        return set_error(SA_ERR_INVALID_ATTRIBUTE, "beam_select: keep %d (1..%d)", keep, SA_MAX_BEAM_KEEP);
    if (vocab < 1 || row_stride < vocab)
        return set_error(SA_ERR_SHAPE_MISMATCH, "beam_select: rows of %lld tokens, %lld apart", (long long)vocab,
                         (long long)row_stride);
    if (vocab > INT32_MAX / num_beams || batch > INT32_MAX / num_beams)
        return set_error(SA_ERR_UNSUPPORTED, "beam_select: %d x %d beams over %lld tokens", batch, num_beams,
                         (long long)vocab);
    if (batch == 0) return SA_OK;
    if (!logits || !scores || !parents || !tokens || !out_scores)
        return set_error(SA_ERR_INVALID_ARGUMENT, "beam_select: NULL argument");
    if (reinterpret_cast<uintptr_t>(logits) % (dtype == SA_DTYPE_FLOAT ? 4 : 2))
        return set_error(SA_ERR_INVALID_ARGUMENT, "beam_select: logits must be aligned to their elements");
    const int64_t need = sa_beam_select_workspace_bytes(batch, num_beams, vocab);
    if (!workspace || workspace_bytes < need)
        return set_error(SA_ERR_INVALID_ARGUMENT, "beam_select: workspace of %lld bytes, needs %lld",
                         workspace ? (long long)workspace_bytes : 0ll, (long long)need);
    if (reinterpret_cast<uintptr_t>(workspace) & 255)
        return set_error(SA_ERR_INVALID_ARGUMENT, "beam_select: workspace must be 256-byte aligned");
    BeamArgs a{};
    a.logits = logits;
    a.row_stride = row_stride;
    a.dtype = dtype;
    a.batch = batch;
    a.beams = num_beams;
    a.keep = keep;
    a.end_token = end_token;
    a.vocab = (int)vocab;
    a.scores = scores;
    a.finished = finished;
    a.parents = parents;
    a.tokens = tokens;
    a.out_scores = out_scores;
    return launch_beam_select(a, workspace, static_cast<cudaStream_t>(stream));
}

int sa_kv_pages_reorder(sa_kv_pages *pages, const int32_t *page_table, int64_t table_stride, int32_t *new_table,
                        int64_t new_stride, int32_t max_pages, const int32_t *seq_lens, const int32_t *parents,
                        int32_t batch, int32_t num_beams, sa_stream_t stream) {
    if (!pages) return set_error(SA_ERR_INVALID_ARGUMENT, "kv_pages_reorder: NULL pages");
    const kv_pages_impl *k = impl(pages);
    if (batch < 0) return set_error(SA_ERR_SHAPE_MISMATCH, "kv_pages_reorder: negative batch");
    if (num_beams < 1 || num_beams > SA_MAX_BEAMS)
        return set_error(SA_ERR_INVALID_ATTRIBUTE, "kv_pages_reorder: %d beams (1..%d)", num_beams, SA_MAX_BEAMS);
    if (max_pages < 0 || max_pages > INT32_MAX / kPageTokens || table_stride < max_pages || new_stride < max_pages)
        return set_error(SA_ERR_SHAPE_MISMATCH, "kv_pages_reorder: table rows of %d pages, %lld and %lld apart", max_pages,
                         (long long)table_stride, (long long)new_stride);
    if (batch > 65535 || k->cfg.num_layers > 65535)
        return set_error(SA_ERR_UNSUPPORTED, "kv_pages_reorder: %d groups, %d layers", batch, k->cfg.num_layers);
    if (batch == 0 || max_pages == 0) return SA_OK;
    if (!page_table || !new_table || !seq_lens || !parents)
        return set_error(SA_ERR_INVALID_ARGUMENT, "kv_pages_reorder: NULL argument");
    if (tables_overlap(page_table, table_stride, new_table, new_stride, (int64_t)batch * num_beams, max_pages))
        return set_error(SA_ERR_INVALID_ARGUMENT, "kv_pages_reorder: the new table overlaps the old one");
    ReorderArgs a{};
    a.records = k->records;
    a.layer_bytes = k->layer_bytes;
    a.layers = k->cfg.num_layers;
    a.heads = k->cfg.kv_head_count;
    a.code_bytes = k->code_bytes;
    a.table = page_table;
    a.table_stride = table_stride;
    a.out = new_table;
    a.out_stride = new_stride;
    a.max_pages = max_pages;
    a.lens = seq_lens;
    a.parents = parents;
    a.batch = batch;
    a.beams = num_beams;
    a.num_pages = k->cfg.num_pages;
    a.dev_status = k->dev_status;
    OnDevice on(k->device);
    return launch_pages_reorder(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
