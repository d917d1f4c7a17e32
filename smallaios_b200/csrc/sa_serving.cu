// C entry points of the serving operators: attention of a draft tree, keeping
// the accepted drafts, block means, block selection and block-sparse attention
// (argument checks and workspace layout; the kernels are in gqa_tree_umma.cu,
// gqa_attend.cu, kv_keep.cu, kv_blocks.cu, gqa_decode_mma.cu and
// gqa_decode_g8.cu).
#include "sa_common.cuh"
#include "sa_internal.h"

using namespace sa;

namespace {

bool dtype_ok(int32_t dt) { return dt == SA_DTYPE_FLOAT || dt == SA_DTYPE_FLOAT16 || dt == SA_DTYPE_BFLOAT16; }

// Checks shared by the calls that take query tokens at the cache position.
int check_queries(const char *op, const kv_cache_impl *k, int32_t layer, int32_t dtype, int32_t batch, int32_t seq_len,
                  int64_t num_heads) {
    if (layer < 0 || layer >= k->cfg.num_layers)
        return set_error(SA_ERR_INVALID_ARGUMENT, "%s: layer_idx %d", op, layer);
    if (!dtype_ok(dtype)) return set_error(SA_ERR_UNSUPPORTED, "%s: dtype %d not supported", op, dtype);
    if (batch != k->cfg.batch)
        return set_error(SA_ERR_SHAPE_MISMATCH, "%s: batch %d != cache batch %d", op, batch, k->cfg.batch);
    if (num_heads != k->cfg.num_heads)
        return set_error(SA_ERR_SHAPE_MISMATCH, "%s: num_heads %lld != cache num_heads %d", op, (long long)num_heads,
                         k->cfg.num_heads);
    if (k->group > 8) return set_error(SA_ERR_UNSUPPORTED, "%s: group size %d > 8 not supported", op, k->group);
    if (seq_len < 0) return set_error(SA_ERR_SHAPE_MISMATCH, "%s: negative sequence length", op);
    if (k->position + seq_len > k->cfg.max_seq_len)
        return set_error(SA_ERR_CAPACITY, "%s: tokens past max_seq_len (%lld + %d > %d)", op, (long long)k->position,
                         seq_len, k->cfg.max_seq_len);
    if (k->gather.n != 0)
        return set_error(SA_ERR_UNSUPPORTED, "%s: not with a head-sharded gather set on the cache", op);
    return SA_OK;
}

int check_workspace(const char *op, const void *workspace, int64_t have, int64_t need) {
    if (need == 0) return SA_OK;
    if (!workspace || have < need)
        return set_error(SA_ERR_INVALID_ARGUMENT, "%s: workspace of %lld bytes, needs %lld", op,
                         workspace ? (long long)have : 0ll, (long long)need);
    if (reinterpret_cast<uintptr_t>(workspace) & 255)
        return set_error(SA_ERR_INVALID_ARGUMENT, "%s: workspace must be 256-byte aligned", op);
    return SA_OK;
}

AttendArgs attend_args(kv_cache_impl *k, int32_t layer, const void *query, void *out, int32_t dtype, int32_t batch,
                       int32_t seq_len, int32_t has_scale, float scale) {
    sa_kv_layer_view v;
    sa_kv_cache_layer_view(reinterpret_cast<sa_kv_cache *>(k), layer, &v);
    AttendArgs a{};
    a.query = query;
    a.out = out;
    a.dtype = dtype;
    a.batch = batch;
    a.seq_len = seq_len;
    a.heads = v.kv_heads;
    a.group = k->group;
    a.head_dim = v.head_dim;
    a.bits = v.bits;
    a.code_bytes = v.code_bytes;
    a.capacity = v.capacity;
    a.pos0 = k->position;
    a.k_codes = v.k_codes;
    a.v_codes = v.v_codes;
    a.k_meta = v.lr_vtr ? v.lr_kmeta : v.k_meta;  // low-rank K: {0, U*S[t]} and q'.V^T, as in sa_gqa_attend
    a.v_meta = v.v_meta;
    a.signs = v.signs;
    a.wht_scale = v.wht_scale;
    a.scale = has_scale ? scale : 1.0f / host_sqrt_f32((float)v.head_dim);
    a.workspace = k->workspace;
    a.workspace_floats = k->workspace_floats;
    a.sm_count = k->sm_count;
    a.qprep = k->qprep;
    a.dev_status = k->dev_status;
    a.lr_vtr = v.lr_vtr;
    return a;
}

// Query rows of one launch of the tensor-core decode over block lists: bounds its workspace.
constexpr int64_t kListUnits = 16384;

int64_t list_rows_per_launch(const kv_cache_impl *k, int64_t rows) {
    const int64_t most = kListUnits / k->cfg.kv_head_count > 0 ? kListUnits / k->cfg.kv_head_count : 1;
    return rows < most ? rows : most;
}

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// Bytes of the partial records, and of the q digits behind them, of a launch of `rows` query rows.
void list_workspace(const kv_cache_impl *k, int64_t rows, size_t *records, size_t *digits) {
    const int64_t units = rows * k->cfg.kv_head_count;
    *records = align256(decode_workspace_floats(k->sm_count, units, k->cfg.head_dim, k->group) * sizeof(float));
    *digits = align256((size_t)units * decode_qprep_words(k->group) * sizeof(uint32_t));
}

// Whether block lists go to the tensor-core decode.
bool list_decode_format(const kv_cache_impl *k) {
    return (k->cfg.bits == 4 || k->cfg.bits == 8) && (k->cfg.head_dim == 64 || k->cfg.head_dim == 128) &&
           k->group <= 8;
}

}  // namespace

extern "C" {

int64_t sa_gqa_tree_workspace_bytes(const sa_kv_cache *cache, int32_t nodes, int32_t dtype) {
    const kv_cache_impl *k = reinterpret_cast<const kv_cache_impl *>(cache);
    if (!cache || nodes <= 0 || nodes > SA_MAX_DRAFT_NODES || !dtype_ok(dtype) || k->group > 8) return 0;
    return (int64_t)tree_workspace_bytes(k->cfg.batch, k->cfg.kv_head_count, k->group, k->cfg.head_dim, k->cfg.bits,
                                         k->sm_count, k->capacity, nodes, dtype, k->tree_full);
}

int sa_kv_cache_set_tree_precision(sa_kv_cache *cache, int32_t full) {
    if (!cache) return set_error(SA_ERR_INVALID_ARGUMENT, "kv_cache_set_tree_precision: NULL cache");
    reinterpret_cast<kv_cache_impl *>(cache)->tree_full = full != 0;
    return SA_OK;
}

int sa_gqa_tree_attend(sa_kv_cache *cache, int32_t layer, const void *query, const int32_t *parents, void *attn_out,
                       int32_t dtype, int32_t batch, int32_t nodes, int64_t num_heads, int32_t has_scale, float scale,
                       void *workspace, int64_t workspace_bytes, sa_stream_t stream) {
    if (!cache) return set_error(SA_ERR_INVALID_ARGUMENT, "gqa_tree_attend: NULL cache");
    kv_cache_impl *k = reinterpret_cast<kv_cache_impl *>(cache);
    int rc = check_queries("gqa_tree_attend", k, layer, dtype, batch, nodes, num_heads);
    if (rc != SA_OK) return rc;
    if (nodes > SA_MAX_DRAFT_NODES)
        return set_error(SA_ERR_UNSUPPORTED, "gqa_tree_attend: %d nodes, at most %d", nodes, SA_MAX_DRAFT_NODES);
    if (nodes == 0) return SA_OK;
    if (!query || !parents || !attn_out)
        return set_error(SA_ERR_INVALID_ARGUMENT, "gqa_tree_attend: NULL query/parents/attn_out");
    const int64_t need = sa_gqa_tree_workspace_bytes(cache, nodes, dtype);
    rc = check_workspace("gqa_tree_attend", workspace, workspace_bytes, need);
    if (rc != SA_OK) return rc;
    AttendArgs a = attend_args(k, layer, query, attn_out, dtype, batch, nodes, has_scale, scale);
    a.parents = parents;
    a.tree_full = k->tree_full;
    if (need > 0) return launch_gqa_tree_umma(a, workspace, static_cast<cudaStream_t>(stream));
    return launch_gqa_attend_generic(a, static_cast<cudaStream_t>(stream));
}

int sa_kv_cache_keep_drafts(sa_kv_cache *cache, const int32_t *path, int32_t batch, int32_t n, int32_t drafted,
                            sa_stream_t stream) {
    if (!cache) return set_error(SA_ERR_INVALID_ARGUMENT, "kv_cache_keep_drafts: NULL cache");
    kv_cache_impl *k = reinterpret_cast<kv_cache_impl *>(cache);
    if (k->cfg.lowrank_k > 0)
        return set_error(SA_ERR_UNSUPPORTED, "kv_cache_keep_drafts: low-rank K state follows writes in order");
    if (batch != k->cfg.batch)
        return set_error(SA_ERR_SHAPE_MISMATCH, "kv_cache_keep_drafts: batch %d != cache batch %d", batch,
                         k->cfg.batch);
    if (drafted < 0 || drafted > SA_MAX_DRAFT_NODES)
        return set_error(SA_ERR_UNSUPPORTED, "kv_cache_keep_drafts: %d drafts, at most %d", drafted,
                         SA_MAX_DRAFT_NODES);
    if (n < 0 || n > drafted)
        return set_error(SA_ERR_SHAPE_MISMATCH, "kv_cache_keep_drafts: %d of %d drafts", n, drafted);
    if (k->position + drafted > k->cfg.max_seq_len)
        return set_error(SA_ERR_CAPACITY, "kv_cache_keep_drafts: drafts past max_seq_len");
    if (n == 0) return SA_OK;
    if (!path) return set_error(SA_ERR_INVALID_ARGUMENT, "kv_cache_keep_drafts: NULL path");
    KeepArgs a{};
    a.k_codes = k->k_codes;
    a.v_codes = k->v_codes;
    a.k_meta = k->k_meta;
    a.v_meta = k->v_meta;
    a.k_qjl_bits = k->k_qjl_bits;
    a.v_qjl_bits = k->v_qjl_bits;
    a.k_qjl_mag = k->k_qjl_mag;
    a.v_qjl_mag = k->v_qjl_mag;
    a.path = path;
    a.layers = k->cfg.num_layers;
    a.batch = batch;
    a.heads = k->cfg.kv_head_count;
    a.head_dim = k->cfg.head_dim;
    a.code_bytes = k->code_bytes;
    a.capacity = k->capacity;
    a.n = n;
    a.drafted = drafted;
    a.pos0 = k->position;
    a.dev_status = k->dev_status;
    return launch_keep_drafts(a, static_cast<cudaStream_t>(stream));
}

int sa_kv_block_means(sa_kv_cache *cache, int32_t layer, void *means, int64_t row_stride, int32_t block_begin,
                      int32_t block_end, sa_stream_t stream) {
    if (!cache) return set_error(SA_ERR_INVALID_ARGUMENT, "kv_block_means: NULL cache");
    kv_cache_impl *k = reinterpret_cast<kv_cache_impl *>(cache);
    if (layer < 0 || layer >= k->cfg.num_layers)
        return set_error(SA_ERR_INVALID_ARGUMENT, "kv_block_means: layer_idx %d", layer);
    if (k->cfg.lowrank_k > 0) return set_error(SA_ERR_UNSUPPORTED, "kv_block_means: not with low-rank K");
    if (block_begin < 0 || block_end < block_begin || block_end > k->capacity / SA_BLOCK_TOKENS)
        return set_error(SA_ERR_SHAPE_MISMATCH, "kv_block_means: blocks [%d, %d) of %d", block_begin, block_end,
                         k->capacity / SA_BLOCK_TOKENS);
    if (block_begin == block_end) return SA_OK;
    if (row_stride < (int64_t)(block_end - block_begin) * k->cfg.head_dim)
        return set_error(SA_ERR_SHAPE_MISMATCH, "kv_block_means: row stride %lld below %d blocks of %d values",
                         (long long)row_stride, block_end - block_begin, k->cfg.head_dim);
    if (!means) return set_error(SA_ERR_INVALID_ARGUMENT, "kv_block_means: NULL means");
    if ((reinterpret_cast<uintptr_t>(means) & 15) || row_stride % 8 != 0)
        return set_error(SA_ERR_UNSUPPORTED, "kv_block_means: means rows must be 16-byte aligned");
    sa_kv_layer_view v;
    sa_kv_cache_layer_view(cache, layer, &v);
    MeansArgs a{};
    a.k_codes = v.k_codes;
    a.k_meta = v.k_meta;
    a.means = means;
    a.row_stride = row_stride;
    a.units = v.batch * v.kv_heads;
    a.head_dim = v.head_dim;
    a.bits = v.bits;
    a.code_bytes = v.code_bytes;
    a.capacity = v.capacity;
    a.first = block_begin;
    a.blocks = block_end - block_begin;
    return launch_block_means(a, static_cast<cudaStream_t>(stream));
}

int sa_gqa_select_blocks(sa_kv_cache *cache, int32_t layer, const void *query, int32_t dtype, int32_t batch,
                         int32_t seq_len, int64_t num_heads, const void *means, int64_t row_stride,
                         int64_t means_blocks, int32_t max_blocks, int32_t sink_blocks, int32_t local_blocks,
                         int32_t *block_ids, sa_stream_t stream) {
    if (!cache) return set_error(SA_ERR_INVALID_ARGUMENT, "gqa_select_blocks: NULL cache");
    kv_cache_impl *k = reinterpret_cast<kv_cache_impl *>(cache);
    int rc = check_queries("gqa_select_blocks", k, layer, dtype, batch, seq_len, num_heads);
    if (rc != SA_OK) return rc;
    if (k->cfg.lowrank_k > 0) return set_error(SA_ERR_UNSUPPORTED, "gqa_select_blocks: not with low-rank K");
    if (sink_blocks < 0 || local_blocks < 1 || (int64_t)sink_blocks + local_blocks > max_blocks)
        return set_error(SA_ERR_INVALID_ATTRIBUTE,
                         "gqa_select_blocks: %d first and %d last blocks (at least 1) in %d blocks", sink_blocks,
                         local_blocks, max_blocks);
    if (seq_len == 0) return SA_OK;
    const int64_t earlier = (k->position + seq_len - 1) / SA_BLOCK_TOKENS;  // blocks before the last query's own
    if (means_blocks < earlier || (earlier > 0 && row_stride < earlier * k->cfg.head_dim))
        return set_error(SA_ERR_SHAPE_MISMATCH, "gqa_select_blocks: means of %lld blocks (row stride %lld), needs %lld",
                         (long long)means_blocks, (long long)row_stride, (long long)earlier);
    if (!query || !block_ids || (!means && earlier > 0))
        return set_error(SA_ERR_INVALID_ARGUMENT, "gqa_select_blocks: NULL query/means/block_ids");
    if ((reinterpret_cast<uintptr_t>(means) & 15) || row_stride % 8 != 0)
        return set_error(SA_ERR_UNSUPPORTED, "gqa_select_blocks: means rows must be 16-byte aligned");
    sa_kv_layer_view v;
    sa_kv_cache_layer_view(cache, layer, &v);
    SelectArgs a{};
    a.query = query;
    a.dtype = dtype;
    a.batch = batch;
    a.seq_len = seq_len;
    a.heads = v.kv_heads;
    a.group = k->group;
    a.head_dim = v.head_dim;
    a.sm_count = k->sm_count;
    a.pos0 = k->position;
    a.signs = v.signs;
    a.means = means;
    a.row_stride = row_stride;
    a.max_blocks = max_blocks;
    a.sink = sink_blocks;
    a.local = local_blocks;
    a.block_ids = block_ids;
    return launch_select_blocks(a, static_cast<cudaStream_t>(stream));
}

int64_t sa_gqa_sparse_workspace_bytes(const sa_kv_cache *cache, int32_t seq_len) {
    const kv_cache_impl *k = reinterpret_cast<const kv_cache_impl *>(cache);
    // one query token per sequence fits the cache's own workspace, which the decode step uses too
    if (!cache || seq_len <= 1 || !list_decode_format(k)) return 0;
    size_t records, digits;
    list_workspace(k, list_rows_per_launch(k, (int64_t)k->cfg.batch * seq_len), &records, &digits);
    return (int64_t)(records + digits);
}

int sa_gqa_sparse_attend(sa_kv_cache *cache, int32_t layer, const void *query, const int32_t *block_ids,
                         int32_t max_blocks, void *attn_out, int32_t dtype, int32_t batch, int32_t seq_len,
                         int64_t num_heads, int32_t has_scale, float scale, void *workspace, int64_t workspace_bytes,
                         sa_stream_t stream) {
    if (!cache) return set_error(SA_ERR_INVALID_ARGUMENT, "gqa_sparse_attend: NULL cache");
    kv_cache_impl *k = reinterpret_cast<kv_cache_impl *>(cache);
    int rc = check_queries("gqa_sparse_attend", k, layer, dtype, batch, seq_len, num_heads);
    if (rc != SA_OK) return rc;
    if (max_blocks < 1)
        return set_error(SA_ERR_INVALID_ATTRIBUTE, "gqa_sparse_attend: max_blocks must be > 0 (got %d)", max_blocks);
    // tokens along a list are counted in 32 bits; no cache has more blocks
    if (max_blocks > INT32_MAX / SA_BLOCK_TOKENS)
        return set_error(SA_ERR_UNSUPPORTED, "gqa_sparse_attend: lists of %d blocks, at most %d", max_blocks,
                         INT32_MAX / SA_BLOCK_TOKENS);
    if (seq_len == 0) return SA_OK;
    if (!query || !block_ids || !attn_out)
        return set_error(SA_ERR_INVALID_ARGUMENT, "gqa_sparse_attend: NULL query/block_ids/attn_out");
    rc = check_workspace("gqa_sparse_attend", workspace, workspace_bytes,
                         sa_gqa_sparse_workspace_bytes(cache, seq_len));
    if (rc != SA_OK) return rc;
    AttendArgs a = attend_args(k, layer, query, attn_out, dtype, batch, seq_len, has_scale, scale);
    a.block_ids = block_ids;
    a.max_blocks = max_blocks;
    if (!list_decode_format(k)) return launch_gqa_attend_generic(a, static_cast<cudaStream_t>(stream));
    const int64_t rows = (int64_t)batch * seq_len, per = seq_len == 1 ? rows : list_rows_per_launch(k, rows);
    const int64_t row_bytes = (int64_t)a.heads * a.group * a.head_dim * (dtype == SA_DTYPE_FLOAT ? 4 : 2);
    a.list_rows = seq_len;
    a.seq_len = 1;
    if (seq_len > 1) {
        size_t records, digits;
        list_workspace(k, per, &records, &digits);
        a.workspace = static_cast<float *>(workspace);
        a.workspace_floats = records / sizeof(float);
        a.qprep = reinterpret_cast<uint32_t *>(static_cast<char *>(workspace) + records);
    }
    for (int64_t r0 = 0; r0 < rows; r0 += per) {
        a.batch = (int)(rows - r0 < per ? rows - r0 : per);
        a.row0 = (int)r0;
        a.query = static_cast<const char *>(query) + r0 * row_bytes;
        a.out = static_cast<char *>(attn_out) + r0 * row_bytes;
        a.block_ids = block_ids + r0 * a.heads * max_blocks;
        if (a.batch > 65535 || !decode_fast_eligible(a))
            return set_error(SA_ERR_UNSUPPORTED, "gqa_sparse_attend: %d rows of %d blocks in one launch", a.batch,
                             max_blocks);
        rc = launch_gqa_decode_fast(a, nullptr, static_cast<cudaStream_t>(stream));
        if (rc != SA_OK) return rc;
    }
    return SA_OK;
}

}  // extern "C"
