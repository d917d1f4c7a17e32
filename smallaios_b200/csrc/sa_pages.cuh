// The page pool's structures and device helpers shared by its kernels: the
// record layout, the rows of a call, and the Walsh-Hadamard and rotary steps
// of vectors that four lanes hold.
#pragma once

#include "sa_common.cuh"
#include "sa_internal.h"

namespace sa {

constexpr int kPageTokens = SA_PAGE_TOKENS;

// Status bits of sa_kv_pages_device_status.
constexpr int kPagesTimeout = 1, kPagesBadPage = 2, kPagesBadPosition = 4, kPagesBadBeam = 8;

// Offsets in the record of a (page, KV head): K codes, K metadata, V metadata, V codes.
__host__ __device__ constexpr int page_k_meta(int cb) { return kPageTokens * cb; }
__host__ __device__ constexpr int page_v_meta(int cb) { return kPageTokens * (cb + 8); }
__host__ __device__ constexpr int page_v_codes(int cb) { return kPageTokens * (cb + 16); }
__host__ __device__ constexpr int page_record(int cb) { return kPageTokens * (2 * cb + 16); }

struct kv_pages_impl {
    sa_kv_pages_config cfg;
    int device;
    int sm_count;
    int code_bytes;
    int group;  // num_heads / num_kv_heads
    float wht_scale;
    int full;   // 24 bits of queries and weights for f16 and bf16 callers too
    void *base;
    uint8_t *records;  // [L][P][H][record]
    float *signs;      // [L][H][D]
    int *dev_status;
    size_t layer_bytes;  // P*H*record
};

// Rows of a call: the sequences' pages and lengths.
struct PageRows {
    const int32_t *table;
    int64_t table_stride;
    int max_pages;
    const int32_t *lens;
    const int32_t *counts;  // nullptr: every row has all new tokens
    int num_pages;
    int *dev_status;
};

struct RopeArgs {
    const float *cos_cache, *sin_cache;
    int rows, on, interleaved;
    int aligned;  // both tables begin on 16 bytes
};

struct PagesAppendArgs {
    const void *key, *value;
    int64_t batch_stride, token_stride;
    int aligned;  // every vector starts on 16 bytes
    int dtype, batch, seq_len, heads, head_dim, bits;
    uint8_t *records;  // of the layer
    const float *signs;
    float wht_scale;
    PageRows rows;
    RopeArgs rope;
};

struct PagesAttendArgs {
    const void *query;
    int64_t batch_stride, token_stride;
    void *out;
    int dtype, batch, seq_len, heads, group, head_dim, bits, full;
    const uint8_t *records;
    const float *signs;
    float wht_scale, scale;
    int sm_count;
    PageRows rows;
    RopeArgs rope;
};

// Beam selection (sa_beam_select).
struct BeamArgs {
    const void *logits;
    int64_t row_stride;
    int dtype, batch, beams, keep, end_token;
    int vocab;
    const float *scores;
    const uint8_t *finished;  // nullptr: none
    int32_t *parents, *tokens;
    float *out_scores;
};

// Beams over pages (sa_kv_pages_reorder).
struct ReorderArgs {
    uint8_t *records;  // [L][P][H][record]
    size_t layer_bytes;
    int layers, heads, code_bytes;
    const int32_t *table;
    int64_t table_stride;
    int32_t *out;
    int64_t out_stride;
    int max_pages;
    const int32_t *lens, *parents;
    int batch, beams;
    int num_pages;
    int *dev_status;
};

int64_t beam_select_workspace(int64_t rows, int64_t vocab);
int launch_beam_select(const BeamArgs &a, void *workspace, cudaStream_t stream);
int launch_pages_reorder(const ReorderArgs &a, cudaStream_t stream);
int launch_pages_append(const PagesAppendArgs &a, cudaStream_t stream);
size_t pages_attend_workspace(const kv_pages_impl *k, int batch, int seq_len, int dtype);
int launch_pages_attend(const PagesAttendArgs &a, void *workspace, cudaStream_t stream);

// New tokens of row b, and the position of its first one; 0 tokens for a row that takes no part.
__device__ __forceinline__ int row_tokens(const PageRows &r, int b, int seq_len, int64_t &pos0) {
    const int len = __ldcg(r.lens + b);
    pos0 = len;
    if (len < 0) return 0;
    if (!r.counts) return seq_len;
    const int n = __ldcg(r.counts + b);
    return n < 0 ? 0 : (n < seq_len ? n : seq_len);
}

// Pairs of floats: two operations to an instruction.  (A product and a sum of its result may be contracted.)
using f2 = unsigned long long;
__device__ __forceinline__ f2 pair(float x, float y) {
    f2 v;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ void split(f2 v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ f2 add2(f2 x, f2 y) {
    f2 v;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(v) : "l"(x), "l"(y));
    return v;
}
__device__ __forceinline__ f2 mul2(f2 x, f2 y) {
    f2 v;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(v) : "l"(x), "l"(y));
    return v;
}
__device__ __forceinline__ f2 fma2(f2 x, f2 y, f2 z) {
    f2 v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(v) : "l"(x), "l"(y), "l"(z));
    return v;
}
// x - y (a product with -1 is exact).
__device__ __forceinline__ f2 sub2(f2 x, f2 y) { return fma2(y, pair(-1.0f, -1.0f), x); }

// N consecutive elements as f32, 16 bytes at a time when `aligned`.
template <typename T, int N>
__device__ __forceinline__ void load_run(const T *p, bool aligned, float *x) {
    constexpr int kPer = 16 / (int)sizeof(T);
    static_assert(N % kPer == 0, "whole 16-byte pieces");
    if (aligned) {
#pragma unroll
        for (int i = 0; i < N / kPer; i++) {
            union {
                uint4 v;
                T t[kPer];
            } u;
            u.v = reinterpret_cast<const uint4 *>(p)[i];
#pragma unroll
            for (int j = 0; j < kPer; j++) x[i * kPer + j] = DT<T>::to_f32(u.t[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = ld_f32(p + i);
    }
}

}  // namespace sa
