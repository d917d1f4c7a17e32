// Keeping the accepted path of a draft tree: in every layer, the rows of the
// accepted drafts (codes, scale, zero point and QJL residual of K and V) move
// to the first slots after the prefix.
//
// One CTA per (layer, batch row, KV head) reads the n rows into shared memory,
// then writes them, so a path may name its rows in any order.  A thread keeps
// its byte (V: bytes of a token lie 4 apart) or word (K) of the row and steps
// over the rows, so an element costs one load, one store and no division.
// Bound by the latency of its two round trips to L2 and HBM.
#include "sa_common.cuh"
#include "sa_internal.h"

namespace sa {

namespace {

constexpr int kKeepThreads = 256;

// Bytes of shared memory per row: K and V codes, their scale and zero point, and the QJL residuals.
__host__ __device__ __forceinline__ int keep_row_bytes(int cb, int qb) { return 2 * cb + 16 + (qb ? 2 * qb + 8 : 0); }

// a.bytes, a.words: the row's code bytes and words, up to a power of two (at most 256).
__global__ void __launch_bounds__(kKeepThreads) keep_drafts_kernel(KeepArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int s_path[kMaxDraftNodes];
    const int tid = threadIdx.x;
    const int64_t unit = blockIdx.x;  // (layer * batch + b) * heads + h
    const int b = (int)(unit / a.heads % a.batch);
    const int cb = a.code_bytes, n = a.n, qb = a.k_qjl_bits ? a.head_dim / 8 : 0;
    if (tid < n) {
        const int p = a.path[(int64_t)b * n + tid];
        const bool ok = p >= 0 && p < a.drafted;
        if (!ok) atomicOr(a.dev_status, 2);
        s_path[tid] = ok ? p : tid;
    }
    __syncthreads();
    const int64_t row0 = unit * a.capacity;
    uint8_t *kc = a.k_codes + row0 * cb, *vc = a.v_codes + row0 * cb;
    float2 *km = reinterpret_cast<float2 *>(a.k_meta) + row0, *vm = reinterpret_cast<float2 *>(a.v_meta) + row0;
    uint8_t *kq = qb ? a.k_qjl_bits + row0 * qb : nullptr, *vq = qb ? a.v_qjl_bits + row0 * qb : nullptr;
    float *kg = qb ? a.k_qjl_mag + row0 : nullptr, *vg = qb ? a.v_qjl_mag + row0 : nullptr;
    // shared arrays, [n] rows each
    float2 *s_meta = reinterpret_cast<float2 *>(smem);  // K, then V
    float *s_mag = reinterpret_cast<float *>(s_meta + 2 * n);
    uint8_t *s_k = reinterpret_cast<uint8_t *>(s_mag + (qb ? 2 * n : 0));
    uint8_t *s_v = s_k + n * cb, *s_kq = s_v + n * cb, *s_vq = s_kq + n * qb;
    const int64_t pos0 = a.pos0;
    // K: word jw of row i; V: byte jv of row i
    const int cw = cb / 4, jw = tid & (a.words - 1), jv = tid & (a.bytes - 1);
    const int iw = tid / a.words, iv = tid / a.bytes, dw = kKeepThreads / a.words, dv = kKeepThreads / a.bytes;
    const uint32_t *kw = reinterpret_cast<const uint32_t *>(kc);
    uint32_t *s_kw = reinterpret_cast<uint32_t *>(s_k);
    const int64_t vat = (jv >> 2) * 64 + (jv & 3) * 4;  // of byte jv within a 16-token block
    auto v_row = [&](int64_t t) { return (t >> 4) * (16 * cb) + ((t >> 2) & 3) * 16 + (t & 3) + vat; };
    if (jw < cw) {
#pragma unroll 4
        for (int i = iw; i < n; i += dw) s_kw[i * cw + jw] = kw[(pos0 + s_path[i]) * cw + jw];
    }
    if (jv < cb) {
#pragma unroll 4
        for (int i = iv; i < n; i += dv) s_v[i * cb + jv] = vc[v_row(pos0 + s_path[i])];
    }
    for (int i = tid; i < n; i += kKeepThreads) {
        const int64_t t = pos0 + s_path[i];
        s_meta[i] = km[t];
        s_meta[n + i] = vm[t];
        if (qb) {
            s_mag[i] = kg[t];
            s_mag[n + i] = vg[t];
        }
    }
    for (int i = tid; i < n * qb; i += kKeepThreads) {
        const int64_t t = pos0 + s_path[i / qb];
        s_kq[i] = kq[t * qb + i % qb];
        s_vq[i] = vq[t * qb + i % qb];
    }
    __syncthreads();
    if (jw < cw) {
#pragma unroll 4
        for (int i = iw; i < n; i += dw) reinterpret_cast<uint32_t *>(kc)[(pos0 + i) * cw + jw] = s_kw[i * cw + jw];
    }
    if (jv < cb) {
#pragma unroll 4
        for (int i = iv; i < n; i += dv) vc[v_row(pos0 + i)] = s_v[i * cb + jv];
    }
    for (int i = tid; i < n; i += kKeepThreads) {
        const int64_t t = pos0 + i;
        km[t] = s_meta[i];
        vm[t] = s_meta[n + i];
        if (qb) {
            kg[t] = s_mag[i];
            vg[t] = s_mag[n + i];
        }
    }
    for (int i = tid; i < n * qb; i += kKeepThreads) {
        const int64_t t = pos0 + i / qb;
        kq[t * qb + i % qb] = s_kq[i];
        vq[t * qb + i % qb] = s_vq[i];
    }
}

}  // namespace

int launch_keep_drafts(const KeepArgs &a, cudaStream_t stream) {
    const int64_t units = (int64_t)a.layers * a.batch * a.heads;
    if (units > 0x7fffffff)
        return set_error(SA_ERR_UNSUPPORTED, "kv_cache_keep_drafts: %lld units", (long long)units);
    // at most 64 rows of 2 * 256 code bytes and 88 others: 38400 bytes, below the default limit
    const size_t smem = (size_t)a.n * keep_row_bytes(a.code_bytes, a.k_qjl_bits ? a.head_dim / 8 : 0);
    KeepArgs k = a;
    for (k.bytes = 4; k.bytes < a.code_bytes;) k.bytes *= 2;
    k.words = k.bytes / 4;
    keep_drafts_kernel<<<(unsigned)units, kKeepThreads, smem, stream>>>(k);
    count_launch();
    return check_cuda(cudaGetLastError(), "kv_cache_keep_drafts launch");
}

}  // namespace sa
