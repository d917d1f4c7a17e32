// Keeping the accepted path of a draft tree: in every layer, the rows of the
// accepted drafts (codes, scale, zero point and QJL residual of K and V) move
// to the first slots after the prefix.
//
// One CTA per (layer, batch row, KV head) reads before it writes, so a path may
// name its rows in any order.  K rows move as 16-byte pieces.  A token's V bytes
// lie 4 apart among those of its neighbours (16-token blocks), so the drafts' V
// blocks are read whole -- their addresses do not depend on the path, and row by
// row each byte would cost a 4-byte access and each row half the sectors of its
// block -- and a thread puts together a 16-byte piece (four code bytes of four
// tokens) from the four pieces that hold its tokens by twelve byte permutations.
// Bound by latency, two dependent loads per unit: 16 layers, 64 sequences, 8 heads,
// 11 of 48 int4 drafts (52 MB read, 18 MB written) in 20 us; moving the V bytes one
// by one through shared memory took 29.
#include "sa_common.cuh"
#include "sa_internal.h"

namespace sa {

namespace {

// Two warps per unit: many units in flight, several loads of a thread under way at once.
constexpr int kKeepThreads = 64;

// Shared memory: the drafts' V blocks, the kept K rows, metadata and QJL residuals.
__host__ __device__ __forceinline__ int keep_blocks(int64_t pos0, int drafted) {
    return (int)(((pos0 + drafted - 1) >> 4) - (pos0 >> 4)) + 1;
}
__host__ __device__ __forceinline__ size_t keep_smem(int64_t pos0, int drafted, int n, int cb, int qb) {
    return (size_t)keep_blocks(pos0, drafted) * 16 * cb + (size_t)n * (cb + 16 + (qb ? 2 * qb + 8 : 0));
}

// U: the widest aligned access of the K rows; 2^piece_bits of them cover a row.
template <typename U>
__global__ void __launch_bounds__(kKeepThreads) keep_drafts_kernel(KeepArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int s_path[kMaxDraftNodes];
    const int tid = threadIdx.x;
    const int64_t unit = blockIdx.x;  // (layer * batch + b) * heads + h
    const int b = (int)(unit / a.heads % a.batch);
    const int cb = a.code_bytes, n = a.n, qb = a.k_qjl_bits ? a.head_dim / 8 : 0;
    const int64_t pos0 = a.pos0, row0 = unit * a.capacity;
    const int nblk = keep_blocks(pos0, a.drafted);
    uint8_t *kc = a.k_codes + row0 * cb;
    uint4 *vblk = reinterpret_cast<uint4 *>(a.v_codes + row0 * cb + (pos0 >> 4) * (16 * cb));
    float2 *km = reinterpret_cast<float2 *>(a.k_meta) + row0, *vm = reinterpret_cast<float2 *>(a.v_meta) + row0;
    uint8_t *kq = qb ? a.k_qjl_bits + row0 * qb : nullptr, *vq = qb ? a.v_qjl_bits + row0 * qb : nullptr;
    float *kg = qb ? a.k_qjl_mag + row0 : nullptr, *vg = qb ? a.v_qjl_mag + row0 : nullptr;
    uint4 *s_blk = reinterpret_cast<uint4 *>(smem);
    float2 *s_meta = reinterpret_cast<float2 *>(smem + nblk * 16 * cb);  // K, then V
    uint8_t *s_k = reinterpret_cast<uint8_t *>(s_meta + 2 * n);
    float *s_mag = reinterpret_cast<float *>(s_k + n * cb);
    uint8_t *s_kq = reinterpret_cast<uint8_t *>(s_mag + (qb ? 2 * n : 0)), *s_vq = s_kq + n * qb;

    for (int i = tid; i < n; i += kKeepThreads) {
        const int p = a.path[(int64_t)b * n + i];
        const bool ok = p >= 0 && p < a.drafted;
        if (!ok) atomicOr(a.dev_status, 2);
        s_path[i] = ok ? p : i;
    }
#pragma unroll 4
    for (int i = tid; i < nblk * cb; i += kKeepThreads) s_blk[i] = vblk[i];
    __syncthreads();
    // x counts the pieces of the rows, a row's number of them rounded up to a power of two
    const int np = cb / (int)sizeof(U), off = (int)(pos0 & 15);
#pragma unroll 4
    for (int x = tid; x < n << a.piece_bits; x += kKeepThreads) {
        const int i = x >> a.piece_bits, j = x & ((1 << a.piece_bits) - 1);
        if (j < np) reinterpret_cast<U *>(s_k)[i * np + j] = reinterpret_cast<const U *>(kc)[(pos0 + s_path[i]) * np + j];
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
#pragma unroll 4
    for (int x = tid; x < n << a.piece_bits; x += kKeepThreads) {
        const int i = x >> a.piece_bits, j = x & ((1 << a.piece_bits) - 1);
        if (j < np) reinterpret_cast<U *>(kc)[(pos0 + i) * np + j] = reinterpret_cast<const U *>(s_k)[i * np + j];
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
    // piece i: code bytes c .. c + 3 of token group i % 4 of block i / cb (a block has cb pieces)
    for (int i = tid; i < keep_blocks(pos0, n) * cb; i += kKeepThreads) {
        const int blk = i / cb, c = (i - blk * cb) & ~3;
        const int t0 = blk * 16 + (i & 3) * 4 - off;  // the group's first token, from the first draft
        if (t0 + 3 < 0 || t0 >= n) continue;
        uint4 w[4];
        uint32_t at[4];
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const int t = t0 + y, from = off + (t >= 0 && t < n ? s_path[t] : t);  // (neighbours stay)
            w[y] = s_blk[(from >> 4) * cb + c + ((from >> 2) & 3)];
            at[y] = from & 3;
        }
        const uint32_t s01 = at[0] | (4 + at[1]) << 4, s23 = at[2] | (4 + at[3]) << 4;
        auto word = [&](uint32_t p, uint32_t q, uint32_t r, uint32_t s) {
            return __byte_perm(__byte_perm(p, q, s01), __byte_perm(r, s, s23), 0x5410);
        };
        vblk[i] = make_uint4(word(w[0].x, w[1].x, w[2].x, w[3].x), word(w[0].y, w[1].y, w[2].y, w[3].y),
                             word(w[0].z, w[1].z, w[2].z, w[3].z), word(w[0].w, w[1].w, w[2].w, w[3].w));
    }
}

}  // namespace

int launch_keep_drafts(const KeepArgs &a, cudaStream_t stream) {
    const int64_t units = (int64_t)a.layers * a.batch * a.heads;
    if (units > 0x7fffffff)
        return set_error(SA_ERR_UNSUPPORTED, "kv_cache_keep_drafts: %lld units", (long long)units);
    const int qb = a.k_qjl_bits ? a.head_dim / 8 : 0;
    // at most 42.5 KB (64 drafts over five V blocks, head_dim 256, 8 bits, QJL): no attribute needed
    const size_t smem = keep_smem(a.pos0, a.drafted, a.n, a.code_bytes, qb);
    KeepArgs k = a;
    const bool wide = a.code_bytes % 16 == 0;
    while (((wide ? 16 : 4) << k.piece_bits) < a.code_bytes) k.piece_bits++;
    auto kern = wide ? keep_drafts_kernel<uint4> : keep_drafts_kernel<uint32_t>;
    kern<<<(unsigned)units, kKeepThreads, smem, stream>>>(k);
    count_launch();
    return check_cuda(cudaGetLastError(), "kv_cache_keep_drafts launch");
}

}  // namespace sa
