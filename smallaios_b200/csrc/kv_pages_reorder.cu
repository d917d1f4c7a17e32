// Reordering the states of beams: the new page table, and copies of the pages
// in use that more than one beam goes on filling.
//
// In a group of K beams each one owns its page in use, so as many beams have to
// take another page as beams end: the further children of a parent take the pages
// of the beams without children.  No such page is read, no page that is read is
// written, so every CTA works out the same matching and copies its part without
// waiting for another.  One launch, a CTA per (KV head, group, layer); only the
// rows in use move, 2 * rows * (2 CB + 16) bytes per copy and head.  16 groups of 8 beams, 8 layers, 45 rows in use,
// three copies a group: 12 us for 40 MB, latency of the lookups (lengths, parents, pages) and of loads that wait for
// their stores; four loads of a thread at once and twice the threads made no difference.
#include "sa_decode_common.cuh"
#include "sa_pages.cuh"

namespace sa {

namespace {

constexpr int kReorderThreads = 128;

__global__ void __launch_bounds__(kReorderThreads) pages_reorder_kernel(ReorderArgs a) {
    __shared__ int s_from[SA_MAX_BEAMS];          // slot whose full pages a slot takes
    __shared__ int s_own[SA_MAX_BEAMS];           // slot whose page in use it takes
    __shared__ int s_src[SA_MAX_BEAMS], s_dst[SA_MAX_BEAMS];  // pages of the copies
    __shared__ int s_copies, s_len;
    const int tid = threadIdx.x, h = blockIdx.x, b = blockIdx.y, layer = blockIdx.z;
    const int K = a.beams;
    const int32_t *table = a.table + (int64_t)b * K * a.table_stride;
    dec::griddep_launch_dependents();
    dec::griddep_wait();
    if (tid < 32) {
        const unsigned all = K == 32 ? 0xffffffffu : (1u << K) - 1u;
        const bool on = tid < K;
        const int len = on ? a.lens[(int64_t)b * K + tid] : 0;
        const int len0 = __shfl_sync(0xffffffffu, len, 0);
        int p = on ? a.parents[(int64_t)b * K + tid] : tid;
        const bool stray = on && (p < -1 || p >= K);
        if (p < 0 || p >= K) p = tid;
        const bool uneven = __any_sync(0xffffffffu, on && len != len0);
        const bool past = len0 > 0 && (int64_t)len0 > (int64_t)a.max_pages * kPageTokens;
        const bool moves = !uneven && !past && len0 > 0;  // else the group stays as it is
        if (!moves) p = tid;
        const unsigned same = __match_any_sync(0xffffffffu, on ? p : 64 + tid);
        const int heir = ((same >> p) & 1u) ? p : __ffs(same) - 1;  // bit p: slot p continues itself
        const bool takes = on && heir != tid;
        const unsigned takers = __ballot_sync(0xffffffffu, takes);
        const unsigned alive = __reduce_or_sync(0xffffffffu, on ? 1u << p : 0u);
        const unsigned ended = all & ~alive;
        int own = p;
        if (takes) own = __fns(ended, 0, __popc(takers & ((1u << tid) - 1u)) + 1);
        const int cur = moves ? len0 / kPageTokens : 0, fill = moves ? len0 % kPageTokens : 0;
        if (fill == 0) own = tid;
        int src = -1, dst = -1;
        bool copy = takes && fill > 0;
        if (copy) {
            src = table[p * a.table_stride + cur];
            dst = table[own * a.table_stride + cur];
            if (src < 0 || src >= a.num_pages || dst < 0 || dst >= a.num_pages) {
                copy = false;
                if (h == 0 && layer == 0) atomicOr(a.dev_status, kPagesBadPage);
            }
        }
        const unsigned copies = __ballot_sync(0xffffffffu, copy);
        if (copy) {
            const int at = __popc(copies & ((1u << tid) - 1u));
            s_src[at] = src;
            s_dst[at] = dst;
        }
        s_from[tid] = p;
        s_own[tid] = own;
        if (tid == 0) {
            s_copies = __popc(copies);
            s_len = moves ? len0 : 0;
        }
        if (h == 0 && layer == 0) {
            if (__any_sync(0xffffffffu, stray) || uneven) {
                if (tid == 0) atomicOr(a.dev_status, kPagesBadBeam);
            }
            if (past && tid == 0) atomicOr(a.dev_status, kPagesBadPage);
        }
    }
    __syncthreads();
    const int cur = s_len / kPageTokens, fill = s_len % kPageTokens;
    if (layer == 0) {  // the heads share the table's columns
        int32_t *out = a.out + (int64_t)b * K * a.out_stride;
        for (int j = h * kReorderThreads + tid; j < a.max_pages; j += a.heads * kReorderThreads)
            for (int k = 0; k < K; k++) {
                const int from = j < cur ? s_from[k] : j == cur ? s_own[k] : k;
                out[k * a.out_stride + j] = table[from * a.table_stride + j];
            }
    }
    const int copies = s_copies, cb = a.code_bytes;
    if (copies == 0) return;
    uint8_t *base = a.records + (size_t)layer * a.layer_bytes;
    // pieces of a record: K codes in 16 bytes, K and V metadata in 8, V codes as 16-byte pieces of four tokens' bytes
    const int kp = fill * cb / 16, vb = (fill + 15) / 16 * cb;  // cb 16-byte pieces per 16 tokens of V
    const int total = kp + 2 * fill + vb;
    for (int i = tid; i < copies * total; i += kReorderThreads) {
        const int c = i / total, x = i - c * total;
        const uint8_t *src = base + ((int64_t)s_src[c] * a.heads + h) * page_record(cb);
        uint8_t *dst = base + ((int64_t)s_dst[c] * a.heads + h) * page_record(cb);
        if (x < kp) {
            reinterpret_cast<uint4 *>(dst)[x] = reinterpret_cast<const uint4 *>(src)[x];
        } else if (x < kp + 2 * fill) {
            const int m = x - kp, off = m < fill ? page_k_meta(cb) + 8 * m : page_v_meta(cb) + 8 * (m - fill);
            *reinterpret_cast<float2 *>(dst + off) = *reinterpret_cast<const float2 *>(src + off);
        } else {
            const int y = x - kp - 2 * fill;
            const int left = fill - (y / cb * 16 + (y & 3) * 4);  // tokens in use from the piece's first one on
            const int off = page_v_codes(cb) + 16 * y;
            uint4 v = *reinterpret_cast<const uint4 *>(src + off);
            if (left <= 0) continue;
            if (left < 4) {
                const uint32_t mask = (1u << (8 * left)) - 1u;
                const uint4 o = *reinterpret_cast<const uint4 *>(dst + off);
                v = make_uint4((v.x & mask) | (o.x & ~mask), (v.y & mask) | (o.y & ~mask), (v.z & mask) | (o.z & ~mask),
                               (v.w & mask) | (o.w & ~mask));
            }
            *reinterpret_cast<uint4 *>(dst + off) = v;
        }
    }
}

}  // namespace

int launch_pages_reorder(const ReorderArgs &a, cudaStream_t stream) {
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.heads, a.batch, a.layers);
    cfg.blockDim = dim3(kReorderThreads);
    cfg.stream = stream;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    const int rc = check_cuda(cudaLaunchKernelEx(&cfg, pages_reorder_kernel, a), "kv_pages_reorder launch");
    count_launch();
    return rc;
}

}  // namespace sa
