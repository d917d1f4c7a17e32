// Quantize-on-append into pages: RoPE of K, PolarQuant encode (bit-exact with
// sa_kv_append: every operation of polar_encode_warp, in its order and with
// its roundings) and the stores into the pages' records.
//
// A vector is held by four lanes, a warp encodes eight at once.  Lane q holds,
// of every 32 dimensions, the eight from 8q: of the butterfly's stages only two
// (h = 8 and 16) cross lanes, both partners of a rotary pair lie in one lane,
// and the loads of four lanes make whole 64-byte runs.  Beside one warp per
// vector (kv_append.cu) that saves most of the shuffles, reductions and the
// per-vector bookkeeping.
//
// Codes: (y - z)/s rounded half away from zero, the quotient itself rounded to
// f32 first.  t = (y - z) * RN(1/s) is within 3 * 2^-24 * 255 of that quotient,
// so round(t) is the same unless t lies within kTie of a half; a vector with
// such a t (or a scale outside the range where 1/s is safe) is done again by the
// exact quotient.
#include "sa_async.cuh"
#include "sa_append.cuh"
#include "sa_decode_common.cuh"
#include "sa_pages.cuh"

namespace sa {

namespace {

constexpr int kWarps = 4;

// STEP: one new token per row, the warp's vectors are eight consecutive (row, head); else the eight positions of one
// (row, head) that share p >> 3.
template <typename T, int BITS, int D, bool STEP>
__global__ void __launch_bounds__(32 * kWarps) pages_append_kernel(PagesAppendArgs a, uint32_t octs, uint32_t items) {
    constexpr int N = D / 4;            // elements per lane
    constexpr int CH = N / 8;           // runs of eight
    constexpr int CB = D * BITS / 8;
    constexpr int WPC = BITS / 4;       // code words per run
    constexpr uint32_t kLevels = (1u << BITS) - 1u;
    const int lane = threadIdx.x & 31, q = lane & 3, vi = lane >> 2;
    const uint32_t item = blockIdx.x * kWarps + (threadIdx.x >> 5);
    dec::griddep_launch_dependents();
    if (item >= items) return;
    const int which = (int)(item & 1);  // 0 = K, 1 = V
    dec::griddep_wait();  // the inputs, the table and the lengths may come from the kernel before
    int b, h, s;
    int64_t pos;
    bool live;
    int tokens = 0;
    if constexpr (STEP) {
        const uint32_t u = (item >> 1) * 8 + vi;
        live = u < (uint32_t)a.batch * (uint32_t)a.heads;
        b = live ? (int)(u / (uint32_t)a.heads) : 0;
        h = live ? (int)(u - (uint32_t)b * (uint32_t)a.heads) : 0;
        s = 0;
        live = live && row_tokens(a.rows, b, 1, pos) > 0;
        if (!live) pos = 0;
    } else {
        const uint32_t u = item >> 1, bh = u / octs, oct = u - bh * octs;
        b = (int)(bh / (uint32_t)a.heads);
        h = (int)(bh - (uint32_t)b * (uint32_t)a.heads);
        int64_t pos0;
        tokens = row_tokens(a.rows, b, a.seq_len, pos0);
        pos = (pos0 & ~(int64_t)7) + (int64_t)oct * 8 + vi;
        live = pos >= pos0 && pos < pos0 + tokens;
        s = (int)(pos - pos0);
    }
    // the vector's place
    uint8_t *rec = nullptr;
    if (live) {
        const int64_t j = pos / kPageTokens;
        int page = -1;
        if (j < a.rows.max_pages) page = a.rows.table[b * a.rows.table_stride + j];
        if (page < 0 || page >= a.rows.num_pages) {
            if (q == 0) atomicOr(a.rows.dev_status, kPagesBadPage);
            live = false;
        } else if (a.rope.on && pos >= a.rope.rows) {
            if (q == 0) atomicOr(a.rows.dev_status, kPagesBadPosition);
            live = false;
        } else {
            rec = a.records + ((int64_t)page * a.heads + h) * page_record(CB);
        }
    }
    if (!__any_sync(0xffffffffu, live)) return;

    float x[N];
    if (live) {
        const T *src = static_cast<const T *>(which ? a.value : a.key) + b * a.batch_stride + s * a.token_stride +
                       (int64_t)h * D + 8 * q;
#pragma unroll
        for (int c = 0; c < CH; c++) load_run<T, 8>(src + 32 * c, a.aligned, x + 8 * c);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = 0.0f;
    }
    if (which == 0 && a.rope.on) {  // warp-uniform
        const float *cs = a.rope.cos_cache + (live ? pos : 0) * (D / 2), *sn = a.rope.sin_cache + (live ? pos : 0) * (D / 2);
        if (a.rope.interleaved) {
#pragma unroll
            for (int c = 0; c < CH; c++) {
                const int p0 = 16 * c + 4 * q;  // pairs of this run
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float co = cs[p0 + i], si = sn[p0 + i], x0 = x[8 * c + 2 * i], x1 = x[8 * c + 2 * i + 1];
                    x[8 * c + 2 * i] = __fsub_rn(__fmul_rn(co, x0), __fmul_rn(si, x1));
                    x[8 * c + 2 * i + 1] = __fadd_rn(__fmul_rn(si, x0), __fmul_rn(co, x1));
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < CH / 2; c++) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int p = 32 * c + 8 * q + i;
                    const float co = cs[p], si = sn[p], x0 = x[8 * c + i], x1 = x[8 * (c + CH / 2) + i];
                    x[8 * c + i] = __fsub_rn(__fmul_rn(co, x0), __fmul_rn(si, x1));
                    x[8 * (c + CH / 2) + i] = __fadd_rn(__fmul_rn(si, x0), __fmul_rn(co, x1));
                }
            }
        }
    }
    {
        const float *sg = a.signs + (int64_t)h * D + 8 * q;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) x[8 * c + i] = __fmul_rn(x[8 * c + i], sg[32 * c + i]);
    }
    // butterfly stages h = 1, 2, 4 (in a run), 8, 16 (across lanes), 32, 64 (between runs)
#pragma unroll
    for (int hs = 1; hs < 8; hs <<= 1)
#pragma unroll
        for (int i = 0; i < N; i++)
            if ((i & hs) == 0) {
                const float p0 = x[i], p1 = x[i + hs];
                x[i] = __fadd_rn(p0, p1);
                x[i + hs] = __fsub_rn(p0, p1);
            }
#pragma unroll
    for (int lm = 1; lm < 4; lm <<= 1) {
        // upper lane: other - x, lower lane: x + other = other - (-x), exactly
        const uint32_t flip = (lane & lm) ? 0u : 0x80000000u;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float other = __shfl_xor_sync(0xffffffffu, x[i], lm);
            x[i] = __fsub_rn(other, __uint_as_float(__float_as_uint(x[i]) ^ flip));
        }
    }
#pragma unroll
    for (int hs = 8; hs < N; hs <<= 1)
#pragma unroll
        for (int i = 0; i < N; i++)
            if ((i & hs) == 0) {
                const float p0 = x[i], p1 = x[i + hs];
                x[i] = __fadd_rn(p0, p1);
                x[i + hs] = __fsub_rn(p0, p1);
            }
    float mn = INFINITY, mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; i++) {
        x[i] = __fmul_rn(x[i], a.wht_scale);
        mn = fminf(mn, x[i]);
        mx = fmaxf(mx, x[i]);
    }
#pragma unroll
    for (int lm = 1; lm < 4; lm <<= 1) {
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, lm));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, lm));
    }
    if (__any_sync(0xffffffffu, mn == 0.0f)) {
        // a minimum of zero has the sign of its first occurrence
        int first = 0x7fffffff;
#pragma unroll
        for (int i = N - 1; i >= 0; i--)
            if (x[i] == 0.0f) first = 2 * ((i >> 3) * 32 + 8 * q + (i & 7)) + (__float_as_int(x[i]) < 0);
#pragma unroll
        for (int lm = 1; lm < 4; lm <<= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, lm));
        if (mn == 0.0f) mn = (first & 1) ? -0.0f : 0.0f;
    }
    const float range = __fsub_rn(mx, mn);
    const float sc = range > 0.0f ? __fdiv_rn(range, (float)kLevels) : 1.0f;
    constexpr float kTie = BITS == 4 ? 0.5f - 0x1p-17f : 0.5f - 0x1p-13f;
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: a sum with it is rounded to whole numbers
    // (a vector of NaN leaves the minimum above the maximum, one with infinities an infinite one of them)
    const bool safe = sc >= 0x1p-90f && sc <= 0x1p100f && mn <= mx && fabsf(mn) < INFINITY && mx < INFINITY;
    uint32_t word[CH * WPC];
    {
        const float rcp = safe ? __frcp_rn(sc) : 1.0f;
        float far = 0.0f;
#pragma unroll
        for (int w = 0; w < CH * WPC; w++) {
            constexpr int kPer = 32 / BITS;  // codes per word
            uint32_t acc = 0;
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                const float num = __fsub_rn(x[w * kPer + i], mn);
                const float k = __fmaf_rn(num, rcp, kMagic);
                far = fmaxf(far, fabsf(__fmaf_rn(num, rcp, -__fsub_rn(k, kMagic))));
                // the code sits in the low bits of k; the exponent's bits cancel in the constant below
                acc += (__float_as_uint(k) - 0x4B400000u) << (BITS * i);
            }
            word[w] = acc;
        }
        const bool redo = !safe || !(far < kTie);
        if (__any_sync(0xffffffffu, redo) && redo) {
#pragma unroll
            for (int w = 0; w < CH * WPC; w++) {
                constexpr int kPer = 32 / BITS;
                uint32_t acc = 0;
#pragma unroll
                for (int i = 0; i < kPer; i++) {
                    const float num = __fsub_rn(x[w * kPer + i], mn);
                    uint32_t c = sc > 0.0f ? __float2uint_rz(rust_round_f32(__fdiv_rn(num, sc))) : 0u;
                    acc |= min(c, kLevels) << (BITS * i);
                }
                word[w] = acc;
            }
        }
    }

    // stores: word w of run c holds code bytes 4*j0 .. of the vector, j0 = (c*4 + q)*WPC + w
    const int t = (int)(pos & (kPageTokens - 1));
    if (live && q == 0)
        *reinterpret_cast<float2 *>(rec + (which ? page_v_meta(CB) : page_k_meta(CB)) + t * 8) = make_float2(sc, mn);
    if (which == 0) {
        if (live) {
            uint32_t *dst = reinterpret_cast<uint32_t *>(rec + t * CB);
#pragma unroll
            for (int c = 0; c < CH; c++) {
                if constexpr (WPC == 2)
                    reinterpret_cast<uint2 *>(dst)[c * 4 + q] = make_uint2(word[2 * c], word[2 * c + 1]);
                else
                    dst[c * 4 + q] = word[c];
            }
        }
        return;
    }
    // V: the bytes of four tokens interleave (v_byte_offset); word k of a 16-byte chunk holds byte k of the
    // four tokens' words.  A full quad transposes its words between its lanes.
    uint8_t *vdst = rec + page_v_codes(CB) + (t >> 4) * (16 * CB) + ((t >> 2) & 3) * 16;
    const unsigned alive = __ballot_sync(0xffffffffu, live);
    const bool full = !STEP && ((alive >> (lane & 16)) & 0xffffu) == 0xffffu;
    if constexpr (!STEP) {
        const int tt = vi & 3;
        const uint32_t s1 = (tt & 1) ? 0x3715u : 0x6240u, s2 = (tt & 2) ? 0x3276u : 0x5410u;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int w = 0; w < WPC; w++) {
                uint32_t v = word[c * WPC + w];
                v = __byte_perm(v, __shfl_xor_sync(0xffffffffu, v, 4), s1);
                v = __byte_perm(v, __shfl_xor_sync(0xffffffffu, v, 8), s2);
                if (full) *reinterpret_cast<uint32_t *>(vdst + ((c * 4 + q) * WPC + w) * 64 + tt * 4) = v;
            }
    }
    if (live && !full) {
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int w = 0; w < WPC; w++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    vdst[((c * 4 + q) * WPC + w) * 64 + k * 4 + (t & 3)] =
                        (uint8_t)(word[c * WPC + w] >> (8 * k));
    }
}

template <typename T, int BITS, int D>
int launch_shape(const PagesAppendArgs &a, cudaStream_t stream) {
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(32 * kWarps);
    cfg.stream = stream;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    const int64_t bh = (int64_t)a.batch * a.heads;
    // the new tokens of a row touch one run of eight positions more than they fill, wherever they begin
    const int64_t octs = a.seq_len == 1 ? 1 : (a.seq_len + 7) / 8 + 1;
    const int64_t items = 2 * (a.seq_len == 1 ? (bh + 7) / 8 : bh * octs);
    if (items > (int64_t)1 << 31) return set_error(SA_ERR_UNSUPPORTED, "kv_pages_append: too many vectors");
    cfg.gridDim = dim3((unsigned)((items + kWarps - 1) / kWarps));
    const int rc =
        a.seq_len == 1
            ? check_cuda(cudaLaunchKernelEx(&cfg, pages_append_kernel<T, BITS, D, true>, a, (uint32_t)octs, (uint32_t)items),
                         "kv_pages_append launch")
            : check_cuda(cudaLaunchKernelEx(&cfg, pages_append_kernel<T, BITS, D, false>, a, (uint32_t)octs, (uint32_t)items),
                         "kv_pages_append launch");
    count_launch();
    return rc;
}

template <typename T>
int launch_t(const PagesAppendArgs &a, cudaStream_t stream) {
    if (a.bits == 4) return a.head_dim == 128 ? launch_shape<T, 4, 128>(a, stream) : launch_shape<T, 4, 64>(a, stream);
    return a.head_dim == 128 ? launch_shape<T, 8, 128>(a, stream) : launch_shape<T, 8, 64>(a, stream);
}

}  // namespace

int launch_pages_append(const PagesAppendArgs &a, cudaStream_t stream) {
    switch (a.dtype) {
        case SA_DTYPE_FLOAT: return launch_t<float>(a, stream);
        case SA_DTYPE_FLOAT16: return launch_t<__half>(a, stream);
        default: return launch_t<__nv_bfloat16>(a, stream);
    }
}

}  // namespace sa
