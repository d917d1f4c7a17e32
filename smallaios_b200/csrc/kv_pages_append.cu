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
// Sums and differences are taken in pairs (f2).  A product that a sum follows is not: a product of a pair may be
// contracted with the sum to one rounding, __fmul_rn never is.  (Products with signs are exact either way.)
//
// Eight ragged prompts of up to 2048 bf16 tokens, 8 heads of 128, int4, take 27 us (44.5 MB, 1.6 TB/s) at 2.4 of 4
// instructions per cycle, no single pipe full (L1 50%, ALU and FMA 37% busy); a decode step of 64 rows 5.6 us, which is
// latency.  Eight CTAs per SM leave 64 registers, and D = 128 spills 48 bytes a thread there, 80 in a step; six, without
// spills, take 27.8 and 5.3 us, seven 27.2 and 5.5.  A warp for many vectors, with the next ones on their way and none
// idle for rows that end early, took 31.
//
// Codes: (y - z)/s rounded half away from zero, the quotient itself rounded to
// f32 first.  t = (y - z) * RN(1/s) is within 3 * 2^-24 times the largest code of
// that quotient (less than 2^-18 and 2^-14), so round(t) is the same unless t lies
// as near to a half (kTie); a vector with such a t (or a scale outside the range
// where 1/s is safe) is done again by the exact quotient.
#include "sa_append.cuh"
#include "sa_decode_common.cuh"
#include "sa_pages.cuh"

namespace sa {

namespace {

constexpr int kWarps = 4;

// STEP: one new token per row, the warp's vectors are eight consecutive (row, head); else the eight positions of one
// (row, head) that share p >> 3.
template <typename T, int BITS, int D, bool STEP>
__global__ void __launch_bounds__(32 * kWarps, 8) pages_append_kernel(PagesAppendArgs a, uint32_t octs, uint32_t items) {
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
    f2 x[N / 2];
    auto load_vector = [&]() {
        const T *src = static_cast<const T *>(which ? a.value : a.key) + b * a.batch_stride + s * a.token_stride +
                       (int64_t)h * D + 8 * q;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            float v[8];
            load_run<T, 8>(src + 32 * c, a.aligned, v);
#pragma unroll
            for (int i = 0; i < 4; i++) x[4 * c + i] = pair(v[2 * i], v[2 * i + 1]);
        }
    };
    if constexpr (STEP) {
        const uint32_t u = (item >> 1) * 8 + vi;
        live = u < (uint32_t)a.batch * (uint32_t)a.heads;
        b = live ? (int)(u / (uint32_t)a.heads) : 0;
        h = live ? (int)(u - (uint32_t)b * (uint32_t)a.heads) : 0;
        s = 0;
        load_vector();  // (of row 0 behind the last one) while the row's length and page are looked up
        live = live && row_tokens(a.rows, b, 1, pos) > 0;
        if (!live) pos = 0;
    } else {
        // the heads of eight tokens are neighbours in the input and in the page: they go together
        const uint32_t u = item >> 1, bo = u / (uint32_t)a.heads, oct = bo % octs;
        h = (int)(u - bo * (uint32_t)a.heads);
        b = (int)(bo / octs);
        int64_t pos0;
        tokens = row_tokens(a.rows, b, a.seq_len, pos0);
        pos = (pos0 & ~(int64_t)7) + (int64_t)oct * 8 + vi;
        live = pos >= pos0 && pos < pos0 + tokens;
        s = (int)(pos - pos0);
    }
    if (live && a.rope.on && pos >= a.rope.rows) {
        if (q == 0) atomicOr(a.rows.dev_status, kPagesBadPosition);
        live = false;
    }
    if (!__any_sync(0xffffffffu, live)) return;
    // the vector's page is on its way along with the vector; it is wanted for the stores only
    int page = -1;
    if (live && pos / kPageTokens < a.rows.max_pages) page = a.rows.table[b * a.rows.table_stride + pos / kPageTokens];
    if (!STEP && live) load_vector();
    if (!live) {
#pragma unroll
        for (int i = 0; i < N / 2; i++) x[i] = 0;
    }
    if (which == 0 && a.rope.on) {  // warp-uniform
        const float *cs = a.rope.cos_cache + (live ? pos : 0) * (D / 2), *sn = a.rope.sin_cache + (live ? pos : 0) * (D / 2);
        if (a.rope.interleaved) {
#pragma unroll
            for (int c = 0; c < CH; c++) {
                float co[4], si[4];  // the pairs of this run
                load_run<float, 4>(cs + 16 * c + 4 * q, a.rope.aligned, co);
                load_run<float, 4>(sn + 16 * c + 4 * q, a.rope.aligned, si);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float x0, x1;
                    split(x[4 * c + i], x0, x1);
                    x[4 * c + i] = pair(__fsub_rn(__fmul_rn(co[i], x0), __fmul_rn(si[i], x1)),
                                        __fadd_rn(__fmul_rn(si[i], x0), __fmul_rn(co[i], x1)));
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < CH / 2; c++) {
                float co[8], si[8];
                load_run<float, 8>(cs + 32 * c + 8 * q, a.rope.aligned, co);
                load_run<float, 8>(sn + 32 * c + 8 * q, a.rope.aligned, si);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    f2 &lo = x[4 * c + i], &hi = x[4 * (c + CH / 2) + i];
                    float x0[2], x1[2];
                    split(lo, x0[0], x0[1]);
                    split(hi, x1[0], x1[1]);
                    const float c0 = co[2 * i], c1 = co[2 * i + 1], s0 = si[2 * i], s1 = si[2 * i + 1];
                    lo = sub2(pair(__fmul_rn(c0, x0[0]), __fmul_rn(c1, x0[1])), pair(__fmul_rn(s0, x1[0]), __fmul_rn(s1, x1[1])));
                    hi = add2(pair(__fmul_rn(s0, x0[0]), __fmul_rn(s1, x0[1])), pair(__fmul_rn(c0, x1[0]), __fmul_rn(c1, x1[1])));
                }
            }
        }
    }
    {
        const float *sg = a.signs + (int64_t)h * D + 8 * q;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            float sgn[8];
            load_run<float, 8>(sg + 32 * c, true, sgn);
#pragma unroll
            for (int i = 0; i < 4; i++) x[4 * c + i] = mul2(x[4 * c + i], pair(sgn[2 * i], sgn[2 * i + 1]));
        }
    }
    // butterfly stages h = 1 (in a pair), 2, 4 (in a run), 8, 16 (across lanes), 32, 64 (between runs)
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        float p0, p1;
        split(x[i], p0, p1);
        x[i] = pair(__fadd_rn(p0, p1), __fsub_rn(p0, p1));
    }
    auto butterfly = [&](int hs) {  // of pairs
#pragma unroll
        for (int i = 0; i < N / 2; i++)
            if ((i & hs) == 0) {
                const f2 p0 = x[i], p1 = x[i + hs];
                x[i] = add2(p0, p1);
                x[i + hs] = sub2(p0, p1);
            }
    };
    butterfly(1);
    butterfly(2);
#pragma unroll
    for (int lm = 1; lm < 4; lm <<= 1) {
        // upper lane: other - x, lower lane: x + other
        const float side = (lane & lm) ? -1.0f : 1.0f;
        const f2 sides = pair(side, side);
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            float p0, p1;
            split(x[i], p0, p1);
            x[i] = fma2(x[i], sides, pair(__shfl_xor_sync(0xffffffffu, p0, lm), __shfl_xor_sync(0xffffffffu, p1, lm)));
        }
    }
#pragma unroll
    for (int hs = 4; hs < N / 2; hs <<= 1) butterfly(hs);
    float mn = INFINITY, mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        float p0, p1;
        split(x[i], p0, p1);
        p0 = __fmul_rn(p0, a.wht_scale);
        p1 = __fmul_rn(p1, a.wht_scale);
        x[i] = pair(p0, p1);
        mn = fminf(mn, fminf(p0, p1));
        mx = fmaxf(mx, fmaxf(p0, p1));
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
        for (int i = N - 1; i >= 0; i--) {
            float p[2];
            split(x[i / 2], p[0], p[1]);
            if (p[i & 1] == 0.0f) first = 2 * ((i >> 3) * 32 + 8 * q + (i & 7)) + (__float_as_int(p[i & 1]) < 0);
        }
#pragma unroll
        for (int lm = 1; lm < 4; lm <<= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, lm));
        if (mn == 0.0f) mn = (first & 1) ? -0.0f : 0.0f;
    }
    const float range = __fsub_rn(mx, mn);
    const float sc = range > 0.0f ? __fdiv_rn(range, (float)kLevels) : 1.0f;
    constexpr float kTie = BITS == 4 ? 0.5f - 0x1p-18f : 0.5f - 0x1p-14f;
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: a sum with it is rounded to whole numbers
    // (a vector of NaN leaves the minimum above the maximum, one with infinities an infinite one of them)
    const bool safe = sc >= 0x1p-90f && sc <= 0x1p100f && mn <= mx && fabsf(mn) < INFINITY && mx < INFINITY;
    uint32_t word[CH * WPC];
    {
        const float rcp = safe ? __frcp_rn(sc) : 1.0f;
        const f2 rcps = pair(rcp, rcp), magic = pair(kMagic, kMagic), least = pair(-mn, -mn);
        float far = 0.0f;
        constexpr int kPer = 32 / BITS;  // codes per word
        // a code sits in the low bits of its sum with kMagic, whose own bits a constant takes off again
        constexpr uint32_t kOff = BITS == 4 ? 0x4B400000u * 0x11111111u : 0x4B400000u * 0x01010101u;
#pragma unroll
        for (int w = 0; w < CH * WPC; w++) {
            uint32_t acc = 0u - kOff;
#pragma unroll
            for (int i = 0; i < kPer; i += 2) {
                const f2 num = add2(x[(w * kPer + i) / 2], least), k = fma2(num, rcps, magic);
                float d0, d1, k0, k1;
                split(fma2(num, rcps, sub2(magic, k)), d0, d1);
                split(k, k0, k1);
                far = fmaxf(far, fmaxf(fabsf(d0), fabsf(d1)));
                acc += (__float_as_uint(k0) << (BITS * i)) + (__float_as_uint(k1) << (BITS * (i + 1)));
            }
            word[w] = acc;
        }
        const bool redo = !safe || !(far < kTie);
        if (__any_sync(0xffffffffu, redo) && redo) {
#pragma unroll
            for (int w = 0; w < CH * WPC; w++) {
                uint32_t acc = 0;
#pragma unroll
                for (int i = 0; i < kPer; i++) {
                    float p[2];
                    split(x[(w * kPer + i) / 2], p[0], p[1]);
                    const float num = __fsub_rn(p[i & 1], mn);
                    const uint32_t c = sc > 0.0f ? __float2uint_rz(rust_round_f32(__fdiv_rn(num, sc))) : 0u;
                    acc |= min(c, kLevels) << (BITS * i);
                }
                word[w] = acc;
            }
        }
    }

    if (live && (page < 0 || page >= a.rows.num_pages)) {
        if (q == 0) atomicOr(a.rows.dev_status, kPagesBadPage);
        live = false;
    }
    uint8_t *rec = a.records + ((int64_t)(live ? page : 0) * a.heads + h) * page_record(CB);

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
