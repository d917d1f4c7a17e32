// Decode attention over pages: one query token per row, rows of any lengths,
// 4/8-bit codes, head_dim 64/128.
//
// pages_attend_kernel: every SM runs one CTA of twelve independent warps.  The
// chunks (64 tokens, or 32 where a token has 128 code bytes) of all units (row,
// KV head, block of query heads) lie end to end and each warp owns an equal range,
// so rows of very different lengths keep all SMs busy; a CTA's warps have
// neighbouring ranges and prepare the queries of their few units together.  A warp
// streams its chunks through two shared-memory stages, one bulk copy per chunk (a
// record's K codes, metadata and V codes are contiguous).
//
// The arithmetic of a chunk stays in registers.  With A = the query digits (row r
// of the MMA: head r's high byte, row r + 8 its low byte) and B = K codes (columns:
// tokens), lane (r, q) of the accumulator holds head r's scores of tokens, and with
// the tokens assigned to columns as below these are exactly the tokens whose
// weights the lane has to supply as the A operand of the value product, whose B
// operand is a word of the V layout.  So scores become weights without passing
// through shared memory, and one MMA carries eight query heads: 16 rows = 8 heads x
// 2 digits.  Callers of f32, and others by choice, get three digits and four heads
// (12 rows).
//
//   s_t = ks_t (q'.c_t) + kz_t sum(q')           (log2 units, scale folded in)
//   R >= max (s_t + log2 vs_t), u_t = 2^(s_t - R) vs_t in (0, 1], 16 or 24 bits of it
//   L = sum 2^(s_t - R), Z = sum 2^(s_t - R) vz_t, X = sum u_t c_t
//   out = S.H.((X + Z) / L) / sqrt(D)
//
// R is each chunk's own, and its sums are moved to the running reference when they
// are added: a weight far below the context's largest keeps 16 bits relative to its
// neighbours, not to that largest one.  R is that maximum, or, where the value scales
// of a chunk lie within a factor of 4, max s + log2 max vs, which exceeds it by 2 at
// most and needs one logarithm.  Codes enter both products less their middle
// (8 or 128), their zero points raised by as much, so that the large common part of
// q'.c and of X need not cancel after both were rounded.  Products are exact
// integers.  A vector whose codes are all 0 is its zero point alone: the scale of 1
// that the format gives it would count codes of -128 there (drop_constant_scales).
//
// pages_merge_kernel: per unit, the sum of its warps' partial records, the
// division, the inverse rotation and the store.
//
// 64 sequences of 8192 int4 tokens, 8 KV heads of 4, 115 us for 605 MB (5.2 TB/s, 0.80
// of the measured copy); 32 of 32768, 8 heads of 8, 207 us for 1209 MB (0.89).  Some 9 us
// pass before the first product (lengths, table, queries; the first 33 MB arrive
// meanwhile), warps of a range end 6 us apart, the merge takes 4; what is left over is
// near the copy's rate, with half of the issue slots in use.
// Tried: sixteen warps of half chunks (128 registers spill; D = 64 and 8 bits, which do
// not, got 4 to 10% slower; with twelve only three digits at int4, D = 128 spill, 12
// bytes); the merge by the last CTA of a unit (6% slower: code that runs once costs its
// fetch); the queries in a launch of their own (2% slower, and a launch more).
#include "sa_async.cuh"
#include "sa_decode_common.cuh"
#include "sa_pages.cuh"

namespace sa {

namespace {

using namespace dec;

constexpr int kNWP = 12;         // warps per CTA, one CTA per SM
constexpr int kMaxRows = 512;    // rows of a launch: their lengths and prefix sums fit in 4 KB
constexpr int64_t kMaxUnits = 16384;  // units of a launch: bounds the workspace
// What a unit counts for beside its chunks, in chunks: its queries' preparation and the change to it.  At 1, 2 and 8, in
// us: 48 sequences of 0 to 16000 tokens 75.6, 75.6, 76.7 (and 3 more than at 2 without); 64 of 8192 115.3, 116.2, 119.2,
// of D = 64 82.0, 81.4, 84.1; 64 of 4096 int8 ones 105, 105, 108; 64 of up to 200 15.7, 17.2, 20.1.
constexpr int kUnitCost = 2;

template <int BITS, int D, int ND>
struct PGeo {
    static constexpr int KB = D * BITS / 8;
    static constexpr int CT = KB > 64 ? 32 : 64;    // tokens per chunk
    static constexpr int CPP = kPageTokens / CT;    // chunks per page
    static constexpr int STAGE = CT * (2 * KB + 16);
    static constexpr int NST = 2;                   // stages per warp
    static constexpr int HB = ND == 2 ? 8 : 4;      // query heads per unit
    static constexpr int NCH = D / 32;              // QK k-steps
    static constexpr int SEGW = KB / 16;            // K words per lane and token
    static constexpr int NPR = CT / 16;             // token pairs of tiles: 16 tokens each
    static constexpr int VV = KB / 32;              // 16-byte V loads per 16-token block
    static constexpr int NF = D / 4;                // value sums per lane
    static constexpr int REC = HB * (D + 4);        // floats per partial record: values, then R, L, Z (and padding)
    static constexpr int PREP = 32 * (NCH + 1);     // 16-byte words of a unit's query digits and score constants
    static constexpr int SMEM = kNWP * NST * STAGE + kNWP * NST * 8;
    static constexpr float LOG2UMAX = ND == 2 ? 15.99997798605f : 23.99999991400867f;
    static constexpr int QMAX = ND == 2 ? 32639 : 8355711;  // 127 in the top digit
    static constexpr float CENTRE = BITS == 4 ? 8.0f : 128.0f;  // the codes' middle, which the products leave out
    static constexpr float UNIT = BITS == 4 ? 0.0625f : 1.0f;  // high nibbles enter the products as 16 (c - 8)
    static_assert(SMEM + (2 * kMaxRows + 1) * 4 + kNWP * D * (ND == 2 ? 2 : 4) + 256 <= 227 * 1024, "shared memory");
};

// Value scales this near to each other, as the difference of their bits: a factor of 4 (R above).  The maximum over the
// tokens in every chunk, with the logarithms shared by a warp's lanes, took 64 sequences of 8192 tokens 116.6 us, and
// those of D = 64 86.3; so, 115.2 and 81.9; without either, and with the errors that it keeps out, 112.7 and 78.4.
constexpr uint32_t kEvenScales = 2u << 23;

// d = a.b + c, signed or unsigned digits times signed codes; c may be constant (the first product of a sum).
__device__ __forceinline__ void mma_s8s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, int c0, int c1,
                                         int c2, int c3) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}

__device__ __forceinline__ void mma_u8s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, int c0, int c1,
                                         int c2, int c3) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}

__device__ __forceinline__ void mma_u8u8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, int c0, int c1,
                                         int c2, int c3) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}

// Codes of a word as signed bytes: 8-bit ones less 128; 16 times the high nibbles less 8 (low nibbles: of w * 16).
__device__ __forceinline__ uint32_t codes8(uint32_t w) { return w ^ 0x80808080u; }
__device__ __forceinline__ uint32_t codes4(uint32_t w) { return (w & 0xF0F0F0F0u) ^ 0x80808080u; }

constexpr uint32_t kOnes = 0x01010101u;

// A weight as a whole number up to `most`: of 16 bits the conversion saturates by itself.
template <int ND>
__device__ __forceinline__ uint32_t weight_digits(float u) {
    if constexpr (ND == 2) {
        uint16_t x;
        asm("cvt.rni.u16.f32 %0, %1;\n" : "=h"(x) : "f"(u));
        return x;
    } else {
        return __float2uint_rn(fminf(u, 16777215.0f));
    }
}

// bulk_g2s whose lines leave L2 first: a row's pages are read once by a block of its query heads, and everything else that
// the call needs (queries, tables, partial records, the merge's code) stays.  64 sequences of 8192 tokens 116 us, 119
// without.  Rows that share pages do not lose by it: 16 groups of 8 beams over 8000 common tokens 209 and 214 us.
__device__ __forceinline__ uint64_t read_once_policy() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;\n" : "=l"(p));
    return p;
}
__device__ __forceinline__ void bulk_g2s_once(void *dst, const void *src, uint32_t bytes, uint64_t *bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;\n" ::"r"(
            smem_u32(dst)),
        "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

// Sets a scale of 1 to 0, in a copied chunk, where the vector's codes are all 0: so the format holds vectors of equal
// components.  At scale 1 such a value's centred codes, -8 or -128 throughout, are the largest step of the chunk, and such
// a key's are off by 128 times the sum of the query digits' errors: zero values in every seventh token cost the others
// log2(1 / scale) bits, 8 to 16 of them.  Not for speed: 64 sequences of 8192 tokens whose every fourth value is constant
// take 146 us (114 without any), and 129 where every sixteenth scale is a twentieth of the others'.
template <int KB, int CT>
__device__ __forceinline__ void drop_constant_scales(unsigned char *sp, int n_tok, int lane) {
#pragma unroll 1
    for (int t = lane; t < n_tok; t += 32) {
        float *ks = reinterpret_cast<float *>(sp + CT * KB + 8 * t), *vs = ks + 2 * CT;
        const bool key = *ks == 1.0f, value = *vs == 1.0f;
        if (!key && !value) continue;
        if (key) {
            uint32_t any = 0;
#pragma unroll 4
            for (int i = 0; i < KB / 16; i++) {
                const uint4 x = reinterpret_cast<const uint4 *>(sp + t * KB)[i];
                any |= x.x | x.y | x.z | x.w;
            }
            if (any == 0) *ks = 0.0f;
        }
        if (value) {
            const unsigned char *v = sp + CT * (KB + 16) + (t >> 4) * (16 * KB) + 16 * ((t >> 2) & 3);
            uint32_t any = 0;
#pragma unroll 4
            for (int i = 0; i < KB / 4; i++) {
                const uint4 x = *reinterpret_cast<const uint4 *>(v + 64 * i);
                any |= x.x | x.y | x.z | x.w;
            }
            if ((any & (0xffu << (8 * (t & 3)))) == 0) *vs = 0.0f;
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // before the next copy into this stage
    }
    __syncwarp();
}

// Where a range is: at chunk c of unit (KV head h, block hb of its query heads) of row r, whose units have n chunks;
// b: the row's sequence, f: the chunk's position among all.
struct Place {
    int r, h, hb, c, n, b, f;
};

// Tokens that query row r (row0 + r of batch x seq_len) attends to; their negative where its own position lies behind them,
// as its table is too short.
__device__ __forceinline__ int visible(const PagesAttendArgs &a, int row, bool report) {
    const int b = row / a.seq_len, s = row - b * a.seq_len;
    int64_t pos0;
    if (s >= row_tokens(a.rows, b, a.seq_len, pos0)) return 0;
    const int64_t pos = pos0 + s;
    if (a.rope.on && pos >= a.rope.rows) {
        if (report) atomicOr(a.rows.dev_status, kPagesBadPosition);
        return 0;
    }
    const int64_t most = (int64_t)a.rows.max_pages * kPageTokens;
    if (pos >= most) {
        if (report) atomicOr(a.rows.dev_status, kPagesBadPage);
        return -(int)most;
    }
    return (int)pos + 1;
}

// Warps that share F positions.
__host__ __device__ __forceinline__ int sharing_warps(int F, int warps) { return min(warps, F); }

// One query head of a unit by one warp: rotated to its position and into the pages' frame, as digits arranged as the A
// fragments of the scores' product, with the score constants and the row's tokens behind them.  Head w of the unit
// fills fragment row w (three digits: rows w and w + 4); head 0 also clears the rows of the heads that the unit lacks.
// `v`: room for D digits.  Kept short: it runs once per head, and fetching long straight code costs more than running it.
template <typename T, int BITS, int D, int ND>
__device__ __forceinline__ void prepare_head(const PagesAttendArgs &a, int grow, int sees, int h, int hb, int w, int lane,
                                             std::conditional_t<ND == 2, int16_t, int> *v, uint4 *unit) {
    using G = PGeo<BITS, D, ND>;
    constexpr int EPL = D / 32, N = D / 4, kHalf = G::NCH / 2;
    const int b = grow / a.seq_len, s = grow - b * a.seq_len, g = hb * G::HB + w;
    float x[EPL], sg[EPL];
    load_elems<float, EPL>(a.signs + (int64_t)h * D + lane * EPL, sg);
    load_elems<T, EPL>(static_cast<const T *>(a.query) + b * a.batch_stride + s * a.token_stride +
                           ((int64_t)h * a.group + g) * D + lane * EPL, x);
    const int len = abs(sees);
    // (a position in the rotary tables, that is below 2^31: visible)
    if (a.rope.on) rope_lane<EPL>(x, lane, D, sees > 0 ? len - 1 : __ldcg(a.rows.lens + b) + s, a.rope.cos_cache, a.rope.sin_cache, a.rope.interleaved);
#pragma unroll
    for (int i = 0; i < EPL; i++) x[i] *= sg[i];
    warp_wht_butterfly<EPL>(x, lane, D);
    float sum = 0.0f, mabs = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        x[i] *= a.wht_scale;
        sum += x[i];
        mabs = fmaxf(mabs, fabsf(x[i]));
    }
    sum = warp_sum(sum);
    mabs = warp_max(mabs);
    const float sigma = mabs > 0.0f ? mabs / (float)G::QMAX : 1.0f;
    const float inv = 1.0f / sigma, sl2 = a.scale * kLog2eF, c1 = sigma * sl2 * G::UNIT, c2 = sum * sl2;
#pragma unroll
    for (int i = 0; i < EPL; i++) v[lane * EPL + i] = min(max(__float2int_rn(x[i] * inv), -G::QMAX), G::QMAX);
    __syncwarp();
    // lane (side, k, q): the word of k-step k for quarter q, of row w or (side 1, three digits) w + 4
    const int q = lane & 3, k = (lane >> 2) & 3, side = lane >> 4;
    if (k < G::NCH && side <= ND - 2) {
        uint32_t word[4] = {0, 0, 0, 0};
#pragma unroll
        for (int hf = 0; hf < 2; hf++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                // byte e of k-group hf: the dimension as the K words hold it.  8 bits: bytes of words 2k, 2k + 1;
                // 4 bits: low nibbles of words 2k, 2k + 1 (first half of the steps), then high ones
                const int i = BITS == 4 ? 16 * (k % kHalf) + 8 * hf + 2 * e + k / kHalf : 8 * k + 4 * hf + e;
                const int x = v[q * N + i], d2 = (int)(int8_t)(x & 0xff), rest = (x - d2) >> 8;
                int up = rest, low = d2;
                if constexpr (ND == 3) {
                    const int d1 = (int)(int8_t)(rest & 0xff);
                    up = side ? d1 : (rest - d1) >> 8;
                    low = side ? 0 : d2;
                }
                word[2 * hf] |= ((uint32_t)up & 0xffu) << (8 * e);
                word[2 * hf + 1] |= ((uint32_t)low & 0xffu) << (8 * e);
            }
        unit[32 * k + 4 * (w + 4 * side) + q] = make_uint4(word[0], word[1], word[2], word[3]);
    }
    if (lane < 4 * (ND - 1))
        unit[32 * G::NCH + 4 * (w + 4 * (lane >> 2)) + q] = make_uint4(__float_as_uint(c1), __float_as_uint(c2), (uint32_t)len, 0);
    if (w == 0) {
        const int mine = (lane >> 2) & (G::HB - 1);  // the head of this lane's row
        if (hb * G::HB + mine >= a.group)
            for (int i = 0; i <= G::NCH; i++) unit[32 * i + lane] = make_uint4(0, 0, i == G::NCH ? (uint32_t)len : 0, 0);
    }
    __syncwarp();
}

template <typename T, int BITS, int D, int ND>
__global__ void __launch_bounds__(kNWP * 32, 1)
    pages_attend_kernel(PagesAttendArgs a, int row0, int rows, int hblocks, uint4 *qprep, int *prefix_out, float *records) {
    using G = PGeo<BITS, D, ND>;
    constexpr int KB = G::KB, CT = G::CT, N = D / 4;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int s_prefix[kMaxRows + 1];  // of the rows' units: chunks and kUnitCost, nothing for rows without tokens
    __shared__ int s_len[kMaxRows];
    __shared__ int s_warp[kNWP];
    __shared__ std::conditional_t<ND == 2, int16_t, int> s_digits[kNWP][D];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = lane >> 2, q = lane & 3;
    unsigned char *ring = smem + warp * G::NST * G::STAGE;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + kNWP * G::NST * G::STAGE) + warp * G::NST;
    if (lane == 0)
        for (int i = 0; i < G::NST; i++) mbar_init(bars + i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    griddep_launch_dependents();
    griddep_wait();  // pages, table, lengths and the query may come from the kernels before

    // lengths of the rows, and prefix sums of what their units cost
    {
        int carry = 0;
        if (tid == 0) s_prefix[0] = 0;
        for (int base = 0; base < rows; base += kNWP * 32) {
            const int i = base + tid;
            const int len = i < rows ? visible(a, row0 + i, blockIdx.x == 0) : 0;
            if (i < rows) s_len[i] = len;
            int v = len != 0 ? (abs(len) + CT - 1) / CT + kUnitCost : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += up;
            }
            if (lane == 31) s_warp[warp] = v;
            __syncthreads();
            int before = carry;
#pragma unroll
            for (int w = 0; w < kNWP; w++) {
                if (w < warp) before += s_warp[w];
                carry += s_warp[w];
            }
            if (i < rows) s_prefix[i + 1] = before + v;
            __syncthreads();
        }
    }
    const int upr = a.heads * hblocks;  // units per row
    if (blockIdx.x == 0)
        for (int i = tid; i <= rows; i += kNWP * 32) prefix_out[i] = s_prefix[i];
    const int F = s_prefix[rows] * upr;  // positions; fits: the launch bounds it
    const int W = sharing_warps(F, (int)gridDim.x * kNWP);
    const int C = min((int)gridDim.x, W), cta = blockIdx.x;
    if (cta >= C) return;
    // this CTA's warps of the W, and this warp
    const int w0 = (int)((int64_t)cta * W / C), w1 = (int)((int64_t)(cta + 1) * W / C), w = w0 + warp;
    const int f0 = (int)((int64_t)min(w, w1) * F / W), f1 = w < w1 ? (int)((int64_t)(w + 1) * F / W) : f0;

    // where position f lies; a unit's first kUnitCost positions stand for its first chunk
    auto place = [&](int f) {
        // the last row that begins at or before f and has tokens
        int lo = 0, hi = rows;
        const int target = f / upr;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_prefix[mid] <= target) lo = mid;
            else hi = mid;
        }
        Place p;
        p.r = lo;
        const int cost = s_prefix[lo + 1] - s_prefix[lo], off = f - s_prefix[lo] * upr, k = off / cost;
        p.n = cost - kUnitCost;
        p.c = max(off - k * cost - kUnitCost, 0);
        p.f = s_prefix[lo] * upr + k * cost + kUnitCost + p.c;
        p.h = k / hblocks;
        p.hb = k - p.h * hblocks;
        p.b = (row0 + lo) / a.seq_len;
        return p;
    };
    Place cur = place(min(f0, F - 1));
    auto advance = [&](Place &p) {
        p.f++;
        if (++p.c < p.n) return;
        p.c = 0;
        p.f += kUnitCost;
        if (++p.hb < hblocks) return;
        p.hb = 0;
        if (++p.h < a.heads) return;
        p.h = 0;
        do {
            if (++p.r >= rows) {  // past the last chunk: never used again
                p.r = rows - 1;
                return;
            }
            p.n = s_prefix[p.r + 1] - s_prefix[p.r] - kUnitCost;
        } while (p.n <= 0);
        p.b = (row0 + p.r) / a.seq_len;
    };
    auto page_of = [&](const Place &p) { return __ldcg(a.rows.table + (int64_t)p.b * a.rows.table_stride + p.c / G::CPP); };

    // copies run NST chunks ahead; the page of the next chunk to copy is fetched one step before
    const uint64_t policy = read_once_policy();
    Place ahead = cur;
    int page = page_of(ahead);
    unsigned pend = 0, bad = 0;
    bool failed = false;
    auto issue = [&](int st) {
        if (ahead.f < f1) {
            uint64_t *bar = bars + st;
            if (page < 0 || page >= a.rows.num_pages) {
                bad |= 1u << st;
                if (lane == 0) {
                    atomicOr(a.rows.dev_status, kPagesBadPage);
                    mbar_arrive(bar);
                }
            } else {
                bad &= ~(1u << st);
                const uint8_t *rec = a.records + ((int64_t)page * a.heads + ahead.h) * page_record(KB);
                unsigned char *dst = ring + st * G::STAGE;
                if (lane == 0) mbar_expect_tx(bar, G::STAGE);
                if constexpr (G::CPP == 1) {
                    if (lane == 0) {
                        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // after the warp's reads of the stage
                        bulk_g2s_once(dst, rec, G::STAGE, bar, policy);
                    }
                } else if (lane < 4) {
                    const int part = ahead.c % G::CPP;
                    const bool codes = lane == 0 || lane == 3;
                    const uint32_t nb = codes ? CT * KB : CT * 8;
                    const int from = lane == 0 ? 0 : lane == 1 ? page_k_meta(KB) : lane == 2 ? page_v_meta(KB) : page_v_codes(KB);
                    const int to = lane == 0 ? 0 : CT * KB + (lane - 1) * CT * 8;
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    bulk_g2s_once(dst + to, rec + from + part * nb, nb, bar, policy);
                }
            }
            pend |= 1u << st;
            advance(ahead);
            if (ahead.f < f1) page = page_of(ahead);
        }
    };
#pragma unroll
    for (int i = 0; i < G::NST; i++) issue(i);

    // the queries of the CTA's units, a warp per head, while the first copies are under way
    uint4 *cta_prep = qprep + (int64_t)cta * G::PREP;  // unit u at u + cta: no two CTAs write the same words
    {
        const Place lo = place((int)((int64_t)w0 * F / W)), hi = place((int)((int64_t)w1 * F / W) - 1);
        const int u0 = lo.r * upr + lo.h * hblocks + lo.hb, u1 = hi.r * upr + hi.h * hblocks + hi.hb;
        const int per = min(a.group, G::HB);  // heads of a unit, but in a last block that has fewer
        for (int t = warp; t < (u1 - u0 + 1) * per; t += kNWP) {
            const int u = u0 + t / per, hw = t % per, row = u / upr, k = u - row * upr, h = k / hblocks, hb = k - h * hblocks;
            if (s_len[row] != 0 && hb * G::HB + hw < a.group)
                prepare_head<T, BITS, D, ND>(a, row0 + row, s_len[row], h, hb, hw, lane, s_digits[warp],
                                             cta_prep + (int64_t)u * G::PREP);
        }
    }
    __syncthreads();

    uint32_t qa[G::NCH][4];       // query digits, A fragments; 4 bits: of even dimensions, then of odd ones
    float c1 = 0.0f, c2 = 0.0f, c3 = 0.0f;  // score constants of the lane's head
    // what the digit in the accumulators' upper rows counts, beside 1 for the one in the lower rows
    const float wtop = ND == 3 && r < 4 ? 65536.0f : 256.0f;
    f2 facc[G::NF / 2];           // value sums in the frame of R, two columns each
    float R = -INFINITY, L = 0.0f, Z = 0.0f;
    // One chunk's scores, weights and value sums; `part`: only its first n_tok tokens count.
    auto chunk = [&](unsigned char *sp, int n_tok, auto part) {
        constexpr bool PART = decltype(part)::value;
        const unsigned char *kmeta = sp + CT * KB, *vmeta = kmeta + CT * 8, *vcodes = vmeta + CT * 8;
        // largest value scale: lanes share the tokens (scales are not negative; their bits order as they do)
        uint32_t vbits[CT / 32], most = 0;
        bool other = false;  // a scale of 1, or value scales that are not even
#pragma unroll
        for (int i = 0; i < CT / 32; i++) {
            vbits[i] = 0x7fffffffu;
            if (!PART || 32 * i + lane < n_tok) {
                vbits[i] = __float_as_uint(*reinterpret_cast<const float *>(vmeta + (32 * i + lane) * 8)) & 0x7fffffffu;
                other |= vbits[i] == __float_as_uint(1.0f);
                most = max(most, vbits[i]);
            }
        }
        most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
        for (int i = 0; i < CT / 32; i++) other |= vbits[i] + kEvenScales < most;
        // ---- scores: tile pair p holds tokens 16 p + 4 q + e of the lane's head ----
        float sc[4 * G::NPR];
        float smax = -INFINITY;
#pragma unroll
        for (int p = 0; p < G::NPR; p++) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const unsigned char *kp = sp + (16 * p + 4 * (r >> 1) + 2 * j + (r & 1)) * KB + q * (KB / 4);
                uint32_t wv[G::SEGW];
                if constexpr (G::SEGW == 2) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(kp);
                    wv[0] = v.x;
                    wv[1] = v.y;
                } else {
#pragma unroll
                    for (int i = 0; i < G::SEGW / 4; i++) {
                        const uint4 v = reinterpret_cast<const uint4 *>(kp)[i];
                        wv[4 * i] = v.x;
                        wv[4 * i + 1] = v.y;
                        wv[4 * i + 2] = v.z;
                        wv[4 * i + 3] = v.w;
                    }
                }
                int d[4];
                if constexpr (BITS == 4) {
                    constexpr int kHalf = G::NCH / 2;
                    mma_s8s8(d, qa[0], codes4(wv[0] * 16u), codes4(wv[1] * 16u), 0, 0, 0, 0);
                    if constexpr (kHalf == 2)
                        mma_s8s8(d, qa[1], codes4(wv[2] * 16u), codes4(wv[3] * 16u), d[0], d[1], d[2], d[3]);
                    mma_s8s8(d, qa[kHalf], codes4(wv[0]), codes4(wv[1]), d[0], d[1], d[2], d[3]);
                    if constexpr (kHalf == 2)
                        mma_s8s8(d, qa[kHalf + 1], codes4(wv[2]), codes4(wv[3]), d[0], d[1], d[2], d[3]);
                } else {
                    mma_s8s8(d, qa[0], codes8(wv[0]), codes8(wv[1]), 0, 0, 0, 0);
#pragma unroll
                    for (int k = 1; k < G::NCH; k++)
                        mma_s8s8(d, qa[k], codes8(wv[2 * k]), codes8(wv[2 * k + 1]), d[0], d[1], d[2], d[3]);
                }
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    float &dot = sc[4 * p + 2 * j + x];
                    if constexpr (ND == 2) {
                        dot = (float)(d[x] * 256 + d[2 + x]);
                    } else {  // the other digits' part is the lane's that is four heads away
                        dot = fmaf((float)d[x], wtop, (float)d[2 + x]);
                        dot += __shfl_xor_sync(0xffffffffu, dot, 16);
                    }
                }
            }
            const float4 km0 = *reinterpret_cast<const float4 *>(kmeta + (16 * p + 4 * q) * 8);
            const float4 km1 = *reinterpret_cast<const float4 *>(kmeta + (16 * p + 4 * q) * 8 + 16);
            const float ks[4] = {km0.x, km0.z, km1.x, km1.z}, kz[4] = {km0.y, km0.w, km1.y, km1.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                // ks (q'.(c - C)) + (kz + C ks) sum(q')
                float s = fmaf(ks[e], fmaf(c1, sc[4 * p + e], c3), kz[e] * c2);
                if (PART && 16 * p + 4 * q + e >= n_tok) s = -INFINITY;
                sc[4 * p + e] = s;
                smax = fmaxf(smax, s);
                other |= ks[e] == 1.0f;
            }
        }
        // the chunk's reference: the largest weight times value scale, or a little more where the scales are alike
        float Rc;
        if (!__any_sync(0xffffffffu, other)) {
            Rc = smax + __log2f(fmaxf(__uint_as_float(most), kVScaleMin));
        } else {
            drop_constant_scales<KB, CT>(sp, n_tok, lane);
            Rc = -INFINITY;
#pragma unroll
            for (int p = 0; p < G::NPR; p++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float2 km = *reinterpret_cast<const float2 *>(kmeta + (16 * p + 4 * q + e) * 8);
                    const float vs = *reinterpret_cast<const float *>(vmeta + (16 * p + 4 * q + e) * 8);
                    float &s = sc[4 * p + e];
                    if (km.x == 0.0f && s > -INFINITY) s = km.y * c2;
                    Rc = fmaxf(Rc, s + __log2f(fmaxf(fabsf(vs), kVScaleMin)));
                }
        }
#pragma unroll
        for (int lm = 1; lm < 4; lm <<= 1) Rc = fmaxf(Rc, __shfl_xor_sync(0xffffffffu, Rc, lm));
        // the running reference, and the factors that bring both sums to it
        const float Rn = fmaxf(R, Rc);
        const float fo = R == -INFINITY ? 0.0f : ex2_approx(R - Rn), fn = Rc == -INFINITY ? 0.0f : ex2_approx(Rc - Rn);
        R = Rn;
        const float base = Rc == -INFINITY ? 0.0f : Rc - G::LOG2UMAX;
        // ---- weights: u = 2^(s - Rc) vs as fixed-point digits, A fragments of 32 tokens each ----
        uint32_t ua[CT / 32][4];
        float lc = 0.0f, zc = 0.0f;
#pragma unroll
        for (int p = 0; p < G::NPR; p++) {
            const float4 vm0 = *reinterpret_cast<const float4 *>(vmeta + (16 * p + 4 * q) * 8);
            const float4 vm1 = *reinterpret_cast<const float4 *>(vmeta + (16 * p + 4 * q) * 8 + 16);
            float vs[4] = {vm0.x, vm0.z, vm1.x, vm1.z}, vz[4] = {vm0.y, vm0.w, vm1.y, vm1.w};
            uint32_t U[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (PART && 16 * p + 4 * q + e >= n_tok) vs[e] = vz[e] = 0.0f;  // whatever a page holds there
                const float ee = ex2_approx(sc[4 * p + e] - base);
                lc += ee;
                zc = fmaf(ee, fmaf(G::CENTRE, vs[e], vz[e]), zc);
                U[e] = weight_digits<ND>(ee * vs[e]);
            }
            if constexpr (ND == 2) {
                const uint32_t p01 = __byte_perm(U[0], U[1], 0x5410), p23 = __byte_perm(U[2], U[3], 0x5410);
                ua[p >> 1][2 * (p & 1)] = __byte_perm(p01, p23, 0x7531);
                ua[p >> 1][2 * (p & 1) + 1] = __byte_perm(p01, p23, 0x6420);
            } else {
                const uint32_t top = r < 4 ? 0x0062u : 0x0051u;
                ua[p >> 1][2 * (p & 1)] = __byte_perm(__byte_perm(U[0], U[1], top), __byte_perm(U[2], U[3], top), 0x5410);
                ua[p >> 1][2 * (p & 1) + 1] =
                    r < 4 ? __byte_perm(__byte_perm(U[0], U[1], 0x0040), __byte_perm(U[2], U[3], 0x0040), 0x5410) : 0u;
            }
        }
        L = fmaf(L, fo, lc * fn);
        Z = fmaf(Z, fo, zc * fn);
        if (__any_sync(0xffffffffu, fo != 1.0f)) {
#pragma unroll
            for (int i = 0; i < G::NF / 2; i++) facc[i] = mul2(facc[i], pair(fo, fo));
        }
        // ---- values: 16-byte piece v of the V blocks at a time, its integer sums folded at once ----
        // 4 bits: one sum over the bytes as they are, u (lo + 16 hi), and one over 16 (hi - 8); the first starts at
        // -(8 + 128) sum(u), so that their difference is the sum of u (lo - 8)
        [[maybe_unused]] int first[4] = {0, 0, 0, 0};
        if constexpr (BITS == 4) {
#pragma unroll
            for (int t = 0; t < CT / 32; t++) mma_u8u8(first, ua[t], kOnes, kOnes, first[0], first[1], first[2], first[3]);
#pragma unroll
            for (int i = 0; i < 4; i++) first[i] *= -136;
        }
        // adds n-tile sums, weighed w, to the value sums
        auto fold = [&](f2 &sum, const int (&d)[4], float w) {
            if constexpr (ND == 2) {
                sum = fma2(pair((float)(d[0] * 256 + d[2]), (float)(d[1] * 256 + d[3])), pair(w, w), sum);
            } else {
                sum = fma2(pair((float)d[0], (float)d[1]), pair(w * wtop, w * wtop), sum);
                sum = fma2(pair((float)d[2], (float)d[3]), pair(w, w), sum);
            }
        };
#pragma unroll
        for (int v = 0; v < G::VV; v++) {
            constexpr int NJ = BITS == 4 ? 8 : 4;  // n-tiles of the piece
            int acc[NJ][4];
#pragma unroll
            for (int t = 0; t < CT / 32; t++) {
                const unsigned char *vb = vcodes + 2 * t * (16 * KB) + (8 * v + r) * 64 + 16 * q;
                const uint4 x0 = *reinterpret_cast<const uint4 *>(vb);
                const uint4 x1 = *reinterpret_cast<const uint4 *>(vb + 16 * KB);
                const uint32_t y0[4] = {x0.x, x0.y, x0.z, x0.w}, y1[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (BITS == 4) {
                        int (&raw)[4] = acc[2 * j], (&hi)[4] = acc[2 * j + 1];
                        if (t == 0) {
                            mma_u8u8(raw, ua[t], y0[j], y1[j], first[0], first[1], first[2], first[3]);
                            mma_u8s8(hi, ua[t], codes4(y0[j]), codes4(y1[j]), 0, 0, 0, 0);
                        } else {
                            mma_u8u8(raw, ua[t], y0[j], y1[j], raw[0], raw[1], raw[2], raw[3]);
                            mma_u8s8(hi, ua[t], codes4(y0[j]), codes4(y1[j]), hi[0], hi[1], hi[2], hi[3]);
                        }
                    } else {
                        int (&d)[4] = acc[j];
                        if (t == 0) mma_u8s8(d, ua[t], codes8(y0[j]), codes8(y1[j]), 0, 0, 0, 0);
                        else mma_u8s8(d, ua[t], codes8(y0[j]), codes8(y1[j]), d[0], d[1], d[2], d[3]);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (BITS == 4) {
                    int (&raw)[4] = acc[2 * j], (&hi)[4] = acc[2 * j + 1];
#pragma unroll
                    for (int i = 0; i < 4; i++) raw[i] -= hi[i];
                    fold(facc[v * NJ + 2 * j], raw, fn);
                    fold(facc[v * NJ + 2 * j + 1], hi, fn * G::UNIT);
                } else {
                    fold(facc[v * NJ + j], acc[j], fn);
                }
            }
        }
    };
    int len = 0;
    bool fresh = true;
    int st = 0;
    uint32_t phase = 0;
    while (cur.f < f1) {
        if (fresh) {
            // ---- a new unit: its digits and constants ----
            fresh = false;
            R = -INFINITY;
            L = Z = 0.0f;
#pragma unroll
            for (int i = 0; i < G::NF / 2; i++) facc[i] = 0;
            const uint4 *src = cta_prep + ((int64_t)cur.r * upr + cur.h * hblocks + cur.hb) * G::PREP + lane;
#pragma unroll
            for (int k = 0; k < G::NCH; k++) {
                const uint4 v = src[32 * k];
                qa[k][0] = v.x;
                qa[k][1] = v.y;
                qa[k][2] = v.z;
                qa[k][3] = v.w;
            }
            const uint4 v = src[32 * G::NCH];
            c1 = __uint_as_float(v.x);
            c2 = __uint_as_float(v.y);
            c3 = G::CENTRE * c2;
            len = (int)v.z;
        }
        if (!mbar_wait_bounded(bars + st, phase)) failed = true;
        if (__any_sync(0xffffffffu, failed)) {
            failed = true;
            break;
        }
        pend &= ~(1u << st);
        const int n_tok = (bad >> st) & 1u ? 0 : min(CT, len - cur.c * CT);
        if (n_tok == CT) chunk(ring + st * G::STAGE, CT, std::false_type());
        else if (n_tok > 0) chunk(ring + st * G::STAGE, n_tok, std::true_type());
        __syncwarp();
        issue(st);
        if (++st == G::NST) {
            st = 0;
            phase ^= 1u;
        }
        const Place was = cur;
        advance(cur);
        if (cur.f >= f1 || cur.c == 0) {
            // ---- the unit's partial record ----
#pragma unroll
            for (int lm = 1; lm < 4; lm <<= 1) {
                L += __shfl_xor_sync(0xffffffffu, L, lm);
                Z += __shfl_xor_sync(0xffffffffu, Z, lm);
            }
            float x[G::NF];
#pragma unroll
            for (int i = 0; i < G::NF / 2; i++) split(facc[i], x[2 * i], x[2 * i + 1]);
            if constexpr (ND == 3) {  // the two lanes of a head hold sums of different digits
#pragma unroll
                for (int i = 0; i < G::NF; i++) x[i] += __shfl_xor_sync(0xffffffffu, x[i], 16);
            }
            if (r < G::HB) {
                float *rec = records + ((int64_t)w + (int64_t)was.r * upr + was.h * hblocks + was.hb) * G::REC;
                float4 *dst = reinterpret_cast<float4 *>(rec + r * D + q * N);
#pragma unroll
                for (int i = 0; i < N / 4; i++) dst[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                if (q == 0) *reinterpret_cast<float4 *>(rec + G::HB * D + 4 * r) = make_float4(R, L, Z, 0.0f);
            }
            fresh = true;
        }
    }
    if (failed) {
        if (lane == 0) {
            atomicOr(a.rows.dev_status, kPagesTimeout);
            // nothing was issued since: let this warp's copies in flight land (bounded)
            for (int i = 0; i < G::NST; i++)
                if (pend & (1u << i)) mbar_wait_bounded(bars + i, i < st ? phase ^ 1u : phase);
        }
    }
}

// One CTA per unit, one warp per query head.
template <typename T, int BITS, int D, int ND>
__global__ void __launch_bounds__(32 * PGeo<BITS, D, ND>::HB)
    pages_merge_kernel(PagesAttendArgs a, int row0, int rows, int hblocks, int warps, const int *prefix,
                       const float *records) {
    using G = PGeo<BITS, D, ND>;
    constexpr int EPL = D / 32, kBatch = 8;
    __shared__ float s_x[G::HB][D];
    const int lane = threadIdx.x & 31, hl = threadIdx.x >> 5;
    const int upr = a.heads * hblocks;
    const int u = blockIdx.x, row = u / upr, k = u - row * upr, h = k / hblocks, g = (k - h * hblocks) * G::HB + hl;
    griddep_launch_dependents();
    float sg[EPL];
#pragma unroll
    for (int e = 0; e < EPL; e++) sg[e] = a.wht_scale * a.signs[(int64_t)h * D + lane * EPL + e];
    griddep_wait();
    if (g >= a.group) return;
    const int p0 = prefix[row], cost = prefix[row + 1] - p0;
    float x[EPL], L = 0.0f, Z = 0.0f;
#pragma unroll
    for (int e = 0; e < EPL; e++) x[e] = 0.0f;
    if (cost > 0) {
        const int F = prefix[rows] * upr, W = sharing_warps(F, warps);
        const int f0 = p0 * upr + k * cost;  // the unit's chunks are at [f0 + kUnitCost, f0 + cost)
        const int w_lo = warp_of_chunk(f0 + kUnitCost, F, W), w_hi = warp_of_chunk(f0 + cost - 1, F, W);
        const float *base = records + ((int64_t)u + w_lo) * G::REC;
        const int nrec = w_hi - w_lo + 1;
        // batches of records are loaded together, the first one along with what weighs them
        using Vec = std::conditional_t<EPL == 4, float4, float2>;
        union {
            Vec v;
            float f[EPL];
        } val[kBatch];
        auto load = [&](int j0) {
#pragma unroll
            for (int j = 0; j < kBatch; j++)
                if (j0 + j < nrec)
                    val[j].v = *reinterpret_cast<const Vec *>(base + (int64_t)(j0 + j) * G::REC + hl * D + lane * EPL);
        };
        load(0);
        float M = -INFINITY;
        for (int i = lane; i < nrec; i += 32) M = fmaxf(M, base[(int64_t)i * G::REC + G::HB * D + 4 * hl]);
        M = warp_max(M);
        for (int i0 = 0; i0 < nrec; i0 += 32) {
            float wt = 0.0f;
            if (i0 + lane < nrec) {
                const float4 m = *reinterpret_cast<const float4 *>(base + (int64_t)(i0 + lane) * G::REC + G::HB * D + 4 * hl);
                wt = m.x == -INFINITY ? 0.0f : exp2f(m.x - M);
                L = fmaf(wt, m.y, L);
                Z = fmaf(wt, m.z, Z);
                if (m.x == -INFINITY) L += m.y;  // NaN sums spoil the row
            }
            for (int j0 = i0; j0 < min(nrec, i0 + 32); j0 += kBatch) {
                if (j0 > 0) load(j0);
#pragma unroll
                for (int j = 0; j < kBatch; j++) {
                    const float wj = __shfl_sync(0xffffffffu, wt, (j0 + j) & 31);
                    if (j0 + j < nrec)
#pragma unroll
                        for (int e = 0; e < EPL; e++) x[e] = fmaf(wj, val[j].f[e], x[e]);
                }
            }
        }
    }
    L = warp_sum(L);
    Z = warp_sum(Z);
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
    // records hold a lane's sums in its order: entry (q, v, n-tile, column pair) -> dimension
#pragma unroll
    for (int e = 0; e < EPL; e++) {
        const int i = lane * EPL + e, q = i / (D / 4), rest = i % (D / 4);
        constexpr int NJ = BITS == 4 ? 8 : 4;
        const int v = rest / (2 * NJ), j = rest / 2 % NJ, col = 2 * q + (rest & 1);
        const int dim = BITS == 4 ? 2 * (32 * v + 4 * col + (j >> 1)) + (j & 1) : 32 * v + 4 * col + j;
        s_x[hl][dim] = L != 0.0f ? (x[e] + Z) * inv : 0.0f;
    }
    __syncwarp();
#pragma unroll
    for (int e = 0; e < EPL; e++) x[e] = s_x[hl][lane * EPL + e];
    warp_wht_butterfly<EPL>(x, lane, D);
    T *dst = static_cast<T *>(a.out) + (((int64_t)(row0 + row) * a.heads + h) * a.group + g) * D + lane * EPL;
#pragma unroll
    for (int e = 0; e < EPL; e++) st_from_f32(dst + e, x[e] * sg[e]);
}

constexpr size_t kPrefixBytes = ((kMaxRows + 1) * sizeof(int) + 255) / 256 * 256;

// Whether queries and weights have three digits.  A unit has as many query heads as one product carries, four of three
// digits or eight of two.  64 sequences of 8192 tokens, 8 heads of 4, take bf16 callers 121 us with three and 114 with
// two, and 32 of 32768, 8 heads of 8, which are two units with three, f16 callers 456 and 206; against 64 bits the output
// is off by 1.6662e-3 and 1.6668e-3 of its norm, and by 2.074e-4 and 2.126e-4, nearly all of it its own rounding.
bool three_digits(int dtype, int full) { return dtype == SA_DTYPE_FLOAT || full; }
int head_block(int dtype, int full) { return three_digits(dtype, full) ? 4 : 8; }

int64_t rows_per_launch(int64_t units_per_row) {
    const int64_t n = kMaxUnits / units_per_row;
    return n < 1 ? 1 : (n < kMaxRows ? n : kMaxRows);
}

template <typename T, int BITS, int D, int ND>
int launch_shape(const PagesAttendArgs &a, void *workspace, cudaStream_t stream) {
    using G = PGeo<BITS, D, ND>;
    auto kern = pages_attend_kernel<T, BITS, D, ND>;
    static int configured[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !__atomic_load_n(&configured[dev], __ATOMIC_ACQUIRE)) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
        if (e != cudaSuccess) return check_cuda(e, "gqa_paged_attend smem attribute");
        if (dev >= 0 && dev < 64) __atomic_store_n(&configured[dev], 1, __ATOMIC_RELEASE);
    }
    const int hblocks = (a.group + G::HB - 1) / G::HB;
    const int64_t upr = (int64_t)a.heads * hblocks, rows = (int64_t)a.batch * a.seq_len, per = rows_per_launch(upr);
    const int64_t row_chunks = upr * ((int64_t)a.rows.max_pages * G::CPP + kUnitCost);
    const int64_t most = rows < per ? rows : per;
    int *prefix = static_cast<int *>(workspace);
    uint4 *qprep = reinterpret_cast<uint4 *>(static_cast<char *>(workspace) + kPrefixBytes);
    float *records = reinterpret_cast<float *>(qprep + (most * upr + a.sm_count) * G::PREP);
    for (int64_t row0 = 0; row0 < rows;) {
        int64_t n = rows - row0 < per ? rows - row0 : per;
        if (n * row_chunks >= ((int64_t)1 << 31)) n = (((int64_t)1 << 31) - 1) / row_chunks;  // chunk indices are ints
        if (n == 0)
            return set_error(SA_ERR_UNSUPPORTED, "gqa_paged_attend: rows of %d pages are too long", a.rows.max_pages);
        cudaLaunchAttribute pdl[1];
        pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        pdl[0].val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.stream = stream;
        cfg.attrs = pdl;
        cfg.numAttrs = 1;
        cfg.gridDim = dim3((unsigned)a.sm_count);
        cfg.blockDim = dim3(kNWP * 32);
        cfg.dynamicSmemBytes = G::SMEM;
        int rc = check_cuda(cudaLaunchKernelEx(&cfg, kern, a, (int)row0, (int)n, hblocks, qprep, prefix, records),
                            "gqa_paged_attend launch");
        count_launch();
        if (rc != SA_OK) return rc;
        cfg.gridDim = dim3((unsigned)(n * upr));
        cfg.blockDim = dim3(32 * G::HB);
        cfg.dynamicSmemBytes = 0;
        rc = check_cuda(cudaLaunchKernelEx(&cfg, pages_merge_kernel<T, BITS, D, ND>, a, (int)row0, (int)n, hblocks,
                                           a.sm_count * kNWP, (const int *)prefix, (const float *)records),
                        "gqa_paged_attend merge launch");
        count_launch();
        if (rc != SA_OK) return rc;
        row0 += n;
    }
    return SA_OK;
}

template <typename T, int ND>
int launch_t(const PagesAttendArgs &a, void *workspace, cudaStream_t stream) {
    if (a.bits == 4)
        return a.head_dim == 128 ? launch_shape<T, 4, 128, ND>(a, workspace, stream)
                                 : launch_shape<T, 4, 64, ND>(a, workspace, stream);
    return a.head_dim == 128 ? launch_shape<T, 8, 128, ND>(a, workspace, stream)
                             : launch_shape<T, 8, 64, ND>(a, workspace, stream);
}

}  // namespace

size_t pages_attend_workspace(const kv_pages_impl *k, int batch, int seq_len, int dtype) {
    const int hb = head_block(dtype, k->full);
    const int64_t upr = (int64_t)k->cfg.kv_head_count * ((k->group + hb - 1) / hb);
    const int64_t rows = (int64_t)batch * seq_len, per = rows_per_launch(upr), n = rows < per ? rows : per;
    const int64_t records = (int64_t)k->sm_count * kNWP + n * upr;  // one per warp, and one more per unit
    const size_t prep = (size_t)(n * upr + k->sm_count) * 32 * (k->cfg.head_dim / 32 + 1) * 16;  // digits and constants of a unit
    return kPrefixBytes + prep + (size_t)records * hb * (k->cfg.head_dim + 4) * sizeof(float);
}

int launch_pages_attend(const PagesAttendArgs &a, void *workspace, cudaStream_t stream) {
    const bool three = three_digits(a.dtype, a.full);
    switch (a.dtype) {
        case SA_DTYPE_FLOAT: return launch_t<float, 3>(a, workspace, stream);
        case SA_DTYPE_FLOAT16: return three ? launch_t<__half, 3>(a, workspace, stream) : launch_t<__half, 2>(a, workspace, stream);
        default:
            return three ? launch_t<__nv_bfloat16, 3>(a, workspace, stream) : launch_t<__nv_bfloat16, 2>(a, workspace, stream);
    }
}

}  // namespace sa
