// Block means of the cached keys and the block selection of the sparse
// attention.  Both are exact integer arithmetic on grids that powers of two
// define, so the chosen blocks depend on no order of summation:
//
//   means:   S_t, Z_t = rint(scale_t, zp_t * 2^(15-e)), 2^e above every |scale|
//            and |zp| of the block; M_d = sum_t S_t c_td + Z_t (below 2^30);
//            m_d = M_d rounded half up to 8 bits under the largest |M_d|.
//   queries: n = rint(q * 2^(12-e)) over the group's heads; r = H.S.n (below
//            2^21, exact in f32); r8 = r rounded half to even to 7 bits and a
//            sign under the group's largest |r|.
//   score:   max over the heads of sum_d r8_d m_d: below 2^24, so an f32 sum of
//            the products is exact in any order, and so is the power of two of
//            the mean.
#include "sa_append.cuh"
#include "sa_common.cuh"
#include "sa_internal.h"

namespace sa {

namespace {

constexpr int kMeansThreads = 128;
constexpr float kGridMax = 1.2676506002282294e30f;  // 2^100: larger values (and NaN) count as zero

__device__ __forceinline__ float grid_value(float x) { return fabsf(x) < kGridMax ? x : 0.0f; }

// The least e with x < 2^e, at least -100 (x >= 0).
__device__ __forceinline__ int grid_exponent(float x) {
    if (!(x > 0.0f)) return -100;
    const int e = ((__float_as_int(x) >> 23) & 0xff) - 126;  // a subnormal's is below -100 anyway
    return e < -100 ? -100 : e;
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // -126..127

// Formats without a warp kernel below: grid = (blocks, units), one CTA per block, one thread per dimension.
__global__ void __launch_bounds__(kMeansThreads) block_means_kernel(MeansArgs a) {
    __shared__ int s_s[kBlockTokens], s_z[kBlockTokens];
    __shared__ int s_red[kMeansThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t unit = blockIdx.y;
    const int64_t t0 = (int64_t)(a.first + blockIdx.x) * kBlockTokens;
    const int cb = a.code_bytes, bits = a.bits, d = a.head_dim;
    float2 md = make_float2(0.0f, 0.0f);
    if (tid < kBlockTokens) md = reinterpret_cast<const float2 *>(a.k_meta)[unit * a.capacity + t0 + tid];
    md.x = grid_value(md.x);
    md.y = grid_value(md.y);
    float top = warp_max(fmaxf(fabsf(md.x), fabsf(md.y)));
    if (lane == 0) s_red[warp] = __float_as_int(top);
    __syncthreads();
    for (int w = 0; w < kMeansThreads / 32; w++) top = fmaxf(top, __int_as_float(s_red[w]));
    const int e = grid_exponent(top);
    if (tid < kBlockTokens) {
        const float f = power_of_two(15 - e);
        s_s[tid] = __float2int_rn(md.x * f);
        s_z[tid] = __float2int_rn(md.y * f);
    }
    __syncthreads();
    const uint8_t *codes = a.k_codes + (unit * a.capacity + t0) * cb;
    int sum[2] = {0, 0};  // dimensions tid and tid + kMeansThreads (head_dim <= 256)
    int zsum = 0;
    for (int t = 0; t < kBlockTokens; t++) {
        zsum += s_z[t];
        const uint8_t *row = codes + (int64_t)t * cb;
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int dim = tid + x * kMeansThreads;
            if (dim >= d) continue;
            const int bo = dim * bits, j = bo >> 3, sh = bo & 7;
            uint32_t w = row[j];
            if (sh + bits > 8 && j + 1 < cb) w |= (uint32_t)row[j + 1] << 8;
            sum[x] += s_s[t] * (int)((w >> sh) & ((1u << bits) - 1u));
        }
    }
    int mx = 0;
#pragma unroll
    for (int x = 0; x < 2; x++)
        if (tid + x * kMeansThreads < d) {
            sum[x] += zsum;
            mx = max(mx, abs(sum[x]));
        }
    mx = __reduce_max_sync(0xffffffffu, mx);
    __syncthreads();
    if (lane == 0) s_red[warp] = mx;
    __syncthreads();
    for (int w = 0; w < kMeansThreads / 32; w++) mx = max(mx, s_red[w]);
    const int sh = max(0, 32 - __clz(mx) - 8);
    const float unit_value = power_of_two(sh + e - 21);
    __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(a.means) + unit * a.row_stride + (int64_t)blockIdx.x * d;
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int dim = tid + x * kMeansThreads;
        if (dim < d) out[dim] = __float2bfloat16_rn((float)((sum[x] + ((1 << sh) >> 1)) >> sh) * unit_value);
    }
}

// ---- block means: one warp per block ----------------------------------------------
// A token's CB code bytes are CPT = CB / 16 chunks of 16 bytes; lane L reads chunk L % CPT of the tokens
// L / CPT + (32 / CPT) i, so a warp's loads are contiguous.  Two tokens' codes of a dimension, interleaved as
// bytes, are contracted with their two 16-bit scales by one dp2a: about one instruction per product.  The
// lanes' sums join by halving exchanges, and the rounding needs one maximum over the warp.
// Bound by HBM: 8 x 8 heads x 32768 int8 tokens of 128 dimensions (294 MB) in 49 us, 6.0 TB/s.
constexpr int kMeansWarps = 8;

__device__ __forceinline__ int dp2a_lo(uint32_t s, uint32_t c, int acc) {
    int r;
    asm("dp2a.lo.s32.u32 %0, %1, %2, %3;\n" : "=r"(r) : "r"(s), "r"(c), "r"(acc));
    return r;
}
__device__ __forceinline__ int dp2a_hi(uint32_t s, uint32_t c, int acc) {
    int r;
    asm("dp2a.hi.s32.u32 %0, %1, %2, %3;\n" : "=r"(r) : "r"(s), "r"(c), "r"(acc));
    return r;
}

// grid covers units * blocks warps.
template <int BITS, int CPT>
__global__ void __launch_bounds__(32 * kMeansWarps) block_means_warp_kernel(MeansArgs a) {
    constexpr int ND = 128 / BITS;       // dimensions of a chunk
    constexpr int TPI = 32 / CPT;        // tokens per iteration of the warp
    constexpr int NI = kBlockTokens / TPI;
    constexpr int D = ND * CPT;
    static_assert(NI % 2 == 0, "tokens come in pairs");
    __shared__ short s_s[kMeansWarps][kBlockTokens];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t id = (int64_t)blockIdx.x * kMeansWarps + warp;
    if (id >= (int64_t)a.units * a.blocks) return;
    const int64_t unit = id / a.blocks;
    const int blk = (int)(id % a.blocks);
    const int64_t row = unit * a.capacity + (int64_t)(a.first + blk) * kBlockTokens;
    const float4 md = reinterpret_cast<const float4 *>(a.k_meta + row * 2)[lane];  // tokens 2 lane, 2 lane + 1
    const uint4 *src = reinterpret_cast<const uint4 *>(a.k_codes + row * (D * BITS / 8)) + lane;
    const float m[4] = {grid_value(md.x), grid_value(md.y), grid_value(md.z), grid_value(md.w)};
    float top = warp_max(fmaxf(fmaxf(fabsf(m[0]), fabsf(m[1])), fmaxf(fabsf(m[2]), fabsf(m[3]))));
    const int e = grid_exponent(top);
    const float f = power_of_two(15 - e);
    const int s0 = __float2int_rn(m[0] * f), s1 = __float2int_rn(m[2] * f);  // -32768 .. 32768
    const int zsum = __reduce_add_sync(0xffffffffu, __float2int_rn(m[1] * f) + __float2int_rn(m[3] * f));
    s_s[warp][2 * lane] = (short)min(s0, 32767);
    s_s[warp][2 * lane + 1] = (short)min(s1, 32767);
    bool past = __any_sync(0xffffffffu, s0 > 32767 || s1 > 32767);  // 32768 itself: its 1 in a second round
    __syncwarp();
    int acc[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) acc[d] = 0;
    for (;;) {
        const short *sw = s_s[warp] + lane / CPT;
#pragma unroll
        for (int i0 = 0; i0 < NI; i0 += 8) {
            constexpr int NB = NI < 8 ? NI : 8;  // loads in flight
            uint4 x[NB];
#pragma unroll
            for (int i = 0; i < NB; i++) x[i] = src[(i0 + i) * 32];
#pragma unroll
            for (int i = 0; i < NB; i += 2) {
                const uint32_t s = (uint32_t)(uint16_t)sw[(i0 + i) * TPI] | ((uint32_t)(uint16_t)sw[(i0 + i + 1) * TPI] << 16);
                const uint32_t p[4] = {x[i].x, x[i].y, x[i].z, x[i].w}, q[4] = {x[i + 1].x, x[i + 1].y, x[i + 1].z, x[i + 1].w};
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    if constexpr (BITS == 4) {
                        const uint32_t pl = p[w] & 0x0f0f0f0fu, ph = (p[w] >> 4) & 0x0f0f0f0fu;
                        const uint32_t ql = q[w] & 0x0f0f0f0fu, qh = (q[w] >> 4) & 0x0f0f0f0fu;
                        const uint32_t l0 = __byte_perm(pl, ql, 0x5140), l1 = __byte_perm(pl, ql, 0x7362);
                        const uint32_t h0 = __byte_perm(ph, qh, 0x5140), h1 = __byte_perm(ph, qh, 0x7362);
                        int *t = acc + 8 * w;  // byte b of the word: dimensions 2b (low nibble), 2b + 1
                        t[0] = dp2a_lo(s, l0, t[0]);
                        t[1] = dp2a_lo(s, h0, t[1]);
                        t[2] = dp2a_hi(s, l0, t[2]);
                        t[3] = dp2a_hi(s, h0, t[3]);
                        t[4] = dp2a_lo(s, l1, t[4]);
                        t[5] = dp2a_lo(s, h1, t[5]);
                        t[6] = dp2a_hi(s, l1, t[6]);
                        t[7] = dp2a_hi(s, h1, t[7]);
                    } else {
                        const uint32_t b0 = __byte_perm(p[w], q[w], 0x5140), b1 = __byte_perm(p[w], q[w], 0x7362);
                        int *t = acc + 4 * w;
                        t[0] = dp2a_lo(s, b0, t[0]);
                        t[1] = dp2a_hi(s, b0, t[1]);
                        t[2] = dp2a_lo(s, b1, t[2]);
                        t[3] = dp2a_hi(s, b1, t[3]);
                    }
                }
            }
        }
        if (!past) break;
        past = false;
        __syncwarp();
        s_s[warp][2 * lane] = (short)(s0 > 32767);
        s_s[warp][2 * lane + 1] = (short)(s1 > 32767);
        __syncwarp();
    }
    // sums over the lanes that hold the same chunk: each exchange halves the dimensions a lane keeps
    int at = 0;  // first dimension kept, within the chunk
    constexpr int KEEP = ND / TPI > 0 ? ND / TPI : 1;
#pragma unroll
    for (int h = ND / 2, o = CPT; o < 32; o <<= 1, h >>= 1) {
        const bool up = lane & o;
        if (h >= 1) {
#pragma unroll
            for (int d = 0; d < h; d++) {
                const int mine = up ? acc[d + h] : acc[d], give = up ? acc[d] : acc[d + h];
                acc[d] = mine + __shfl_xor_sync(0xffffffffu, give, o);
            }
            at += up ? h : 0;
        }
    }
    int mx = 0;
#pragma unroll
    for (int d = 0; d < KEEP; d++) {
        acc[d] += zsum;
        mx = max(mx, abs(acc[d]));
    }
    mx = __reduce_max_sync(0xffffffffu, mx);
    const int sh = max(0, 32 - __clz(mx) - 8);
    const float unit_value = power_of_two(sh + e - 21);
    __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(a.means) + unit * a.row_stride + (int64_t)blk * D +
                         (lane % CPT) * ND + at;
#pragma unroll
    for (int d = 0; d < KEEP; d++)
        out[d] = __float2bfloat16_rn((float)((acc[d] + ((1 << sh) >> 1)) >> sh) * unit_value);
}

// The 8-bit queries of the G heads of one KV head, as floats [G][d] in shared memory.  Warp g takes head g.
template <typename T, int EPL>
__device__ __forceinline__ void select_queries(const SelectArgs &a, const T *src, const float *sg, float *s_q,
                                               float (*s_top)[8]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = a.head_dim;
    const bool active = lane * EPL < d;
    float x[EPL], sgn[EPL];
    float top = 0.0f;
    if (warp < a.group) {
#pragma unroll
        for (int r = 0; r < EPL; r++) x[r] = 0.0f;
        if (active) load_elems<T, EPL>(src + (int64_t)warp * d + lane * EPL, x);
#pragma unroll
        for (int r = 0; r < EPL; r++) {
            sgn[r] = active ? sg[lane * EPL + r] : 0.0f;
            x[r] = grid_value(x[r]);
            top = fmaxf(top, fabsf(x[r]));
        }
        top = warp_max(top);
        if (lane == 0) s_top[0][warp] = top;
    }
    __syncthreads();
    if (warp < a.group) {
        top = 0.0f;
        for (int g = 0; g < a.group; g++) top = fmaxf(top, s_top[0][g]);
        const float f = power_of_two(12 - grid_exponent(top));
#pragma unroll
        for (int r = 0; r < EPL; r++) x[r] = rintf(x[r] * f) * sgn[r];
        warp_wht_butterfly<EPL>(x, lane, d);
        top = 0.0f;
#pragma unroll
        for (int r = 0; r < EPL; r++) top = fmaxf(top, active ? fabsf(x[r]) : 0.0f);
        top = warp_max(top);
        if (lane == 0) s_top[1][warp] = top;
    }
    __syncthreads();
    if (warp < a.group && active) {
        top = 0.0f;
        for (int g = 0; g < a.group; g++) top = fmaxf(top, s_top[1][g]);
        const float f = power_of_two(-max(0, grid_exponent(top) - 7));
#pragma unroll
        for (int r = 0; r < EPL; r++)
            s_q[warp * d + lane * EPL + r] = fminf(fmaxf(rintf(x[r] * f), -127.0f), 127.0f);
    }
    __syncthreads();
}

// Largest dot product of 16 blocks' means with the 8 query columns (bf16 mma, f32 accumulators that stay exact: the
// products and sums are whole numbers below 2^24 times the block's power of two).  Thread (g, q) reads 8 dimensions
// (16 bytes) of blocks g and g + 8 at a time; bq holds the columns' values in the same order of dimensions.
template <int D>
struct BlockRows {
    uint4 x[D / 32], y[D / 32];
    // blocks g and g + 8 of `means` (nb > 0 of them are there)
    __device__ __forceinline__ void load(const __nv_bfloat16 *means, int nb, int lane) {
        const int g = lane >> 2, q = lane & 3;
        const uint4 *r0 = reinterpret_cast<const uint4 *>(means + (int64_t)min(g, nb - 1) * D) + q;
        const uint4 *r1 = reinterpret_cast<const uint4 *>(means + (int64_t)min(g + 8, nb - 1) * D) + q;
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
            x[j] = r0[4 * j];
            y[j] = r1[4 * j];
        }
    }
    __device__ __forceinline__ void scores(const uint32_t (&bq)[D / 8], float &s0, float &s1) const {
        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
            const uint32_t a[2][4] = {{x[j].x, y[j].x, x[j].y, y[j].y}, {x[j].z, y[j].z, x[j].w, y[j].w}};
#pragma unroll
            for (int h = 0; h < 2; h++)
                asm volatile(
                    "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                    "{%0, %1, %2, %3};\n"
                    : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                    : "r"(a[h][0]), "r"(a[h][1]), "r"(a[h][2]), "r"(a[h][3]), "r"(bq[4 * j + 2 * h]),
                      "r"(bq[4 * j + 2 * h + 1]));
        }
        s0 = fmaxf(c[0], c[1]);
        s1 = fmaxf(c[2], c[3]);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            s0 = fmaxf(s0, __shfl_xor_sync(0xffffffffu, s0, o));
            s1 = fmaxf(s1, __shfl_xor_sync(0xffffffffu, s1, o));
        }
    }
};

// grid = (heads, seq_len, batch): one CTA per query token and KV head.  The scores by tensor core (the means are read
// once, 16 blocks per warp step), then the k-th largest key bit by bit from the top -- one block-wide count per bit,
// ending as soon as a bit leaves exactly k -- and an ordered compaction.  Bound by the latency of that chain: 32
// sequences of 8 heads, 127 candidates, 8.6 MB of means in 10.9 us alone, 7 among others.  Warp g also prepares head
// g's query.
//
// Eight warps, or four for groups of up to four heads where a warp has two steps at most (128 blocks) and CTAs of
// eight warps (two per SM) would come in waves: 512 CTAs, 127 candidates 7.4 us instead of 10.4, 1024 CTAs 11.4
// instead of 18.7.  At 255 candidates both take 11.9 us; 256 CTAs at 511 take 18.5 with four warps, 11.3 with eight.
template <typename T, int D, int THREADS>
__global__ void __launch_bounds__(THREADS) select_blocks_kernel(SelectArgs a) {
    constexpr int EPL = D >= 32 ? D / 32 : 1, NW = THREADS / 32;
    extern __shared__ uint32_t s_key[];  // one key per candidate block, in unsigned order
    __shared__ float s_q[8 * D];
    __shared__ float s_top[2][8];
    __shared__ int s_scan[NW];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int h = blockIdx.x, s = blockIdx.y, b = blockIdx.z;
    const int64_t row = (int64_t)b * a.seq_len + s;
    const T *src = static_cast<const T *>(a.query) + (row * a.heads + h) * a.group * D;
    int32_t *out = a.block_ids + (row * a.heads + h) * a.max_blocks;
    const int own = (int)((a.pos0 + s) / kBlockTokens), nb = own + 1, k = a.max_blocks;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    if (nb <= k) {  // every block
        for (int i = tid; i < k; i += THREADS) out[i] = i < nb ? i : -1;
        return;
    }
    // ---- scores as order-preserving integers; the forced blocks above all ----
    const __nv_bfloat16 *means = static_cast<const __nv_bfloat16 *>(a.means) + ((int64_t)b * a.heads + h) * a.row_stride;
    if constexpr (D >= 32) {
        BlockRows<D> rows;  // loaded a step ahead, the first ones before the queries
        int i0 = warp * 16;
        if (i0 < own) rows.load(means + (int64_t)i0 * D, own - i0, lane);
        select_queries<T, EPL>(a, src, a.signs + (int64_t)h * D, s_q, s_top);
        uint32_t bq[D / 8];  // query column g (heads past the group repeat the first)
        const float *qg = s_q + ((lane >> 2) < a.group ? lane >> 2 : 0) * D + 8 * (lane & 3);
#pragma unroll
        for (int j = 0; j < D / 32; j++)
#pragma unroll
            for (int p = 0; p < 4; p++) {
                const __nv_bfloat162 v = __floats2bfloat162_rn(qg[32 * j + 2 * p], qg[32 * j + 2 * p + 1]);  // exact
                bq[4 * j + p] = *reinterpret_cast<const uint32_t *>(&v);
            }
        for (; i0 < own; i0 += NW * 16) {  // the means of blocks before the query's own
            const BlockRows<D> now = rows;
            if (i0 + NW * 16 < own) rows.load(means + (int64_t)(i0 + NW * 16) * D, own - i0 - NW * 16, lane);
            float s0, s1;
            now.scores(bq, s0, s1);
            const int i = i0 + (lane >> 2) + ((lane & 1) ? 8 : 0);
            if ((lane & 3) < 2 && i < own) {
                const bool forced = i < a.sink || i > own - a.local;
                s_key[i] = forced ? 0xffffffffu : (uint32_t)order_key(((lane & 1) ? s1 : s0) + 0.0f) ^ 0x80000000u;
            }
        }
    } else {
        select_queries<T, EPL>(a, src, a.signs + (int64_t)h * D, s_q, s_top);
        for (int i = warp; i < own; i += NW) {
            float best = -INFINITY;
            const float m = lane < D ? __bfloat162float(means[(int64_t)i * D + lane]) : 0.0f;
            for (int g = 0; g < a.group; g++) best = fmaxf(best, warp_sum(lane < D ? m * s_q[g * D + lane] : 0.0f));
            const bool forced = i < a.sink || i > own - a.local;
            if (lane == 0) s_key[i] = forced ? 0xffffffffu : (uint32_t)order_key(best + 0.0f) ^ 0x80000000u;
        }
    }
    if (tid == 0) s_key[own] = 0xffffffffu;
    __syncthreads();

    // ---- the largest threshold that at least k keys reach ----
    uint32_t least = 0;
    int reach = nb;  // keys at or above it
    const uint32_t mine = tid < nb ? s_key[tid] : 0u;  // t > 0: a thread without a key never counts
    for (uint32_t bit = 0x80000000u; bit != 0 && reach != k; bit >>= 1) {
        const uint32_t t = least | bit;
        int n = __syncthreads_count(mine >= t);
        for (int i = tid + THREADS; i - tid < nb; i += THREADS)
            n += __syncthreads_count(i < nb && s_key[i] >= t);
        if (n >= k) {
            least = t;
            reach = n;
        }
    }
    // ---- ascending ids of the keys above it, and of the lowest blocks that equal it ----
    int above = 0;
    if (reach != k) {
        for (int i = tid; i - tid < nb; i += THREADS) above += __syncthreads_count(i < nb && s_key[i] > least);
    }
    const int left = reach == k ? 0x7fffffff : k - above;  // how many that equal it
    int taken = 0, equal = 0;  // counts before this round of blocks
    for (int i0 = 0; i0 < nb; i0 += THREADS) {
        const int i = i0 + tid;
        const uint32_t u = i < nb ? s_key[i] : 0u;
        const bool gt = i < nb && u > least, eq = i < nb && u == least;
        // warp and block counts of both, packed (at most 256 a round)
        const unsigned mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq);
        if (lane == 0) s_scan[warp] = __popc(mg) | (__popc(me) << 16);
        __syncthreads();
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            before += w < warp ? s_scan[w] : 0;
            all += s_scan[w];
        }
        const unsigned below = (1u << lane) - 1u;
        const int ng = taken + (before & 0xffff) + __popc(mg & below);
        const int ne = equal + (before >> 16) + __popc(me & below);
        if (gt || (eq && ne < left)) out[ng + min(ne, left)] = i;
        taken += all & 0xffff;
        equal += all >> 16;
        __syncthreads();
    }
}

template <typename T, int D>
int launch_select_t(const SelectArgs &a, cudaStream_t stream) {
    const int64_t blocks = (a.pos0 + a.seq_len - 1) / kBlockTokens + 1;
    const bool four = a.group <= 4 && blocks <= 128 && (int64_t)a.heads * a.seq_len * a.batch > 2 * a.sm_count;
    auto kern = four ? select_blocks_kernel<T, D, 128> : select_blocks_kernel<T, D, 256>;
    constexpr size_t kMost = 192 * 1024, kPlain = 32 * 1024;  // keys; without the attribute (static memory beside them)
    const size_t smem = (size_t)blocks * sizeof(int);
    if (smem > kMost)
        return set_error(SA_ERR_UNSUPPORTED, "gqa_select_blocks: %lld blocks, at most 49152", (long long)blocks);
    if (a.seq_len > 65535 || a.batch > 65535)
        return set_error(SA_ERR_UNSUPPORTED, "gqa_select_blocks: %d x %d query rows, at most 65535 each", a.batch,
                         a.seq_len);
    if (smem > kPlain) {
        // always the most, so that a call of another thread between this and the launch changes nothing
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost);
        if (e != cudaSuccess) return check_cuda(e, "gqa_select_blocks smem attribute");
    }
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.heads, a.seq_len, a.batch);
    cfg.blockDim = dim3(four ? 128 : 256);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
    count_launch();
    return check_cuda(e, "gqa_select_blocks launch");
}

template <typename T>
int launch_select_dtype(const SelectArgs &a, cudaStream_t stream) {
    switch (a.head_dim) {
        case 16: return launch_select_t<T, 16>(a, stream);
        case 32: return launch_select_t<T, 32>(a, stream);
        case 64: return launch_select_t<T, 64>(a, stream);
        case 128: return launch_select_t<T, 128>(a, stream);
        default: return launch_select_t<T, 256>(a, stream);
    }
}

}  // namespace

int launch_block_means(const MeansArgs &a, cudaStream_t stream) {
    const int64_t warps = (int64_t)a.units * a.blocks;
    const int64_t ctas = (warps + kMeansWarps - 1) / kMeansWarps;
    const int fmt = ctas > 0x7fffffff ? 0 : a.bits * 1000 + a.head_dim;
    const unsigned g = (unsigned)(ctas > 0x7fffffff ? 0 : ctas);
    bool fast = true;
    switch (fmt) {
        case 4032: block_means_warp_kernel<4, 1><<<g, 32 * kMeansWarps, 0, stream>>>(a); break;
        case 4064: block_means_warp_kernel<4, 2><<<g, 32 * kMeansWarps, 0, stream>>>(a); break;
        case 4128: block_means_warp_kernel<4, 4><<<g, 32 * kMeansWarps, 0, stream>>>(a); break;
        case 4256: block_means_warp_kernel<4, 8><<<g, 32 * kMeansWarps, 0, stream>>>(a); break;
        case 8064: block_means_warp_kernel<8, 4><<<g, 32 * kMeansWarps, 0, stream>>>(a); break;
        case 8128: block_means_warp_kernel<8, 8><<<g, 32 * kMeansWarps, 0, stream>>>(a); break;
        default: fast = false;
    }
    if (fast) {
        count_launch();
        return check_cuda(cudaGetLastError(), "kv_block_means launch");
    }
    if (a.units > 65535)
        return set_error(SA_ERR_UNSUPPORTED, "kv_block_means: %d rows x heads, at most 65535", a.units);
    block_means_kernel<<<dim3(a.blocks, a.units), kMeansThreads, 0, stream>>>(a);
    count_launch();
    return check_cuda(cudaGetLastError(), "kv_block_means launch");
}

int launch_select_blocks(const SelectArgs &a, cudaStream_t stream) {
    switch (a.dtype) {
        case SA_DTYPE_FLOAT: return launch_select_dtype<float>(a, stream);
        case SA_DTYPE_FLOAT16: return launch_select_dtype<__half>(a, stream);
        default: return launch_select_dtype<__nv_bfloat16>(a, stream);
    }
}

}  // namespace sa
