// Attention of a draft tree over the compressed cache on the 5th-generation
// tensor cores: the R = nodes * G query rows of one KV head against the whole
// context, in the rotated domain, with everything transposed -- tokens (then
// dimensions) are the MMA's M, the query rows its N:
//
//   S^T[t][r]  = sum_d (c_td - C) q^_rd                      (M = 128 tokens, N = rows)
//   s_tr       = ks_t S^T + (kz_t + C ks_t) sum(q^_r)         (log2 units; ks, kz: scale, zero point)
//   u_tr       = vs_t 2^(s_tr - ref_r)
//   O^T[d][r] += sum_t (c_td - C) u_tr                        (M = dimensions, N = rows)
//   l_r += u_tr / vs_t,   z_r += u_tr (vz_t + C vs_t) / vs_t
//   o'_r = (O_r + z_r) / l_r,   out = S.H.o' / sqrt(D)
//
// C = 7.5 or 127.5, the middle of the codes, so that no sum carries the codes' mean,
// which the zero point would have to cancel: the tensor cores' f32 sums lose bits at
// every step, and with C = 8 the half that is left cost f32 callers a factor
// of three at 16,000 tokens (3.3e-6 against 1.0e-6 of the output's norm).  For the same
// reason O^T holds one tile at a time for f32 callers, and the softmax warps add it up
// (summed in tensor memory over the 110 tiles of a range: 2.6e-5; so: 5.9e-7).  q^ is q' = H.S.q scale log2(e) / D^(1/2) on a
// power of two common to the row block, or, in a block whose rows lie more than 2^14
// apart, on one of its own row (kSpread); q^ and u are held in one fp16 plane each
// (11 bits) for bf16 callers, whose outputs' own rounding is eight times as coarse
// (the error against 64 bits grows by 2.2%; with two planes, the cache's choice, by
// nothing, at 388 instead of 300 us for 64 sequences), and in two (22 bits) for f16 and f32:
// with one plane of u the error of f16 outputs was 1.37 times that of f32 arithmetic
// rounded once, at 1,316 instead of 1,412 us in the widest case.  sum(q^) is of the
// rounded values, so their rounding only moves the query by its own.  Everything
// else is f32.
//
// Transposed, a thread of the softmax holds one token: its scale and zero point
// are registers, not loads per score, and N follows the number of rows (16, 32 or
// 64), so a tree of few rows costs few MMA columns.  The codes become fp16 in
// tensor memory, as the A operands: a code zero-extended to 16 bits is an fp16 number, and one
// packed multiply-add centres two.
//
// One persistent CTA per SM; roles by warp:
//   4, 8 or 16 softmax warps (groups of four, 16 rows each): thread = token of
//     the tile: tcgen05.ld of S^T, u, the sums l and z of its token, u to shared
//     memory (the B operand, rows contiguous).  The reference ref_r is only raised
//     when some score of the tile outgrows it by 2^8 (one vote per tile and
//     group); then O is rescaled, in tensor memory or the threads' registers.
//   4 K warps, 4 V warps: codes of the tile from shared memory to fp16 in tensor
//     memory, two buffers each; the K warps also turn the tokens' scales and zero
//     points into what the softmax needs.
//   2 MMA warps: one issues S^T, the other O^T.
//   1 copy warp: codes and metadata of the tiles by bulk copies into a ring.
// The tiles of all units (batch row, KV head) are laid end to end and cut into
// equal ranges; row blocks beyond the first 64 rows run in CTAs of their own that
// walk the same ranges at the same time, so the cache is read from HBM once.  A
// CTA leaves one partial record per unit that it touches; a merge kernel joins
// them, rotates back and stores.
//
// Bound by instruction issue (62% of the cycles; about 5,900 warp instructions per
// tile of 128 tokens and 64 rows, more than half of them the softmax's; tensor pipe
// 20%): 16 sequences of 8 KV heads, 8176 int4 tokens, 64 bf16 rows, 155 MB, 88 us with
// prep and merge (f16, two planes: 110); 64 sequences 300 us.  Groups of 16 rows: with 32 a group's
// registers leave room for half the warps (113 us).
//
// Every mbarrier wait is bounded (2 s); one that gives up sets the abort flag and
// bit 0 of the cache's status word, every role leaves its loop, issued copies and
// MMAs are waited for (bounded) and TMEM is freed; the records are then not valid.
#include <type_traits>

#include "sa_append.cuh"
#include "sa_async.cuh"
#include "sa_common.cuh"
#include "sa_internal.h"
#include "sa_tcgen05.cuh"

namespace sa {

namespace {

constexpr int kTok = 128;       // tokens per tile: M of S^T, K of O^T
constexpr float kHead = 8.0f;   // octaves a score may outgrow its reference before that moves
// Smaller value scales (constant vectors have 0) count as this, at 255 times it in the outputs at most.  The sums of
// u / vs then reach 2^(7 + 80) times the tokens and, in z, the zero points: far from f32's 2^128 at any context.
constexpr float kScaleMin = 0x1p-80f;
constexpr float kShift = 7.0f;  // u <= 2^(kHead + kShift), below fp16's 65504
// Rows whose largest |q'| is within 2^kSpread of the block's keep all 22 bits of two planes on the block's power of
// two: the block's largest is put into [2^11, 2^12), and fp16 numbers are multiples of 2^-24.  A block that spreads
// further has a power of two per row, so that no query, however large, costs other rows bits; each of its tiles takes
// the path that raises references (145 instead of 88 us for 16 sequences in bf16).  A scale per row in every tile
// cost all callers 5%.
constexpr int kSpread = 14;
constexpr int kPrepThreads = 512;
constexpr int kMergeWarps = 8;

// QP, PP: fp16 planes of q^ and u.  F32: the caller's type is f32 (see the top).
template <int BITS, int D, int NR, int QP, int PP, bool F32>
struct Tg {
    static constexpr int CB = D * BITS / 8;
    static constexpr int NC = 16;                           // query rows of a softmax group of four warps
    static constexpr int NG = NR / NC;
    static constexpr int THREADS = 32 * (4 * NG + 11);
    // With four groups the 864 threads are launched with 72 registers each, and the 256 threads of the K and V warps
    // hand some of theirs on to the softmax: 512 * 88 + 256 * 40 + 96 * 72 = 864 * 72 (launch_rows checks the 72).
    static constexpr bool SPLIT = NG == 4;
    static constexpr int LAUNCH = 72, SOFT = 88, STAGE = 40;
    static_assert(!SPLIT || 128 * NG * SOFT + 256 * STAGE + 96 * LAUNCH <= THREADS * LAUNCH, "register split");
    static constexpr int PBUF = PP * kTok * 128;            // u planes of a tile: [128 tokens][64 rows], 128-byte swizzle
    static constexpr int QPLANE = NR * D * 2;               // D/64 tiles of [NR rows][128 B]
    // planes, sum(q^) of the rows, their powers of two, the common one (0: the rows have their own)
    static constexpr int QREC = QP * QPLANE + NR * 8 + 16;
    static constexpr int QBUF = (QREC + 1023) / 1024 * 1024;
    // ring slot: K codes, V codes, K metadata, V metadata; then what the softmax makes of a token's metadata
    static constexpr int META = 2 * kTok * CB, CONST = META + kTok * 16, SLOT = CONST + kTok * 20;
    static constexpr int P_OFF = 0, Q_OFF = 2 * PBUF, SLOT_OFF = Q_OFF + 2 * QBUF;
    static constexpr int MISC = 6 * 1024;
    static constexpr int ROOM = (226 * 1024 - SLOT_OFF - MISC) / SLOT;
    static constexpr int NST = ROOM > 8 ? 8 : ROOM;         // ring slots
    static constexpr int MISC_OFF = SLOT_OFF + NST * SLOT;
    static constexpr int SMEM = MISC_OFF + MISC + 1024;     // + slack to align the base to 1024 B
    // f32: the softmax warps sum the tiles' O^T themselves, from two buffers
    static constexpr bool FOLD = F32;
    // TMEM columns: K and V operands (two buffers each), S^T (two), O^T
    static constexpr uint32_t KA = 0, VA = D, S = VA + kTok, O = S + 2 * NR;
    static constexpr int REC = NR * D + 3 * NR;             // floats of a partial record: O rows, ref, l, z
    static_assert(NST >= 2 && SMEM <= 227 * 1024 && O + (FOLD ? 2 : 1) * NR <= 512, "tree kernel resources");
};

struct TreeArgs {
    AttendArgs a;
    const unsigned char *qimg;  // [unit][row block] query images
    const uint64_t *path;       // [batch][64] ancestors and self of each node, 0: no node
    float *records;
    int rows;                   // nodes * group
    int nb;                     // row blocks
    int ntiles, F, groups;      // tiles per unit, of all units, ranges they are cut into
};

// Byte offset of 16-byte chunk c (0..7) of row r in a [rows][128 B] 128-byte-swizzle tile.
__device__ __forceinline__ uint32_t sw128(int r, int c) {
    return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4));
}

// The operands in tensor memory are stored as fragments of 16 lanes x 8 columns: thread (Q, q) = (lane / 4,
// lane % 4) holds columns 2q and 2q + 1 of lanes Q and Q + 8.
//
// K operand (lane = token): thread q takes the q-th quarter of a token's code bytes; its words become column
// pairs as the conversion leaves the codes -- 4 bits: (0,4) (1,5) (2,6) (3,7) of a word's eight, 8 bits: (0,2)
// (1,3) of four -- and its p-th column goes to column 8 (p / 2) + 2q + p % 2.  Position along K of dimension e:
template <int BITS, int D>
__host__ __device__ __forceinline__ int k_position(int e) {
    constexpr int W = 32 / BITS;              // codes per word
    const int q = e / (D / 4), r = e % (D / 4);
    const int p = r / W * (W / 2) + r % (W / 2);
    return 2 * (8 * (p >> 1) + 2 * q + (p & 1)) + (r % W) / (W / 2);
}

// V operand: lane l of a quarter holds dimension 4 (l % 8) + l / 8, so that a thread's four lanes are the codes of
// one 8-byte (4 bits) or 16-byte (8 bits) load of a group of four tokens.
__device__ __forceinline__ int v_dimension(int l) { return 4 * (l & 7) + (l >> 3); }

// Position along K of token t in the V operand: 0 2 1 3 of every four.
__device__ __forceinline__ int v_slot(int t) { return (t & ~3) | ((t & 1) << 1) | ((t >> 1) & 1); }

// Scores keep the codes' mean unless the caller's type is f32: S^T then carries C sum(q^), a few times the score
// itself, whose f32 rounding bf16 and f16 callers cannot see -- and the bare code, zero-extended to 16 bits, is
// the fp16 number c 2^-24, so the K operand takes one operation per pair.  The odd codes of a byte stay in place
// as 16 c, with q^ / 16.
template <typename T>
constexpr bool kCentredScores = std::is_same<T, float>::value;

// Instruction descriptor, kind::f16: D f32, A and B fp16, A K-major, M = 128, N = n; B K-major or
// (mn != 0) with its rows contiguous.
__host__ __device__ constexpr uint32_t tg_idesc(int n, uint32_t mn) {
    return (1u << 4) | (mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTok >> 4) << 24);
}

// Two codes to fp16, less their middle C: a code (or 16 times one) zero-extended to 16 bits is the fp16 number
// c 2^-24 (16 c 2^-24), and (c - C) 2^-9, a half-integer of at most 8 bits, is exact.
constexpr float kCodeUnit = 0x1p-9f;
template <int BITS>
__device__ __forceinline__ uint32_t centred(uint32_t x, uint32_t mask, __half2 up) {
    const uint32_t bare = x & mask;
    const __half2 v = __hfma2(*reinterpret_cast<const __half2 *>(&bare), up,
                              __float2half2_rn(BITS == 4 ? -7.5f * kCodeUnit : -127.5f * kCodeUnit));
    return *reinterpret_cast<const uint32_t *>(&v);
}

__device__ __forceinline__ float tg_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n.reg .b64 ra, rb, rc, rd;\nmov.b64 ra, {%2, %3};\nmov.b64 rb, {%4, %5};\nmov.b64 rc, {%6, %7};\n"
        "fma.rn.f32x2 rd, ra, rb, rc;\nmov.b64 {%0, %1}, rd;\n}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

__device__ __forceinline__ float tg_rcp(float x) {  // within one ulp
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float tg_lg2(float x) {  // absolute error 2^-22
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 ra, rb, rd;\nmov.b64 ra, {%2, %3};\nmov.b64 rb, {%4, %5};\nadd.rn.f32x2 rd, ra, rb;\n"
        "mov.b64 {%0, %1}, rd;\n}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// Arrival of the warp's lane 0, without a branch.
__device__ __forceinline__ void warp_arrive(uint64_t *bar, int lane) {
    asm volatile("{\n.reg .pred p;\nsetp.eq.s32 p, %1, 0;\n@p mbarrier.arrive.shared::cta.b64 _, [%0];\n}\n" ::"r"(
                     smem_u32(bar)),
                 "r"(lane)
                 : "memory");
}

// 16 lanes x 8N columns of tensor memory from fragments (see k_position): v[4m .. 4m + 3] = columns 8m + 2q, + 1
// of lane Q, then of lane Q + 8.
__device__ __forceinline__ void tmem_st_frag4(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};\n" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr));
}

// Registers per thread of this warpgroup (all four warps execute it).
template <int N>
__device__ __forceinline__ void reg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N));
}

// OR of `v` over the 128 threads of a softmax group (named barrier 1 + group).
__device__ __forceinline__ bool group_or(int group, bool v) {
    uint32_t r;
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.u32 q, %1, 0;\nbarrier.cta.red.or.pred p, %2, 128, q;\nselp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(r)
        : "r"((uint32_t)v), "r"(1 + group)
        : "memory");
    return r != 0;
}

// Sum (or maximum) over the warp of N values per lane: lane L returns that of value L % N.
template <int N, typename Op>
__device__ __forceinline__ float warp_columns(float (&v)[N], int lane, Op op) {
#pragma unroll
    for (int h = N / 2; h >= 1; h >>= 1) {
        const bool up = lane & h;
#pragma unroll
        for (int i = 0; i < h; i++) {
            const float mine = up ? v[i + h] : v[i], give = up ? v[i] : v[i + h];
            v[i] = op(mine, __shfl_xor_sync(0xffffffffu, give, h));
        }
    }
#pragma unroll
    for (int h = N; h < 32; h <<= 1) v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], h));
    return v[0];
}

// ---- query images --------------------------------------------------------------------------------
// grid = units * row blocks.  Rows are query rows r = node * G + head of the KV head; a warp rotates
// NR / 16 of them.
template <typename T, int BITS, int D, int NR, int QP>
__global__ void __launch_bounds__(kPrepThreads) tree_prep_kernel(TreeArgs t, unsigned char *qimg, uint64_t *path) {
    using G0 = Tg<BITS, D, NR, QP, 1, false>;
    constexpr int EPL = D / 32, RW = NR / (kPrepThreads / 32);
    const AttendArgs &a = t.a;
    extern __shared__ __align__(16) unsigned char img[];
    __shared__ int s_max, s_min, s_par[kMaxDraftNodes];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int u = blockIdx.x / t.nb, rb = blockIdx.x % t.nb, h = u % a.heads, b = u / a.heads;
    if (tid == 0) {
        s_max = 0;
        s_min = 0x7f800000;
    }
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const int nodes = a.seq_len;
    const int32_t *parents = a.parents + (int64_t)b * nodes;
    if (h == 0 && rb == 0 && tid < nodes) s_par[tid] = parents[tid];
    __syncthreads();
    if (h == 0 && rb == 0 && tid < nodes) path[(int64_t)b * kMaxDraftNodes + tid] = tree_path(s_par, tid);

    const float *sg = a.signs + (int64_t)h * D + lane * EPL;
    const float mul = a.wht_scale * a.scale * 1.4426950408889634f;
    float x[RW][EPL];
    int row_top[RW];  // largest finite |q'| (non-negative floats order as their bits)
    bool present[RW];
    // row r of the KV head is query head g = r % G of node r / G: step over them without a division per row
    const T *src = static_cast<const T *>(a.query) + ((int64_t)b * nodes * a.heads + h) * a.group * D + lane * EPL;
    int g = (rb * NR + warp * RW) % a.group, node = (rb * NR + warp * RW) / a.group;
    src += ((int64_t)node * a.heads * a.group + g) * D;
#pragma unroll
    for (int i = 0; i < RW; i++) {
#pragma unroll
        for (int e = 0; e < EPL; e++) x[i][e] = 0.0f;
        present[i] = false;
        if (node < nodes) {
            load_elems<T, EPL>(src, x[i]);
            const int up = parents[node];
            present[i] = up >= -1 && up < node;
        }
        src += D;
        if (++g == a.group) {
            g = 0;
            node++;
            src += (int64_t)(a.heads - 1) * a.group * D;
        }
    }
#pragma unroll
    for (int i = 0; i < RW; i++) {
#pragma unroll
        for (int e = 0; e < EPL; e++) x[i][e] *= sg[e];
        warp_wht_butterfly<EPL>(x[i], lane, D);
        float top = 0.0f;
#pragma unroll
        for (int e = 0; e < EPL; e++) {
            x[i][e] = present[i] ? x[i][e] * mul : 0.0f;  // (what a slot without a node holds takes no part)
            const float m = fabsf(x[i][e]);
            if (m < INFINITY) top = fmaxf(top, m);
        }
        row_top[i] = __reduce_max_sync(0xffffffffu, __float_as_int(top));
    }
    int most = 0, least = 0x7f800000;
#pragma unroll
    for (int i = 0; i < RW; i++) {
        most = max(most, row_top[i]);
        least = min(least, row_top[i] > 0 ? row_top[i] : 0x7f800000);
    }
    if (lane == 0) {
        atomicMax(&s_max, most);
        atomicMin(&s_min, least);
    }
    __syncthreads();
    // the block's largest |q'| into [2^11, 2^12)
    auto exponent = [](int bits) { return max(((bits >> 23) & 0xff) - 126, -100); };
    const int common = exponent(s_max);
    const bool apart = common - exponent(s_min) > kSpread;  // (rows of zeros aside)
    const float *vtr = a.lr_vtr ? a.lr_vtr + (int64_t)u * D + lane * EPL : nullptr;
    float *qsum = reinterpret_cast<float *>(img + QP * G0::QPLANE);
#pragma unroll
    for (int i = 0; i < RW; i++) {
        const int row = warp * RW + i;
        const int ex = apart ? exponent(row_top[i]) : common;
        const float up = __int_as_float((12 - ex + 127) << 23), down = __int_as_float((ex - 12 + 127) << 23);
        float sum = 0.0f;
        uint32_t hs[EPL];  // hi, and lo above it
#pragma unroll
        for (int e = 0; e < EPL; e++) {
            // (the odd dimensions of 4-bit codes: see kCentredScores)
            const bool sixteenth = BITS == 4 && !kCentredScores<T> && ((lane * EPL + e) & 1);
            const float y = x[i][e] * (sixteenth ? up * 0.0625f : up);
            const __half hi = __float2half_rn(y);
            const float hf = __half2float(hi);
            float kept = hf;
            hs[e] = __half_as_ushort(hi);
            if (QP == 2) {
                const __half lo = __float2half_rn(y - hf);
                hs[e] |= (uint32_t)__half_as_ushort(lo) << 16;
                kept += __half2float(lo);
            }
            if (sixteenth) kept *= 16.0f;
            sum += vtr ? kept * vtr[e] : kept;  // sum(q^), or q^.V^T with low-rank K
        }
        if constexpr (D == 128) {
            // The lane's four dimensions (and, 4 bits, its neighbour's) make pairs of adjacent 32-bit words:
            // 4 bits: lanes 2m and 2m + 1 hold the halves of four words, each stores two; 8 bits: a lane holds both.
            uint32_t first[2], second[2];  // lower and upper halves of the two words
            if constexpr (BITS == 4) {
                const bool odd = lane & 1;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? hs[k] : hs[2 + k], 1);
                    first[k] = odd ? got : hs[k];
                    second[k] = odd ? hs[2 + k] : got;
                }
            } else {
                first[0] = hs[0], first[1] = hs[1];
                second[0] = hs[2], second[1] = hs[3];
            }
            const int p = k_position<BITS, D>(BITS == 4 ? (lane & ~1) * 4 + 2 * (lane & 1) : lane * 4);
            unsigned char *dst = img + (p >> 6) * (NR * 128) + sw128(row, (p & 63) >> 3) + (p & 7) * 2;
            *reinterpret_cast<uint2 *>(dst) =
                make_uint2(__byte_perm(first[0], second[0], 0x5410), __byte_perm(first[1], second[1], 0x5410));
            if (QP == 2)
                *reinterpret_cast<uint2 *>(dst + G0::QPLANE) =
                    make_uint2(__byte_perm(first[0], second[0], 0x7632), __byte_perm(first[1], second[1], 0x7632));
        } else {
#pragma unroll
            for (int e = 0; e < EPL; e++) {
                const int p = k_position<BITS, D>(lane * EPL + e);
                unsigned char *dst = img + (p >> 6) * (NR * 128) + sw128(row, (p & 63) >> 3) + (p & 7) * 2;
                *reinterpret_cast<uint16_t *>(dst) = (uint16_t)hs[e];
                if (QP == 2) *reinterpret_cast<uint16_t *>(dst + G0::QPLANE) = (uint16_t)(hs[e] >> 16);
            }
        }
        sum = warp_sum(sum);
        if (lane == 0) {
            qsum[row] = sum * down;
            qsum[NR + row] = down;
        }
    }
    if (tid < 4) qsum[2 * NR + tid] = apart ? 0.0f : __int_as_float((common - 12 + 127) << 23);
    __syncthreads();
    uint4 *out = reinterpret_cast<uint4 *>(qimg + (int64_t)blockIdx.x * G0::QBUF);
    for (int i = tid; i < G0::QREC / 16; i += kPrepThreads) out[i] = reinterpret_cast<const uint4 *>(img)[i];
}

// ---- attention -------------------------------------------------------------------------------------
template <int BITS, int D, int NR, int QP, int PP, bool F32>
__global__ void __launch_bounds__(Tg<BITS, D, NR, QP, PP, F32>::THREADS, 1) tree_umma_kernel(TreeArgs t) {
    using GG = Tg<BITS, D, NR, QP, PP, F32>;
    constexpr int CB = GG::CB, NST = GG::NST, NC = GG::NC, SM = 4 * GG::NG;
    constexpr float kCentre = BITS == 4 ? 7.5f : 127.5f;
    const AttendArgs &a = t.a;
    extern __shared__ unsigned char tg_raw[];
    unsigned char *smem = tg_raw + ((1024 - (smem_u32(tg_raw) & 1023)) & 1023);
    unsigned char *slots = smem + GG::SLOT_OFF;
    float *ref = reinterpret_cast<float *>(smem + GG::MISC_OFF);       // [NR], minus the reference
    float *fac = ref + 64;                                             // [NR]
    float *red = fac + 64;                                             // [softmax warps][2][NC]
    uint64_t *bars = reinterpret_cast<uint64_t *>(red + 16 * 2 * NC);
    uint64_t *raw_full = bars, *raw_empty = bars + 8, *ka_full = bars + 16, *va_full = bars + 18, *qk_done = bars + 20,
             *pv_done = bars + 22, *p_full = bars + 24, *q_full = bars + 26, *q_empty = bars + 28, *bar_fin = bars + 30;
    uint32_t *tslot = reinterpret_cast<uint32_t *>(bars + 32);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(bars + 33);

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int grp = blockIdx.x / t.nb, rb = blockIdx.x % t.nb;
    const int f0 = (int)((int64_t)grp * t.F / t.groups), f1 = (int)((int64_t)(grp + 1) * t.F / t.groups);
    const int n = f1 - f0, u0 = f0 / t.ntiles, k0 = f0 % t.ntiles;
    const int total = (int)a.pos0 + a.seq_len;

    if (tid == 0) {
        for (int i = 0; i < NST; i++) {
            mbar_init(raw_full + i, 1);
            mbar_init(raw_empty + i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(ka_full + i, 4);
            mbar_init(va_full + i, 4);
            mbar_init(qk_done + i, 1);
            mbar_init(pv_done + i, 1);
            mbar_init(p_full + i, SM);
            mbar_init(q_full + i, 1);
            mbar_init(q_empty + i, 1);
        }
        mbar_init(bar_fin, 1);
        mbar_init(bar_fin + 1, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 0) tmem_alloc(tslot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = *tslot;
    const uint32_t tl = tbase + ((uint32_t)(32 * (warp & 3)) << 16);  // this warp's lane quarter
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");  // the query images and node paths; the drafts in the cache

    auto wait = [&](uint64_t *bar, int phase) {
        const bool ok = um_try(bar, (uint32_t)(phase & 1)) || tc_wait_sleep(bar, (uint32_t)(phase & 1), abort_flag, a.dev_status);
        return (bool)__all_sync(0xffffffffu, ok);
    };

    // one thread's waits (the single-thread roles)
    auto wait1 = [&](uint64_t *bar, int phase) {
        return um_try(bar, (uint32_t)(phase & 1)) || tc_wait_sleep(bar, (uint32_t)(phase & 1), abort_flag, a.dev_status);
    };
    // every MMA this thread issued has completed (before TMEM is freed)
    auto drain = [&](uint64_t *bar) {
        umma_commit(bar);
        const uint64_t tw = um_clock_ns();
        while (!um_try(bar, 0) && um_clock_ns() - tw < kTcWaitNs) {
        }
    };
    if (warp == SM + 8) {
        // ================= copies: one thread =================
        if (lane == 0) {
            int u = u0, kt = k0, units = 0, issued = 0, st = 0, ph = -1;
            const unsigned char *q = t.qimg + ((int64_t)u0 * t.nb + rb) * GG::QBUF;
            int64_t row = (int64_t)u0 * a.capacity + (int64_t)k0 * kTok;
            for (int i = 0; i < n; i++) {
                if (i >= NST && !wait1(raw_empty + st, ph)) break;
                if (i == 0 || kt == 0) {
                    const int qb = units & 1;
                    if (units >= 2 && !wait1(q_empty + qb, units / 2 - 1)) break;
                    mbar_expect_tx(q_full + qb, GG::QREC);
                    bulk_g2s(smem + GG::Q_OFF + qb * GG::QBUF, q, GG::QREC, q_full + qb);
                    q += (int64_t)t.nb * GG::QBUF;
                    units++;
                }
                // the cache holds whole blocks of 64 tokens: a tile's second half may lie past them
                const uint32_t nt = (uint32_t)min(kTok, a.capacity - kt * kTok);
                unsigned char *slot = slots + st * GG::SLOT;
                uint64_t *bar = raw_full + st;
                mbar_expect_tx(bar, nt * (2 * CB + 16));
                bulk_g2s(slot, a.k_codes + row * CB, nt * CB, bar);
                bulk_g2s(slot + kTok * CB, a.v_codes + row * CB, nt * CB, bar);
                bulk_g2s(slot + GG::META, a.k_meta + row * 2, nt * 8, bar);
                bulk_g2s(slot + GG::META + kTok * 8, a.v_meta + row * 2, nt * 8, bar);
                issued = i + 1;
                row += kTok;
                if (++kt == t.ntiles) {
                    kt = 0;
                    row = (int64_t)++u * a.capacity;
                }
                if (++st == NST) {
                    st = 0;
                    ph++;
                }
            }
            if (*abort_flag) {
                // let the copies in flight land before the CTA ends (bounded)
                for (int i = max(0, issued - NST); i < issued; i++)
                    mbar_wait_bounded(raw_full + i % NST, (uint32_t)(i / NST) & 1);
                for (int i = max(0, units - 2); i < units; i++) mbar_wait_bounded(q_full + (i & 1), (uint32_t)(i / 2) & 1);
            }
        }
    } else if (warp == SM + 9) {
        // ================= S^T: one thread =================
        if (lane == 0) {
            constexpr uint32_t id_s = tg_idesc(NR, 0);
            int kt = k0, units = 0;
            const uint64_t q0 = sw128_kmajor_desc(smem_u32(smem + GG::Q_OFF));
            for (int i = 0; i < n; i++) {
                if (!wait1(ka_full + (i & 1), i >> 1)) break;
                // O^T(i - 2) complete: the softmax had read S^T(i - 2), whose buffer this takes, and with S^T(i) the
                // softmax knows that u's buffer is free
                if (i >= 2 && !wait1(pv_done + (i & 1), (i >> 1) - 1)) break;
                if (i == 0 || kt == 0) {
                    if (!wait1(q_full + (units & 1), units >> 1)) break;
                    units++;
                }
                tc_fence_after();
                const uint64_t q = q0 + (((units - 1) & 1) * (GG::QBUF >> 4));  // start addresses count 16 bytes
                const uint32_t d = tbase + GG::S + (i & 1) * NR, k = tbase + GG::KA + (i & 1) * (D / 2);
#pragma unroll
                for (int pl = QP - 1; pl >= 0; pl--)  // the low plane first, while the sums that its steps round are small
#pragma unroll
                    for (int kk = 0; kk < D / 16; kk++)
                        umma_ts(d, k + 8 * kk, q + ((pl * GG::QPLANE + (kk >> 2) * (NR * 128) + 32 * (kk & 3)) >> 4), id_s,
                                pl != QP - 1 || kk != 0 ? 1u : 0u);
                umma_commit(qk_done + (i & 1));
                if (++kt == t.ntiles) kt = 0;
            }
            drain(bar_fin);
        }
    } else if (warp == SM + 10) {
        // ================= O^T: one thread =================
        if (lane == 0) {
            constexpr uint32_t id_o = tg_idesc(NR, 1);
            int kt = k0, units = 0, st = 0;
            const uint64_t p0 = sw128_kmajor_desc(smem_u32(smem + GG::P_OFF));
            for (int i = 0; i < n; i++) {
                const bool starts = i == 0 || kt == 0;
                if (starts) units++;
                if (!wait1(va_full + (i & 1), i >> 1) || !wait1(p_full + (i & 1), i >> 1)) break;
                tc_fence_after();
                // B: rows contiguous, 8-token groups 1024 B apart -- the same fields as a K-major tile
                const uint64_t p = p0 + ((i & 1) * (GG::PBUF >> 4));
                const uint32_t v = tbase + GG::VA + (i & 1) * (kTok / 2);
#pragma unroll
                for (int pl = PP - 1; pl >= 0; pl--)
#pragma unroll
                    for (int kk = 0; kk < kTok / 16; kk++)
                        umma_ts(tbase + GG::O + (GG::FOLD ? (i & 1) * NR : 0), v + 8 * kk,
                                p + ((pl * (kTok * 128) + 2048 * kk) >> 4), id_o,
                                pl != PP - 1 || kk != 0 || !(GG::FOLD || starts) ? 1u : 0u);
                umma_commit(pv_done + (i & 1));
                // every role is past tile i: its ring slot, and after the unit's last tile its queries, are free
                umma_commit(raw_empty + st);
                if (kt == t.ntiles - 1) umma_commit(q_empty + ((units - 1) & 1));
                if (++kt == t.ntiles) kt = 0;
                if (++st == NST) st = 0;
            }
            drain(bar_fin + 1);
        }
    } else if (warp >= SM + 4) {
        // ================= V codes -> fp16 =================
        if constexpr (GG::SPLIT) reg_dec<GG::STAGE>();
        const int Q = lane >> 2, q = lane & 3;
        const bool live = 32 * (warp & 3) < D;
        const __half2 low = __float2half2_rn(0x1p15f), high = __float2half2_rn(0x1p11f);  // of a byte's codes
        for (int i = 0, st = 0, ph = 0; i < n; i++) {
            if (!wait(raw_full + st, ph)) break;
            if (i >= 2 && !wait(pv_done + (i & 1), (i >> 1) - 1)) break;
            tc_fence_after();
            if (live) {
                // group q of a 16-token block, dimensions 32 w + 4 Q .. + 3
                const unsigned char *src = slots + st * GG::SLOT + kTok * CB + 16 * q +
                                           (BITS == 4 ? (4 * (warp & 3) + (Q >> 1)) * 64 + (Q & 1) * 8
                                                      : (8 * (warp & 3) + Q) * 64);
                const uint32_t dst = tl + GG::VA + (i & 1) * (kTok / 2);
#pragma unroll 1  // (the roles' loops share the instruction caches)
                for (int half = 0; half < 2; half++) {
                    uint32_t v0[16], v1[16];  // lanes Q and Q + 8; Q + 16 and Q + 24
#pragma unroll
                    for (int m = 0; m < 4; m++) {
                        const unsigned char *blk = src + (4 * half + m) * (16 * CB);
                        if constexpr (BITS == 4) {
                            const uint2 w = *reinterpret_cast<const uint2 *>(blk);
                            v0[4 * m] = centred<BITS>(w.x, 0x000f000fu, low);
                            v0[4 * m + 1] = centred<BITS>(w.x >> 8, 0x000f000fu, low);
                            v0[4 * m + 2] = centred<BITS>(w.x, 0x00f000f0u, high);
                            v0[4 * m + 3] = centred<BITS>(w.x >> 8, 0x00f000f0u, high);
                            v1[4 * m] = centred<BITS>(w.y, 0x000f000fu, low);
                            v1[4 * m + 1] = centred<BITS>(w.y >> 8, 0x000f000fu, low);
                            v1[4 * m + 2] = centred<BITS>(w.y, 0x00f000f0u, high);
                            v1[4 * m + 3] = centred<BITS>(w.y >> 8, 0x00f000f0u, high);
                        } else {
                            const uint4 w = *reinterpret_cast<const uint4 *>(blk);
                            const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                            for (int y = 0; y < 4; y++) {
                                uint32_t *v = y < 2 ? v0 : v1;
                                v[4 * m + 2 * (y & 1)] = centred<BITS>(x[y], 0x00ff00ffu, low);
                                v[4 * m + 2 * (y & 1) + 1] =
                                    centred<BITS>(x[y] >> 8, 0x00ff00ffu, low);
                            }
                        }
                    }
                    tmem_st_frag4(dst + 32 * half, v0);
                    tmem_st_frag4(dst + 32 * half + (16u << 16), v1);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            warp_arrive(va_full + (i & 1), lane);
            if (++st == NST) st = 0, ph ^= 1;
        }
    } else if (warp >= SM) {
        // ================= K codes -> fp16, token constants =================
        if constexpr (GG::SPLIT) reg_dec<GG::STAGE>();
        const int Q = lane >> 2, q = lane & 3, tok = 32 * (warp & 3) + lane;
        constexpr int QB = CB / 4, NW = QB / 4;  // bytes and words of a quarter of a token's codes
        constexpr bool KC = F32;                 // kCentredScores
        const __half2 low = __float2half2_rn(0x1p15f), high = __float2half2_rn(0x1p11f);  // of a byte's codes
        for (int i = 0, st = 0, ph = 0; i < n; i++) {
            if (!wait(raw_full + st, ph)) break;
            if (i >= 2 && !wait(qk_done + (i & 1), (i >> 1) - 1)) break;
            tc_fence_after();
            unsigned char *slot = slots + st * GG::SLOT;
            {
                const float2 km = *reinterpret_cast<const float2 *>(slot + GG::META + tok * 8);
                const float2 vm = *reinterpret_cast<const float2 *>(slot + GG::META + kTok * 8 + tok * 8);
                const float vs = vm.x < kScaleMin ? kScaleMin : vm.x, rv = tg_rcp(vs);
                *reinterpret_cast<float4 *>(slot + GG::CONST + tok * 16) =
                    KC ? make_float4(km.x * (1.0f / kCodeUnit), fmaf(kCentre, km.x, km.y), tg_lg2(vs), rv)
                       : make_float4(km.x * 0x1p24f, km.y, tg_lg2(vs), rv);
                *reinterpret_cast<float *>(slot + GG::CONST + kTok * 16 + tok * 4) = fmaf(kCentre, vs, vm.y) * rv;
            }
            const unsigned char *src = slot + (32 * (warp & 3) + Q) * CB + q * QB;
            const uint32_t dst = tl + GG::KA + (i & 1) * (D / 2);
            // tokens Q, Q + 8 of 16 at a time, 16 registers (8 columns by 4 column blocks) at a time
#pragma unroll 1
            for (int half = 0; half < 2; half++) {
                uint32_t w[2][NW];
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const unsigned char *row = src + (16 * half + 8 * y) * CB;
                    if constexpr (QB == 8) {
                        const uint2 x = *reinterpret_cast<const uint2 *>(row);
                        w[y][0] = x.x;
                        w[y][1] = x.y;
                    } else {
#pragma unroll
                        for (int x = 0; x < QB / 16; x++) {
                            const uint4 t4 = reinterpret_cast<const uint4 *>(row)[x];
                            w[y][4 * x] = t4.x;
                            w[y][4 * x + 1] = t4.y;
                            w[y][4 * x + 2] = t4.z;
                            w[y][4 * x + 3] = t4.w;
                        }
                    }
                }
                // columns 2m, 2m + 1 of the thread (of D / 8 in all) go to column block m
#pragma unroll
                for (int m0 = 0; m0 < D / 16; m0 += 4) {
                    uint32_t v[16];
#pragma unroll
                    for (int m = 0; m < 4; m++)
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            if constexpr (BITS == 4) {
                                const uint32_t x = w[y][(m0 + m) >> 1] >> ((m & 1) * 8);
                                v[4 * m + 2 * y] = KC ? centred<BITS>(x, 0x000f000fu, low) : x & 0x000f000fu;
                                v[4 * m + 2 * y + 1] =
                                    KC ? centred<BITS>(x, 0x00f000f0u, high) : x & 0x00f000f0u;
                            } else {
                                const uint32_t x = w[y][m0 + m];
                                v[4 * m + 2 * y] = KC ? centred<BITS>(x, 0x00ff00ffu, low) : x & 0x00ff00ffu;
                                v[4 * m + 2 * y + 1] = KC ? centred<BITS>(x >> 8, 0x00ff00ffu, low)
                                                          : __byte_perm(x, 0, 0x4341);
                            }
                        }
                    tmem_st_frag4(dst + 8 * m0 + (half ? 16u << 16 : 0u), v);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            warp_arrive(ka_full + (i & 1), lane);
            if (++st == NST) st = 0, ph ^= 1;
        }
    } else {
        // ================= softmax: thread = token, NC rows =================
        if constexpr (GG::SPLIT) reg_inc<GG::SOFT>();
        const int group = warp >> 2, wq = warp & 3, c0 = group * NC;
        const int tok = 32 * wq + lane, slot_row = v_slot(tok);
        float *gref = ref + c0, *gfac = fac + c0;
        float *my_red = red + warp * 2 * NC, *grp_red = red + group * 8 * NC;
        unsigned char *pl = smem + GG::P_OFF + (slot_row >> 3) * 1024 + (slot_row & 7) * 128;
        const int ch0 = (group * (NC / 8)) << 4, chx = (slot_row & 7) << 4;  // 16-byte chunk c of its row: (ch0 + 16 c) ^ chx
        int plain_tiles = 0;                               // tiles of the unit that need no raise of themselves
        int u = u0, kt = k0, units = 0;
        int slot = 0;                                      // ring slot of the tile
        int buf = 0, phase = 0;                            // buffer i & 1 and its phase (i >> 1) & 1
        int left = min(n, t.ntiles - k0), rest = n - left;  // tiles to the end of the unit, or of the range; after it
        bool starts = true;                                // the unit's first tile here
        const float *qsum = nullptr;
        float l[NC], z[NC];
        [[maybe_unused]] float o[GG::FOLD ? NC : 8];       // FOLD: the unit's O of dimension `tok`
        auto fold = [&](int b) {
#pragma unroll
            for (int c = 0; c < (GG::FOLD ? NC : 8); c += 8) {
                uint32_t x[8];
                tmem_ld8(tl + GG::O + b * NR + c0 + c, x);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 8; k++) o[c + k] += __uint_as_float(x[k]);
            }
        };
        while (left > 0) {
            // S^T(i); with it the token constants are in place (the K warps wrote them before) and O^T(i - 2),
            // which the S^T warp waited for, is complete: u's buffer is free
            bool ok = wait(qk_done + buf, phase);
            if (__builtin_expect(starts, 0)) {
                if (ok) ok = wait(q_full + (units & 1), units >> 1);
                qsum = reinterpret_cast<const float *>(smem + GG::Q_OFF + (units & 1) * GG::QBUF + QP * GG::QPLANE) + c0;
                units++;
                if (ok) plain_tiles = qsum[2 * NR - c0] == 0.0f ? 0 : (int)a.pos0 / kTok;
#pragma unroll
                for (int c = 0; c < NC; c++) l[c] = z[c] = 0.0f;
                if constexpr (GG::FOLD) {
#pragma unroll
                    for (int c = 0; c < NC; c++) o[c] = 0.0f;
                }
                if (wq == 0 && lane < NC) gref[lane] = INFINITY;  // no token seen yet
                if (group_or(group, !ok)) break;  // (also: the references are written)
            }
            tc_fence_after();
            const unsigned char *consts = slots + slot * GG::SLOT + GG::CONST;
            uint32_t v[NC];
            auto load = [&]() { tmem_ld16(tl + GG::S + buf * NR + c0, v); };
            // S^T in the rows' own powers of two
            auto load_by_row = [&]() {
                load();
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < NC; c++) v[c] = __float_as_uint(__uint_as_float(v[c]) * qsum[NR + c]);
            };
            load();
            // drafts in the tile, or tokens past them: bit c of `sees`: row c sees this token
            const bool masked = (kt + 1) * kTok > (int)a.pos0;  // (the tiles before are seen whole)
            uint32_t sees = 0xffffffffu;
            if (__builtin_expect(masked, 0)) {
                const int pos = kt * kTok + tok, dj = pos - (int)a.pos0;
                if (dj >= 0) {
                    const uint64_t *path = t.path + (int64_t)(u / a.heads) * kMaxDraftNodes;
                    sees = 0;
                    if (pos < total) {
#pragma unroll 1
                        for (int c = 0; c < NC; c++) {
                            const int node = (rb * NR + c0 + c) / a.group;
                            if (node < a.seq_len && ((path[node] >> dj) & 1)) sees |= 1u << c;
                        }
                    }
                }
            }
            const float4 tc = *reinterpret_cast<const float4 *>(consts + tok * 16);
            const float zv = *reinterpret_cast<const float *>(consts + kTok * 16 + tok * 4);
            const float rv = tc.w;
            float ks = tc.x * qsum[2 * NR - c0];
            const float2 kz2 = make_float2(tc.y, tc.y), lv2 = make_float2(tc.z, tc.z);
            unsigned char *dst = pl + buf * GG::PBUF;
            // w = u = vs 2^(s - ref), which also goes to shared memory -- or, raising, the scores themselves; returns the
            // largest score.  u is computed before the vote on its range, so that the exponentials overlap the scores'
            // arithmetic (1.15 times as fast at 64 rows); a raise does it over.
            float w[NC];
            auto pass = [&](auto raising, auto masking) {
                constexpr bool RAISE = decltype(raising)::value, MASK = decltype(masking)::value;
                const float2 ks2 = make_float2(ks, ks);
                float top0 = -INFINITY, top1 = -INFINITY;
                tmem_wait_ld();
#pragma unroll
                for (int hf = 0; hf < NC / 8; hf++) {
                    [[maybe_unused]] uint32_t uh[4], ul[4];
#pragma unroll
                    for (int c = 0; c < 8; c += 4) {
                        const float4 q4 = *reinterpret_cast<const float4 *>(qsum + 8 * hf + c);
                        float4 r4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (!RAISE) r4 = *reinterpret_cast<const float4 *>(gref + 8 * hf + c);  // minus the reference
                        const float2 b0 = fma2(kz2, make_float2(q4.x, q4.y), add2(make_float2(r4.x, r4.y), lv2));
                        const float2 b1 = fma2(kz2, make_float2(q4.z, q4.w), add2(make_float2(r4.z, r4.w), lv2));
                        const float2 s0 = fma2(make_float2(__uint_as_float(v[8 * hf + c]), __uint_as_float(v[8 * hf + c + 1])), ks2, b0);
                        const float2 s1 = fma2(make_float2(__uint_as_float(v[8 * hf + c + 2]), __uint_as_float(v[8 * hf + c + 3])), ks2, b1);
                        float e[4] = {s0.x, s0.y, s1.x, s1.y};
                        if constexpr (MASK) {
#pragma unroll
                            for (int x = 0; x < 4; x++)
                                if (!((sees >> (8 * hf + c + x)) & 1)) e[x] = -INFINITY;
                        }
                        top0 = fmaxf(top0, fmaxf(e[0], e[1]));
                        top1 = fmaxf(top1, fmaxf(e[2], e[3]));
#pragma unroll
                        for (int x = 0; x < 4; x++) w[8 * hf + c + x] = RAISE ? e[x] : tg_ex2(e[x]);
                        if constexpr (!RAISE) {
#pragma unroll
                            for (int x = 0; x < 4; x += 2) {
                                const float2 u2 = make_float2(w[8 * hf + c + x], w[8 * hf + c + x + 1]);
                                const __half2 hh = __floats2half2_rn(u2.x, u2.y);
                                uh[(c + x) / 2] = *reinterpret_cast<const uint32_t *>(&hh);
                                if constexpr (PP == 2) {
                                    const float2 back = __half22float2(hh);
                                    const __half2 ll = __floats2half2_rn(u2.x - back.x, u2.y - back.y);
                                    ul[(c + x) / 2] = *reinterpret_cast<const uint32_t *>(&ll);
                                }
                            }
                        }
                    }
                    if constexpr (!RAISE) {
                        *reinterpret_cast<uint4 *>(dst + ((ch0 + 16 * hf) ^ chx)) = make_uint4(uh[0], uh[1], uh[2], uh[3]);
                        if constexpr (PP == 2)
                            *reinterpret_cast<uint4 *>(dst + kTok * 128 + ((ch0 + 16 * hf) ^ chx)) =
                                make_uint4(ul[0], ul[1], ul[2], ul[3]);
                    }
                }
                return fmaxf(top0, top1);
            };
            // A unit's first tile, and one with a score that outgrew its reference, raise the references to the tile's
            // maxima first (so do tiles where rows may see their first token, and all of a row block spread wide).
            bool failed = false, folded = starts;
            for (bool raise = starts || kt >= plain_tiles;;) {
                if (__builtin_expect(!raise, 1)) {
                    const float top = pass(std::false_type{}, std::false_type{});  // (a masked tile raises)
                    if (__builtin_expect(!group_or(group, !ok || top > kHead + kShift), 1)) break;
                }
                if (ok && !starts) ok = wait(pv_done + (buf ^ 1), phase ^ (buf ^ 1));  // O^T(i - 1): O is at rest
                if (group_or(group, !ok)) {
                    failed = true;
                    break;
                }
                tc_fence_after();
                if constexpr (GG::FOLD) {
                    if (!starts) fold(buf ^ 1);
                    folded = true;
                }
                load_by_row();
                ks = *reinterpret_cast<const float *>(consts + tok * 16);
                if (masked) pass(std::true_type{}, std::true_type{});
                else pass(std::true_type{}, std::false_type{});
                // (8 columns at a time: few registers beside the hot path's)
#pragma unroll
                for (int c = 0; c < NC; c += 8) {
                    float m[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) m[k] = w[c + k];
                    const float cm = warp_columns(m, lane, [](float x, float y) { return fmaxf(x, y); });
                    if (lane < 8) my_red[c + lane] = cm;  // (the group's last reads of it are behind a barrier)
                }
                group_or(group, false);
                if (wq == 0 && lane < NC) {
                    const float old = -gref[lane];
                    float m = old + kShift;
#pragma unroll
                    for (int x = 0; x < 4; x++) m = fmaxf(m, grp_red[x * 2 * NC + lane]);
                    gfac[lane] = old == -INFINITY ? 0.0f : exp2f(old - (m - kShift));
                    gref[lane] = kShift - m;
                }
                group_or(group, false);
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    l[c] *= gfac[c];
                    z[c] *= gfac[c];
                }
                if constexpr (GG::FOLD) {
#pragma unroll
                    for (int c = 0; c < NC; c++) o[c] *= gfac[c];
                } else if (!starts) {
#pragma unroll 1
                    for (int c = 0; c < NC; c += 8) {
                        uint32_t o[8];
                        tmem_ld8(tl + GG::O + c0 + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 8; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * gfac[c + k]);
                        tmem_st8(tl + GG::O + c0 + c, o);
                    }
                    tmem_wait_st();
                }
                load_by_row();
                if (masked) pass(std::false_type{}, std::true_type{});
                else pass(std::false_type{}, std::false_type{});
                break;
            }
            if (failed) break;
            tc_fence_before();
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            warp_arrive(p_full + buf, lane);  // (and the last reads of the ring slot are behind)
            const float2 rv2 = make_float2(rv, rv), zv2 = make_float2(zv, zv);
            // ---- the token's sums; an unseen token takes no part, whatever its metadata holds ----
            if (__builtin_expect(masked, 0)) {
#pragma unroll
                for (int c = 0; c < NC; c++)
                    if ((sees >> c) & 1) {
                        l[c] = fmaf(w[c], rv, l[c]);
                        z[c] = fmaf(w[c], zv, z[c]);
                    }
            } else {
#pragma unroll
                for (int c = 0; c < NC; c += 2) {
                    const float2 w2 = make_float2(w[c], w[c + 1]);
                    const float2 l2 = fma2(w2, rv2, make_float2(l[c], l[c + 1]));
                    const float2 z2 = fma2(w2, zv2, make_float2(z[c], z[c + 1]));
                    l[c] = l2.x;
                    l[c + 1] = l2.y;
                    z[c] = z2.x;
                    z[c + 1] = z2.y;
                }
            }
            if constexpr (GG::FOLD) {
                if (!folded) {
                    ok = wait(pv_done + (buf ^ 1), phase ^ (buf ^ 1));  // O^T(i - 1)
                    tc_fence_after();
                    fold(buf ^ 1);  // (the next arrival at p_full orders it before O^T(i + 1))
                }
            }
            kt++;
            if (++slot == NST) slot = 0;
            starts = false;
            if (__builtin_expect(--left == 0, 0)) {
                // ---- the unit's partial record ----
                const float lc = warp_columns(l, lane, [](float x, float y) { return x + y; });
                const float zc = warp_columns(z, lane, [](float x, float y) { return x + y; });
                if (lane < NC) {
                    my_red[lane] = lc;
                    my_red[NC + lane] = zc;
                }
                ok = ok && wait(pv_done + buf, phase);
                if (group_or(group, !ok)) break;
                tc_fence_after();
                float *rec = t.records + ((int64_t)(grp + u) * t.nb + rb) * GG::REC;
                if (wq == 0 && lane < NC) {
                    float ls = 0.0f, zs = 0.0f;
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        ls += grp_red[w * 2 * NC + lane];
                        zs += grp_red[w * 2 * NC + NC + lane];
                    }
                    rec[NR * D + c0 + lane] = -gref[lane];
                    rec[NR * D + NR + c0 + lane] = ls;
                    rec[NR * D + 2 * NR + c0 + lane] = zs;
                }
                const int dim = 32 * wq + v_dimension(lane);
                if constexpr (GG::FOLD) {
                    fold(buf);
                    if (tok < D) {  // tok is the lane of O
#pragma unroll
                        for (int c = 0; c < NC; c++) rec[(c0 + c) * D + dim] = o[c] * (1.0f / kCodeUnit);
                    }
                } else {
#pragma unroll 1
                    for (int c = 0; c < NC; c += 8) {
                        uint32_t v[8];
                        tmem_ld8(tl + GG::O + c0 + c, v);
                        tmem_wait_ld();
                        if (tok < D) {
#pragma unroll
                            for (int k = 0; k < 8; k++)
                                rec[(c0 + c + k) * D + dim] = __uint_as_float(v[k]) * (1.0f / kCodeUnit);
                        }
                    }
                }
                tc_fence_before();
                group_or(group, false);  // my_red and gref are read before the next unit writes them
                kt = 0;
                u++;
                left = min(rest, t.ntiles);
                rest -= left;
                starts = true;
            }
            phase ^= buf;
            buf ^= 1;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tbase, 512);
    }
}

// ---- merge -------------------------------------------------------------------------------------------
// Range that holds flat tile f when F tiles are cut into `groups` ranges [w F / groups, (w + 1) F / groups).
__device__ __forceinline__ int range_of(int64_t f, int F, int groups) {
    const int64_t x = (f + 1) * groups - 1;
    int w = (int)((float)x / (float)F);  // the guess is off by one at most per 2^23: stepped to the exact one
    while ((int64_t)(w + 1) * F <= x) w++;
    while ((int64_t)w * F > x) w--;
    return w;
}

// A warp joins the records of PER query rows, rotates back and stores: one row where warps are few, four
// records' loads at a time; four rows where they are many, whose loads go out together when the unit has one
// record (a tree of 448 rows over 255 tokens, 440 units: 109 us with one row per warp, 57 with four).
template <typename T, int BITS, int D, int NR, int PER>
__global__ void __launch_bounds__(32 * kMergeWarps) tree_merge_kernel(TreeArgs t) {
    constexpr int EPL = D / 32, REC = NR * D + 3 * NR, BATCH = 4;
    const AttendArgs &a = t.a;
    const int lane = threadIdx.x & 31;
    const int u = blockIdx.x, h = u % a.heads, b = u / a.heads;
    const int r0 = (blockIdx.y * kMergeWarps + (threadIdx.x >> 5)) * PER;
    const float *sg = a.signs + (int64_t)h * D + lane * EPL;
    float sgw[EPL];
#pragma unroll
    for (int e = 0; e < EPL; e++) sgw[e] = a.wht_scale * sg[e];
    // ranges that touch tiles [u ntiles, (u + 1) ntiles)
    const int lo = range_of((int64_t)u * t.ntiles, t.F, t.groups);
    const int hi = range_of((int64_t)(u + 1) * t.ntiles - 1, t.F, t.groups);
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    if (r0 >= t.rows) return;
    const float *unit = t.records + (int64_t)(lo + u) * t.nb * REC;
    // row r's place in the output, and whether its slot holds a node: asked for before the records
    auto place = [&](int r, T *&dst, bool &present) {
        const int node = r / a.group, g = r % a.group;
        dst = static_cast<T *>(a.out) + (((int64_t)b * a.seq_len + node) * (a.heads * a.group) + h * a.group + g) * D +
              lane * EPL;
        present = t.path[(int64_t)b * kMaxDraftNodes + node] != 0;
    };
    auto finish = [&](T *dst, bool present, float (&x)[EPL], float L, float Z) {
        const float inv = 1.0f / L;  // a node sees itself
#pragma unroll
        for (int e = 0; e < EPL; e++) x[e] = (x[e] + Z) * inv;
        warp_wht_butterfly<EPL>(x, lane, D);
#pragma unroll
        for (int e = 0; e < EPL; e++) x[e] = present ? x[e] * sgw[e] : 0.0f;  // zero where the slot holds no node
        if (EPL == 4 && sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(dst) & 7) == 0) {
            union {
                T t[4];
                uint2 v;
            } o;
#pragma unroll
            for (int e = 0; e < EPL && e < 4; e++) o.t[e] = DT<T>::from_f32(x[e]);
            *reinterpret_cast<uint2 *>(dst) = o.v;
        } else {
#pragma unroll
            for (int e = 0; e < EPL; e++) st_from_f32(dst + e, x[e]);
        }
    };
    if (PER > 1 && lo == hi) {
        float l[PER], z[PER], y[PER][EPL];
        T *dst[PER];
        bool present[PER];
#pragma unroll
        for (int k = 0; k < PER; k++) {
            const int r = min(r0 + k, t.rows - 1), rb = r / NR, rr = r % NR;
            const float *rec = unit + (int64_t)rb * REC;
            place(r, dst[k], present[k]);
            l[k] = rec[NR * D + NR + rr];
            z[k] = rec[NR * D + 2 * NR + rr];
            load_elems<float, EPL>(rec + rr * D + lane * EPL, y[k]);
        }
#pragma unroll
        for (int k = 0; k < PER; k++)
            if (r0 + k < t.rows) finish(dst[k], present[k], y[k], l[k], z[k]);
        return;
    }
    const int64_t step = (int64_t)t.nb * REC;
#pragma unroll 1
    for (int r = r0; r < r0 + PER; r++) {
        if (PER > 1 && r >= t.rows) return;
        const int rb = r / NR, rr = r % NR;
        const float *rec0 = unit + (int64_t)rb * REC;
        T *dst;
        bool present;
        place(r, dst, present);
        float M = -INFINITY, L = 0.0f, Z = 0.0f, x[EPL];
#pragma unroll
        for (int e = 0; e < EPL; e++) x[e] = 0.0f;
        for (int w0 = lo; w0 <= hi; w0 += BATCH, rec0 += BATCH * step) {
            float m[BATCH], l[BATCH], z[BATCH], y[BATCH][EPL];
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
                m[k] = -INFINITY;
                l[k] = z[k] = 0.0f;
                if (w0 + k <= hi) {
                    const float *rec = rec0 + k * step;
                    m[k] = rec[NR * D + rr];
                    l[k] = rec[NR * D + NR + rr];
                    z[k] = rec[NR * D + 2 * NR + rr];
                    load_elems<float, EPL>(rec + rr * D + lane * EPL, y[k]);
                } else {
#pragma unroll
                    for (int e = 0; e < EPL; e++) y[k][e] = 0.0f;
                }
            }
            float top = M;
#pragma unroll
            for (int k = 0; k < BATCH; k++)
                if (l[k] != 0.0f) top = fmaxf(top, m[k]);  // (a range that showed the row no token has a sum of zero)
            const float f = M == -INFINITY ? 0.0f : exp2f(M - top);
            L *= f;
            Z *= f;
#pragma unroll
            for (int e = 0; e < EPL; e++) x[e] *= f;
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
                const float wt = l[k] == 0.0f ? 0.0f : exp2f(m[k] - top);
                L = fmaf(wt, l[k], L);
                if (wt != 0.0f) {  // (what a row without tokens left is not read)
                    Z = fmaf(wt, z[k], Z);
#pragma unroll
                    for (int e = 0; e < EPL; e++) x[e] = fmaf(wt, y[k][e], x[e]);
                }
            }
            M = top;
        }
        finish(dst, present, x, L, Z);
    }
}

// ---- host ----------------------------------------------------------------------------------------------
size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Shape of a launch over `batch` sequences.
struct TreePlan {
    int nr, nb, groups, ntiles, F;
    size_t records, qimg, path;  // workspace parts, in this order
};

// Planes of q^ and u.
int tree_planes(int dtype, int full) { return dtype == SA_DTYPE_BFLOAT16 && !full ? 1 : 2; }

TreePlan tree_plan(int64_t batch, int heads, int group, int head_dim, int sm_count, int64_t total, int nodes, int dtype,
                   int full) {
    TreePlan p;
    const int rows = nodes * group;
    p.nr = rows <= 16 ? 16 : rows <= 32 || dtype == SA_DTYPE_FLOAT ? 32 : 64;  // (f32: the sums of O take the registers of the other 32)
    p.nb = (rows + p.nr - 1) / p.nr;
    p.ntiles = (int)((total + kTok - 1) / kTok);
    const int64_t units = batch * heads;
    p.F = (int)(units * p.ntiles);
    const int most = sm_count / p.nb > 0 ? sm_count / p.nb : 1;
    p.groups = p.F < most ? p.F : most;
    p.records = up256((size_t)(p.groups + units) * p.nb * (p.nr * head_dim + 3 * p.nr) * sizeof(float));
    const size_t image = ((size_t)tree_planes(dtype, full) * p.nr * head_dim * 2 + p.nr * 8 + 16 + 1023) / 1024 * 1024;
    p.qimg = (size_t)units * p.nb * image;
    p.path = up256((size_t)batch * kMaxDraftNodes * sizeof(uint64_t));
    return p;
}

// Sequences of one launch: bounds the workspace (a row block's record takes up to 33.5 KB).
int64_t tree_batch(int64_t batch, int heads, int group, int nodes) {
    const int64_t blocks = (int64_t)heads * ((nodes * group + 63) / 64);
    const int64_t most = 4096 / blocks > 0 ? 4096 / blocks : 1;
    return batch < most ? batch : most;
}

template <typename T, int BITS, int D, int NR, int QP, int PP>
int launch_rows(const TreeArgs &t, unsigned char *qimg, uint64_t *path, cudaStream_t stream) {
    constexpr bool F32 = std::is_same<T, float>::value;
    using GG = Tg<BITS, D, NR, QP, PP, F32>;
    const int64_t units = (int64_t)t.a.batch * t.a.heads;
    // each launch is a programmatic dependent of the one before it
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)(units * t.nb));
    cfg.blockDim = dim3(kPrepThreads);
    cfg.dynamicSmemBytes = GG::QREC;
    int rc = check_cuda(cudaLaunchKernelEx(&cfg, tree_prep_kernel<T, BITS, D, NR, QP>, t, qimg, path),
                        "gqa_tree_attend prep launch");
    count_launch();
    if (rc != SA_OK) return rc;
    auto kern = tree_umma_kernel<BITS, D, NR, QP, PP, F32>;
    static int configured[64];  // of this kernel, by device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !__atomic_load_n(&configured[dev], __ATOMIC_ACQUIRE)) {
        cudaFuncAttributes fa;
        cudaError_t e = cudaFuncGetAttributes(&fa, kern);
        if (e == cudaSuccess && GG::SPLIT && fa.numRegs < GG::LAUNCH)  // the split would wait for registers that are not there
            return set_error(SA_ERR_CUDA, "gqa_tree_attend: compiled to %d registers, the split needs %d", fa.numRegs,
                             GG::LAUNCH);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, GG::SMEM);
        if (e != cudaSuccess) return check_cuda(e, "gqa_tree_attend smem attribute");
        if (dev >= 0 && dev < 64) __atomic_store_n(&configured[dev], 1, __ATOMIC_RELEASE);
    }
    cfg.gridDim = dim3((unsigned)(t.groups * t.nb));
    cfg.blockDim = dim3(GG::THREADS);
    cfg.dynamicSmemBytes = GG::SMEM;
    rc = check_cuda(cudaLaunchKernelEx(&cfg, kern, t), "gqa_tree_attend launch");
    count_launch();
    if (rc != SA_OK) return rc;
    const bool many = units * t.rows > 128 * t.a.sm_count;  // (a GPU of warps, twice over)
    const int rows = kMergeWarps * (many ? 4 : 1);
    cfg.gridDim = dim3((unsigned)units, (unsigned)((t.rows + rows - 1) / rows));
    cfg.blockDim = dim3(32 * kMergeWarps);
    cfg.dynamicSmemBytes = 0;
    rc = check_cuda(cudaLaunchKernelEx(&cfg, many ? tree_merge_kernel<T, BITS, D, NR, 4> : tree_merge_kernel<T, BITS, D, NR, 1>, t),
                    "gqa_tree_attend merge launch");
    count_launch();
    return rc;
}

template <typename T, int PL, int BITS, int D>
int launch_format(const TreeArgs &t, int nr, unsigned char *qimg, uint64_t *path, cudaStream_t stream) {
    if (nr == 16) return launch_rows<T, BITS, D, 16, PL, PL>(t, qimg, path, stream);
    if (nr == 32) return launch_rows<T, BITS, D, 32, PL, PL>(t, qimg, path, stream);
    if constexpr (!std::is_same<T, float>::value) return launch_rows<T, BITS, D, 64, PL, PL>(t, qimg, path, stream);
    return set_error(SA_ERR_CUDA, "gqa_tree_attend: no kernel of %d rows", nr);
}

template <typename T, int PL>
int launch_type(const TreeArgs &t, int nr, unsigned char *qimg, uint64_t *path, cudaStream_t stream) {
    if (t.a.bits == 4 && t.a.head_dim == 128) return launch_format<T, PL, 4, 128>(t, nr, qimg, path, stream);
    if (t.a.bits == 8 && t.a.head_dim == 128) return launch_format<T, PL, 8, 128>(t, nr, qimg, path, stream);
    if (t.a.bits == 4 && t.a.head_dim == 64) return launch_format<T, PL, 4, 64>(t, nr, qimg, path, stream);
    return launch_format<T, PL, 8, 64>(t, nr, qimg, path, stream);
}

}  // namespace

// Workspace of the tensor-core tree attention at any context up to `tokens` (0: another kernel's job).
size_t tree_workspace_bytes(int batch, int heads, int group, int head_dim, int bits, int sm_count, int64_t tokens,
                            int nodes, int dtype, int full) {
    if ((bits != 4 && bits != 8) || (head_dim != 64 && head_dim != 128)) return 0;
    const int64_t per = tree_batch(batch, heads, group, nodes);
    const TreePlan p = tree_plan(per, heads, group, head_dim, sm_count, tokens, nodes, dtype, full);
    return p.records + p.qimg + p.path;
}

int launch_gqa_tree_umma(const AttendArgs &a, void *workspace, cudaStream_t stream) {
    const int64_t per = tree_batch(a.batch, a.heads, a.group, a.seq_len);
    const int64_t qrow = (int64_t)a.seq_len * a.heads * a.group * a.head_dim * (a.dtype == SA_DTYPE_FLOAT ? 4 : 2);
    for (int64_t b0 = 0; b0 < a.batch; b0 += per) {
        TreeArgs t{};
        t.a = a;
        t.a.batch = (int)(a.batch - b0 < per ? a.batch - b0 : per);
        const int64_t unit0 = b0 * a.heads;
        t.a.query = static_cast<const char *>(a.query) + b0 * qrow;
        t.a.out = static_cast<char *>(a.out) + b0 * qrow;
        t.a.parents = a.parents + b0 * a.seq_len;
        t.a.k_codes = a.k_codes + unit0 * a.capacity * a.code_bytes;
        t.a.v_codes = a.v_codes + unit0 * a.capacity * a.code_bytes;
        t.a.k_meta = a.k_meta + unit0 * a.capacity * 2;
        t.a.v_meta = a.v_meta + unit0 * a.capacity * 2;
        if (a.lr_vtr) t.a.lr_vtr = a.lr_vtr + unit0 * a.head_dim;
        const TreePlan p = tree_plan(t.a.batch, a.heads, a.group, a.head_dim, a.sm_count, a.pos0 + a.seq_len, a.seq_len,
                                     a.dtype, a.tree_full);
        char *ws = static_cast<char *>(workspace);
        t.records = reinterpret_cast<float *>(ws);
        t.qimg = reinterpret_cast<unsigned char *>(ws + p.records);
        t.path = reinterpret_cast<uint64_t *>(ws + p.records + p.qimg);
        t.rows = a.seq_len * a.group;
        t.nb = p.nb;
        t.ntiles = p.ntiles;
        t.F = p.F;
        t.groups = p.groups;
        unsigned char *qimg = reinterpret_cast<unsigned char *>(ws + p.records);
        uint64_t *path = reinterpret_cast<uint64_t *>(ws + p.records + p.qimg);
        int rc;
        switch (a.dtype) {
            case SA_DTYPE_FLOAT: rc = launch_type<float, 2>(t, p.nr, qimg, path, stream); break;
            case SA_DTYPE_FLOAT16: rc = launch_type<__half, 2>(t, p.nr, qimg, path, stream); break;
            default:
                rc = a.tree_full ? launch_type<__nv_bfloat16, 2>(t, p.nr, qimg, path, stream)
                                 : launch_type<__nv_bfloat16, 1>(t, p.nr, qimg, path, stream);
                break;
        }
        if (rc != SA_OK) return rc;
    }
    return SA_OK;
}

}  // namespace sa
