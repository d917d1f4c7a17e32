// Beam search's selection: log-softmax over the vocabulary and the best
// continuations of a group of beams, in one pass over the logits.
//
// beam_scan_kernel: a warp takes a run of a row in groups of 256 neighbouring
// tokens and leaves, per group, the largest logit, and per run the sum of
// exponentials and its reference (a lane's in f64, over sums of 16 or 32 terms in
// f32).  Nothing else of the row is needed to choose: the best n tokens lie in the n
// groups with the largest maxima (each of n better groups holds a better token;
// between equal maxima the lower group holds the lower token).
//
// beam_pick_kernel, a CTA per group of beams: the beams' logarithms, the best
// `keep` groups over all beams by score + (maximum - log sum), then the best `keep`
// tokens of those groups, which are read again.
//
// 64 x 8 rows of 128256 bf16 (131 MB, a seventh of the rows finished and skipped), 35.5 us: the scan some 25, 4.4 TB/s
// of the 108 MB that it reads, eight instructions a token, 58% of the cycles issue; the choice 11, a chain of dependent
// steps over 16 KB a group, which one group of 4 beams over 32000 tokens needs as well (10.7 us in all).  At 64 registers
// the scan of aligned 16-bit rows spills 16 bytes a thread, the choice 16 to 28.
//
// Equal rows give equal sums: which lane takes which token, and in which order, does
// not depend on where a row begins, so that beams that are equal tie exactly.
#include <math.h>

#include <type_traits>

#include "sa_decode_common.cuh"
#include "sa_pages.cuh"

namespace sa {

namespace {

constexpr int kGroup = 256;      // tokens of a group
constexpr int kScanThreads = 256;
constexpr int kPickThreads = 512;
// Warps that the scan is split into where rows allow it: two waves of the 32 that fit on an SM.  Scan and choice at one,
// two, three and four waves, in us: 64 x 8 rows of 128256 bf16 38.2, 35.5, 38.3, 42.4; of 32000 20.7, 21.0, 24.4, 20.9;
// 16 x 8 of 128256 f32 21.3, 22.8, 24.6, 23.0; 32 x 5 of 50257 f16 18.5 and 18.3 three times; 4 of 32000 10.7 in all;
// 1250 x 4 of 32000 bf16 120, 120, 104, 102 (a row per warp, then two).
constexpr int kScanWarps = 148 * 64;
constexpr float kL = 1.4426950408889634f;  // log2(e)
// How far the largest logit may lie above the reference of a run's sum before the reference is raised to it.  A raise is
// off by 2^-22: one in every step, in rows that climb slowly, added up to 2e-6; with 4, what comes before two or three
// raises no longer counts.
constexpr float kLag = 4.0f;

struct Part {
    double sum;  // of e^(x - top)
    float top;
    float pad;
};

int64_t groups_of(int64_t vocab) { return (vocab + kGroup - 1) / kGroup; }
int parts_per_row(int64_t rows, int64_t groups) {
    const int64_t want = kScanWarps / rows, most = (groups + 3) / 4;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

// Eight tokens of a group that a lane holds, as they were loaded; -inf outside the row.  PIECES (all rows begin on 16
// bytes): neighbours, one 16-byte load (two of f32); else every 32nd, so that the warp's loads are neighbours wherever
// the row begins.  32 x 5 rows of 50257 f16, scan and pick: 21.0 us so, 22.0 with eight neighbours loaded one by one.
template <typename T, bool PIECES>
struct Tokens {
    float x[8];
    __device__ __forceinline__ void load_whole(const T *row, int g, int lane) {  // of a group that is all in the row
        const T *p = row + (int64_t)g * kGroup + (PIECES ? lane * 8 : lane);
        if constexpr (PIECES) {
            load_run<T, 8>(p, true, x);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = ld_f32(p + 32 * i);
        }
    }
    __device__ __forceinline__ void load(const T *row, int vocab, int g, int lane) {
        const int64_t e0 = (int64_t)g * kGroup + (PIECES ? lane * 8 : lane);
        constexpr int kStep = PIECES ? 1 : 32;
        if (PIECES && e0 + 8 <= vocab) {
            load_run<T, 8>(row + e0, true, x);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = e0 + kStep * i < vocab ? ld_f32(row + e0 + kStep * i) : -INFINITY;
        }
    }
    __device__ __forceinline__ float get(int i) const { return x[i]; }
    __device__ __forceinline__ float top() const {
        return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    }
};

// 16-bit pieces stay packed until they are used: four registers, and the largest of two at once.
template <typename T>
struct PackedTokens {
    uint32_t w[4];
    __device__ __forceinline__ void load_whole(const T *row, int g, int lane) {
        const uint4 v = *reinterpret_cast<const uint4 *>(row + (int64_t)g * kGroup + lane * 8);
        w[0] = v.x;
        w[1] = v.y;
        w[2] = v.z;
        w[3] = v.w;
    }
    __device__ __forceinline__ void load(const T *row, int vocab, int g, int lane) {
        const int64_t e0 = (int64_t)g * kGroup + lane * 8;
        if (e0 + 8 <= vocab) {
            load_whole(row, g, lane);
        } else {
            constexpr uint32_t kNone = std::is_same<T, __half>::value ? 0xFC00u : 0xFF80u;  // -inf
            const uint16_t *p = reinterpret_cast<const uint16_t *>(row);
#pragma unroll
            for (int i = 0; i < 4; i++)
                w[i] = (e0 + 2 * i < vocab ? p[e0 + 2 * i] : kNone) | (e0 + 2 * i + 1 < vocab ? p[e0 + 2 * i + 1] : kNone) << 16;
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (std::is_same<T, __half>::value)
            return __half2float(__ushort_as_half((unsigned short)(w[i >> 1] >> (16 * (i & 1)))));
        return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
    }
    __device__ __forceinline__ float top() const {
        using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
        T2 v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = *reinterpret_cast<const T2 *>(&w[i]);
        const T2 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
        return fmaxf(DT<T>::to_f32(m.x), DT<T>::to_f32(m.y));
    }
};
template <>
struct Tokens<__half, true> : PackedTokens<__half> {};
template <>
struct Tokens<__nv_bfloat16, true> : PackedTokens<__nv_bfloat16> {};

// The largest value of a warp; NaN counts for nothing, as in fmaxf.
__device__ __forceinline__ float warp_top(float x) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;\n" : "=f"(m) : "f"(x));
    return m;
}

template <typename T, bool PIECES>
__global__ void __launch_bounds__(kScanThreads, 4) beam_scan_kernel(BeamArgs a, int groups, int parts, float *maxima, Part *sums) {
    // groups that a warp takes at a time, while the next ones are on their way
    constexpr int kAhead = PIECES && sizeof(T) == 2 ? 4 : 2;
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * (kScanThreads / 32) + (threadIdx.x >> 5);
    dec::griddep_launch_dependents();
    const int64_t r = w / parts;
    if (r >= (int64_t)a.batch * a.beams) return;
    dec::griddep_wait();
    if (a.finished && a.finished[r]) return;
    const int part = (int)(w - r * parts);
    const T *row = static_cast<const T *>(a.logits) + r * a.row_stride;
    const int g0 = (int)((int64_t)groups * part / parts), g1 = (int)((int64_t)groups * (part + 1) / parts);
    float top = -INFINITY;  // the reference of the sum: up to kLag below the largest logit
    double sum = 0.0;
    auto consume = [&](const Tokens<T, PIECES> (&now)[kAhead], int g) {
        float most = top, mine = 0.0f;
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const float m = warp_top(now[j].top());
            most = fmaxf(most, m);
            if (lane == j) mine = m;
        }
        if (lane < kAhead && g + lane < g1) maxima[r * groups + g + lane] = mine;
        if (most > top + kLag) {
            if (top > -INFINITY) sum *= exp2f((top - most) * kL);
            top = most;
        }
        const float ref = top == -INFINITY ? 0.0f : top;
        const f2 less = pair(-ref, -ref), log2e = pair(kL, kL);
        float few = 0.0f;  // of 8 * kAhead terms
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            f2 e[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float x0, x1;
                split(mul2(add2(pair(now[j].get(2 * i), now[j].get(2 * i + 1)), less), log2e), x0, x1);
                e[i] = pair(dec::ex2_approx(x0), dec::ex2_approx(x1));
            }
            float s0, s1;
            split(add2(add2(e[0], e[1]), add2(e[2], e[3])), s0, s1);
            few += s0 + s1;
        }
        sum += (double)few;
    };
    // whole groups, the next ones on their way; then the others
    Tokens<T, PIECES> now[kAhead], next[kAhead];
    const int whole = min(g1, a.vocab / kGroup);
    int g = g0;
    bool more = g + kAhead <= whole;
    if (more)
#pragma unroll
        for (int j = 0; j < kAhead; j++) next[j].load_whole(row, g + j, lane);
    while (more) {
#pragma unroll
        for (int j = 0; j < kAhead; j++) now[j] = next[j];
        more = g + 2 * kAhead <= whole;
        if (more)
#pragma unroll
            for (int j = 0; j < kAhead; j++) next[j].load_whole(row, g + kAhead + j, lane);
        consume(now, g);
        g += kAhead;
    }
    for (; g < g1; g += kAhead) {
#pragma unroll
        for (int j = 0; j < kAhead; j++) now[j].load(row, g + j < g1 ? a.vocab : 0, g + j, lane);
        consume(now, g);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sums[r * parts + part] = Part{sum, top, 0.0f};
}

struct Choice {
    double score;
    unsigned place;
};

// Whether x comes before y: the larger score, of equal ones the lower place.
__device__ __forceinline__ bool before(const Choice &x, const Choice &y) {
    return x.score > y.score || (x.score == y.score && x.place < y.place);
}

constexpr int kListed = 1024;  // choices that are ranked against each other
constexpr int kTops = kPickThreads / 4;

// The choice is made twice in the same way, among groups and then among the tokens of the best ones (and the finished
// beams): the keep-th largest of the 128 best scores of four threads each bounds the keep-th best from below (mode 0),
// the few choices that reach it are listed (mode 1) and ranked against each other.  Where they are too many, scores
// that are equal by the hundreds, the best is taken out one at a time (mode 2).  One piece of code serves all of that:
// this kernel runs for a few microseconds, of which fetching its code is a good part (unrolled copies for every step
// took 15 us after the scan of 64 x 8 beams, this takes 11).
template <typename T>
__global__ void __launch_bounds__(kPickThreads) beam_pick_kernel(BeamArgs a, int groups, int parts, const float *maxima,
                                                                 const Part *sums) {
    __shared__ double s_lse[SA_MAX_BEAMS], s_score[SA_MAX_BEAMS];  // of beams that go on; a score of -inf for the others
    __shared__ int s_beam[SA_MAX_BEAM_KEEP], s_first[SA_MAX_BEAM_KEEP];  // of the best groups: beam, first token
    __shared__ double s_top[kTops], s_least;
    __shared__ Choice s_list[kListed], s_out[SA_MAX_BEAM_KEEP], s_box[2][kPickThreads / 32];
    __shared__ int s_listed;
    constexpr Choice kNone{-INFINITY, 0xffffffffu};
    const int tid = threadIdx.x, lane = tid & 31, b = blockIdx.x, K = a.beams, keep = a.keep;
    const int64_t r0 = (int64_t)b * K;
    const T *logits = static_cast<const T *>(a.logits) + r0 * a.row_stride;
    dec::griddep_launch_dependents();
    dec::griddep_wait();
    for (int k = tid >> 5; k < K; k += kPickThreads / 32) {
        // (a finished beam's parts were not written, and are not used)
        const Part *p = sums + (r0 + k) * parts;
        const bool done = a.finished && a.finished[r0 + k];
        float top = -INFINITY;
        for (int i = lane; i < parts; i += 32) top = fmaxf(top, p[i].top);
        top = warp_max(top);
        double total = 0.0;
        for (int i = lane; i < parts; i += 32)  // a part without a largest logit: 0, or NaN
            total += p[i].top > -INFINITY ? p[i].sum * exp((double)p[i].top - (double)top) : p[i].sum;
#pragma unroll 1
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if (lane == 0) {
            s_lse[k] = (double)top + log(total);
            s_score[k] = done ? -INFINITY : (double)a.scores[r0 + k];
        }
    }
    __syncthreads();

    int found = 0;
#pragma unroll 1
    for (int phase = 0; phase < 2; phase++) {
        // keep groups hold a token each that scores what the last of them does
        int mode = phase == 1 && found == keep ? 1 : 0, n = 0;
        double least = mode == 1 ? s_out[keep - 1].score : -INFINITY;
        // a thread's choices in eights; a single eight is worked out once
        // groups: 2^wide threads share a beam's (few groups: several beams side by side)
        int wide = 9;
        while (wide > 0 && 1 << (wide - 1) >= groups) wide--;
        const int side = kPickThreads >> wide, beams8 = (K + 8 * side - 1) / (8 * side);
        const int eights = phase == 0 ? ((groups - 1) >> wide) * beams8 + beams8 : (found + 15) / 16;
        double score[8];
        unsigned place[8];
        bool known = false;
        if (tid == 0) s_listed = 0;
        __syncthreads();
        Choice last = kNone, mine = kNone;  // mode 2: the last one taken from this thread, its best of the others
        bool taken = false, search = true;
#pragma unroll 1
        for (;;) {
            double top = -INFINITY;
            auto take = [&](double sc, unsigned pl) {
                if (!(sc > -INFINITY)) return;  // NaN too
                if (mode == 0) {
                    if (sc > top) top = sc;
                } else if (mode == 1) {
                    if (sc >= least) {
                        const int at = atomicAdd(&s_listed, 1);
                        if (at < kListed) s_list[at] = Choice{sc, pl};
                    }
                } else if (search) {
                    const Choice c{sc, pl};
                    if (before(c, mine) && (!taken || before(last, c))) mine = c;
                }
            };
#pragma unroll 1
            for (int e = 0; e < eights; e++) {
                if (known) {
                } else if (phase == 0) {
                    const int g = (e / beams8 << wide) + (tid & ((1 << wide) - 1)), k0 = e % beams8 * 8 * side + (tid >> wide);
                    float m[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int k = k0 + i * side;
                        m[i] = g < groups && k < K ? maxima[(r0 + k) * groups + g] : -INFINITY;
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int k = min(k0 + i * side, K - 1);
                        score[i] = s_score[k] + ((double)m[i] - s_lse[k]);
                        place[i] = (unsigned)(k * groups + g);
                    }
                } else {  // the threads share the tokens of each group
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int j = 16 * e + 2 * i + tid / kGroup, v = j < found ? s_first[j] + tid % kGroup : a.vocab;
                        x[i] = v < a.vocab ? ld_f32(logits + s_beam[j] * a.row_stride + v) : -INFINITY;
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int j = min(16 * e + 2 * i + tid / kGroup, found - 1), k = s_beam[j];
                        score[i] = s_score[k] + ((double)x[i] - s_lse[k]);
                        place[i] = (unsigned)k * (unsigned)a.vocab + s_first[j] + tid % kGroup;
                    }
                }
                known = eights == 1;
#pragma unroll
                for (int i = 0; i < 8; i++) take(score[i], place[i]);
            }
            if (phase == 1 && tid < K && a.finished && a.finished[r0 + tid] && a.end_token >= 0 && a.end_token < a.vocab)
                take((double)a.scores[r0 + tid], (unsigned)tid * (unsigned)a.vocab + a.end_token);
            if (mode == 0) {
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    const double other = __shfl_xor_sync(0xffffffffu, top, o);
                    if (other > top) top = other;
                }
                if ((tid & 3) == 0) s_top[tid >> 2] = top;
                __syncthreads();
                // four threads rank one of the 128 among all
                const double own = s_top[tid >> 2];
                int ahead = 0;
#pragma unroll 8
                for (int i = 0; i < kTops / 4; i++) {
                    const int j = 4 * i + (tid & 3);
                    ahead += s_top[j] > own || (s_top[j] == own && j < tid >> 2);
                }
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
                if ((tid & 3) == 0 && ahead == keep - 1) s_least = own;
                __syncthreads();
                least = s_least;
                mode = 1;
            } else if (mode == 1) {
                __syncthreads();
                n = s_listed;
                if (n <= kListed) {
#pragma unroll 1
                    for (int i = tid; i < n; i += kPickThreads) {
                        const Choice own = s_list[i];
                        int ahead = 0;
#pragma unroll 4
                        for (int j = 0; j < n; j++) ahead += before(s_list[j], own);
                        if (ahead < keep) s_out[ahead] = own;
                    }
                    n = min(n, keep);
                    break;
                }
                n = 0;
                mode = 2;
            } else {
                search = false;
                Choice best = mine;
#pragma unroll 1
                for (int half = 0; half < 2; half++) {  // of a warp, then of the warps
#pragma unroll 1
                    for (int o = 16; o > 0; o >>= 1) {
                        const Choice other{__shfl_xor_sync(0xffffffffu, best.score, o), __shfl_xor_sync(0xffffffffu, best.place, o)};
                        if (before(other, best)) best = other;
                    }
                    if (half == 1) break;
                    if (lane == 0) s_box[n & 1][tid >> 5] = best;
                    __syncthreads();
                    best = lane < kPickThreads / 32 ? s_box[n & 1][lane] : kNone;
                }
                if (best.place == kNone.place || n == keep) break;
                if (tid == 0) s_out[n] = best;
                n++;
                if (best.place == mine.place) {
                    last = best;
                    taken = search = true;
                    mine = kNone;
                }
            }
        }
        __syncthreads();
        if (phase == 0) {
            found = n;
            if (tid < n) {
                const int k = (int)(s_out[tid].place / (unsigned)groups);
                s_beam[tid] = k;
                s_first[tid] = (int)(s_out[tid].place - (unsigned)(k * groups)) * kGroup;
            }
        } else if (tid < keep) {
            const bool some = tid < n;
            const Choice c = some ? s_out[tid] : Choice{-INFINITY, 0};
            const int k = (int)(c.place / (unsigned)a.vocab);
            const int64_t at = (int64_t)b * keep + tid;
            a.parents[at] = some ? k : -1;
            a.tokens[at] = some ? (int)(c.place - (unsigned)k * (unsigned)a.vocab) : -1;
            a.out_scores[at] = (float)c.score;
        }
        __syncthreads();
    }
}

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

template <typename T>
int launch_t(const BeamArgs &a, void *workspace, cudaStream_t stream) {
    const int64_t rows = (int64_t)a.batch * a.beams;
    const int groups = (int)groups_of(a.vocab), parts = parts_per_row(rows, groups);
    Part *sums = static_cast<Part *>(workspace);
    float *maxima = reinterpret_cast<float *>(static_cast<char *>(workspace) + align256(rows * parts * sizeof(Part)));
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((rows * parts + kScanThreads / 32 - 1) / (kScanThreads / 32)));
    cfg.blockDim = dim3(kScanThreads);
    cfg.stream = stream;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    const bool pieces = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && (rows == 1 || a.row_stride * (int)sizeof(T) % 16 == 0);
    auto scan = pieces ? beam_scan_kernel<T, true> : beam_scan_kernel<T, false>;
    int rc = check_cuda(cudaLaunchKernelEx(&cfg, scan, a, groups, parts, maxima, sums), "beam_select launch");
    count_launch();
    if (rc != SA_OK) return rc;
    cfg.gridDim = dim3((unsigned)a.batch);
    cfg.blockDim = dim3(kPickThreads);
    rc = check_cuda(cudaLaunchKernelEx(&cfg, beam_pick_kernel<T>, a, groups, parts, (const float *)maxima, (const Part *)sums),
                    "beam_select pick launch");
    count_launch();
    return rc;
}

}  // namespace

int64_t beam_select_workspace(int64_t rows, int64_t vocab) {
    const int64_t groups = groups_of(vocab);
    return (int64_t)(align256(rows * parts_per_row(rows, groups) * sizeof(Part)) + align256(rows * groups * sizeof(float)));
}

int launch_beam_select(const BeamArgs &a, void *workspace, cudaStream_t stream) {
    switch (a.dtype) {
        case SA_DTYPE_FLOAT: return launch_t<float>(a, workspace, stream);
        case SA_DTYPE_FLOAT16: return launch_t<__half>(a, workspace, stream);
        default: return launch_t<__nv_bfloat16>(a, workspace, stream);
    }
}

}  // namespace sa
