// Beam search's selection: log-softmax over the vocabulary and the best
// continuations of a group of beams, in one pass over the logits.
//
// beam_scan_kernel: a warp takes a run of a row in groups of 256 neighbouring
// tokens and leaves, per group, the largest logit, and per run the sum of
// exponentials and its reference.  Nothing else of the row is needed to choose:
// the best n tokens lie in the n groups with the largest maxima (each of n better
// groups holds a better token; between equal maxima the lower group holds the lower
// token).
//
// beam_pick_kernel, a CTA per group of beams: the beams' logarithms, the best
// `keep` groups over all beams by score + (maximum - log sum), then the best `keep`
// tokens of those groups, which are read again.
//
// Equal rows give equal sums: which lane takes which token, and in which order, does
// not depend on where a row begins, so that beams that are equal tie exactly.
#include <math.h>

#include "sa_decode_common.cuh"
#include "sa_pages.cuh"

namespace sa {

namespace {

constexpr int kGroup = 256;      // tokens of a group
constexpr int kScanThreads = 256;
constexpr int kPickThreads = 512;
constexpr int kAhead = 4;        // groups a warp loads at once
constexpr int kScanWarps = 148 * 48;  // warps that the scan is split into where rows allow it
constexpr float kL = 1.4426950408889634f;  // log2(e)

struct Part {
    double sum;  // of e^(x - top)
    float top;
    float pad;
};

int64_t groups_of(int64_t vocab) { return (vocab + kGroup - 1) / kGroup; }
int parts_per_row(int64_t rows, int64_t groups) {
    const int64_t want = (kScanWarps + rows - 1) / rows, most = (groups + kAhead - 1) / kAhead;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

// Eight tokens of group g; -inf outside the row.  PIECES (all rows begin on 16 bytes): neighbours, one 16-byte load
// (two of f32); else every 32nd, so that the warp's loads are neighbours wherever the row begins.
template <typename T, bool PIECES>
__device__ __forceinline__ void load_tokens(const T *row, int vocab, int g, int lane, float (&x)[8]) {
    const int64_t e0 = (int64_t)g * kGroup + (PIECES ? lane * 8 : lane);
    constexpr int kStep = PIECES ? 1 : 32;
    if (PIECES && e0 + 8 <= vocab) {
        load_run<T, 8>(row + e0, true, x);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = e0 + kStep * i < vocab ? ld_f32(row + e0 + kStep * i) : -INFINITY;
    }
}

template <typename T, bool PIECES>
__global__ void __launch_bounds__(kScanThreads) beam_scan_kernel(BeamArgs a, int groups, int parts, float *maxima, Part *sums) {
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
    float top = -INFINITY, sum = 0.0f;
    for (int g = g0; g < g1; g += kAhead) {
        float x[kAhead][8], m[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            if (g + j < g1) {
                load_tokens<T, PIECES>(row, a.vocab, g + j, lane, x[j]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) x[j][i] = -INFINITY;
            }
        }
        float most = top;
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            m[j] = x[j][0];
#pragma unroll
            for (int i = 1; i < 8; i++) m[j] = fmaxf(m[j], x[j][i]);
            m[j] = warp_max(m[j]);
            most = fmaxf(most, m[j]);
            if (lane == 0 && g + j < g1) maxima[r * groups + g + j] = m[j];
        }
        if (most > top) {
            sum = top == -INFINITY ? sum : sum * exp2f((top - most) * kL);
            top = most;
        }
        const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; i++) e[i] = dec::ex2_approx((x[j][i] - ref) * kL);
            sum += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
        }
    }
    double total = sum;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) sums[r * parts + part] = Part{total, top, 0.0f};
}

// Scores as unsigned numbers of the same order; 0 for what is never chosen.
__device__ __forceinline__ unsigned long long order_of(double s) {
    if (!(s > -INFINITY)) return 0;
    s += 0.0;  // -0 counts as 0
    const long long b = __double_as_longlong(s);
    return (unsigned long long)(b >= 0 ? b : ~b) ^ (b >= 0 ? 0x8000000000000000ull : 0ull);
}

struct Best {
    unsigned long long key;
    unsigned place;
};

// Whether x comes before y: the larger key, then the lower place.
__device__ __forceinline__ bool before(const Best &x, const Best &y) {
    return x.key > y.key || (x.key == y.key && x.place < y.place);
}

__device__ __forceinline__ Best warp_best(Best b) {
    const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(b.key >> 32));
    const bool at_hi = (unsigned)(b.key >> 32) == hi;
    const unsigned lo = __reduce_max_sync(0xffffffffu, at_hi ? (unsigned)b.key : 0u);
    const unsigned place = __reduce_min_sync(0xffffffffu, at_hi && (unsigned)b.key == lo ? b.place : 0xffffffffu);
    return Best{((unsigned long long)hi << 32) | lo, place};
}

// The best of a CTA, of each thread's own best; `box` alternates between calls.
__device__ __forceinline__ Best block_best(Best b, Best (*box)[kPickThreads / 32], int turn) {
    const int lane = threadIdx.x & 31;
    b = warp_best(b);
    if (lane == 0) box[turn & 1][threadIdx.x >> 5] = b;
    __syncthreads();
    return warp_best(lane < kPickThreads / 32 ? box[turn & 1][lane] : Best{0, 0xffffffffu});
}

template <typename T>
__global__ void __launch_bounds__(kPickThreads) beam_pick_kernel(BeamArgs a, int groups, int parts, const float *maxima,
                                                                 const Part *sums) {
    __shared__ double s_lse[SA_MAX_BEAMS];
    __shared__ float s_score[SA_MAX_BEAMS];
    __shared__ bool s_done[SA_MAX_BEAMS];
    __shared__ unsigned s_group[SA_MAX_BEAM_KEEP];
    __shared__ Best s_box[2][kPickThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, b = blockIdx.x, K = a.beams;
    const int64_t r0 = (int64_t)b * K;
    dec::griddep_launch_dependents();
    dec::griddep_wait();
    for (int k = tid >> 5; k < K; k += kPickThreads / 32) {
        const bool done = a.finished && a.finished[r0 + k];
        double lse = 0.0;
        if (!done) {
            const Part *p = sums + (r0 + k) * parts;
            float top = -INFINITY;
            for (int i = lane; i < parts; i += 32) top = fmaxf(top, p[i].top);
            top = warp_max(top);
            double total = 0.0;
            for (int i = lane; i < parts; i += 32)
                if (p[i].top > -INFINITY) total += p[i].sum * exp((double)p[i].top - (double)top);
                else total += p[i].sum;  // 0, or NaN
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
            lse = (double)top + log(total);
        }
        if (lane == 0) {
            s_lse[k] = lse;
            s_score[k] = a.scores[r0 + k];
            s_done[k] = done;
        }
    }
    __syncthreads();

    // the best groups over all beams
    int turn = 0, found = 0;
    {
        auto group_of = [&](int i) {
            const int k = i / groups, g = i - k * groups;
            double s;
            if (s_done[k]) s = g == 0 && a.end_token >= 0 && a.end_token < a.vocab ? (double)s_score[k] : -INFINITY;
            else s = (double)s_score[k] + ((double)maxima[(r0 + k) * groups + g] - s_lse[k]);
            return Best{order_of(s), (unsigned)i};
        };
        Best last{~0ull, 0}, mine{0, 0xffffffffu};
        bool first = true;
        for (; found < a.keep; found++) {
            if (first) {  // this thread's best that has not been taken
                mine = Best{0, 0xffffffffu};
                for (int i = tid; i < K * groups; i += kPickThreads) {
                    const Best c = group_of(i);
                    if (before(c, mine) && before(last, c)) mine = c;
                }
            }
            const Best best = block_best(mine, s_box, turn++);
            if (best.key == 0) break;
            if (tid == 0) s_group[found] = best.place;
            first = best.place == mine.place;
            if (first) last = best;
        }
    }
    __syncthreads();

    // the best tokens of those groups
    {
        auto token_of = [&](int i) {
            const unsigned gi = s_group[i / kGroup];
            const int k = (int)(gi / (unsigned)groups), g = (int)(gi - (unsigned)k * groups), x = i % kGroup;
            if (s_done[k])
                return x == 0 ? Best{order_of((double)s_score[k]), (unsigned)(k * a.vocab + a.end_token)}
                              : Best{0, 0xffffffffu};
            const T *row = static_cast<const T *>(a.logits) + (r0 + k) * a.row_stride;
            const int64_t v = (int64_t)g * kGroup + x;
            if (v >= a.vocab) return Best{0, 0xffffffffu};
            return Best{order_of((double)s_score[k] + ((double)ld_f32(row + v) - s_lse[k])), (unsigned)(k * a.vocab + (int)v)};
        };
        Best last{~0ull, 0}, mine{0, 0xffffffffu};
        bool first = true;
        int n = 0;
        for (; n < a.keep; n++) {
            if (first) {
                mine = Best{0, 0xffffffffu};
                for (int i = tid; i < found * kGroup; i += kPickThreads) {
                    const Best c = token_of(i);
                    if (before(c, mine) && before(last, c)) mine = c;
                }
            }
            const Best best = block_best(mine, s_box, turn++);
            if (best.key == 0) break;
            if (tid == 0) {
                const int k = (int)(best.place / (unsigned)a.vocab);
                const unsigned long long bits =
                    best.key & 0x8000000000000000ull ? best.key ^ 0x8000000000000000ull : ~best.key;
                a.parents[(int64_t)b * a.keep + n] = k;
                a.tokens[(int64_t)b * a.keep + n] = (int)(best.place - (unsigned)k * (unsigned)a.vocab);
                a.out_scores[(int64_t)b * a.keep + n] = (float)__longlong_as_double((long long)bits);
            }
            first = best.place == mine.place;
            if (first) last = best;
        }
        for (int i = n + tid; i < a.keep; i += kPickThreads) {
            a.parents[(int64_t)b * a.keep + i] = -1;
            a.tokens[(int64_t)b * a.keep + i] = -1;
            a.out_scores[(int64_t)b * a.keep + i] = -INFINITY;
        }
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
