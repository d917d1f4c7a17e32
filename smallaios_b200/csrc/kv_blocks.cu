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
constexpr int kSelectThreads = 256;
constexpr float kGridMax = 1.2676506002282294e30f;  // 2^100: larger values (and NaN) count as zero

__device__ __forceinline__ float grid_value(float x) { return fabsf(x) < kGridMax ? x : 0.0f; }

// The least e with x < 2^e, at least -100 (x >= 0).
__device__ __forceinline__ int grid_exponent(float x) {
    if (!(x > 0.0f)) return -100;
    const int e = ((__float_as_int(x) >> 23) & 0xff) - 126;  // a subnormal's is below -100 anyway
    return e < -100 ? -100 : e;
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // -126..127

// grid = (blocks, units): one CTA per block, one thread per dimension.
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

// The 8-bit queries of the G heads of one KV head, as floats [G][d] in shared memory.
template <typename T, int EPL>
__device__ __forceinline__ void select_queries(const SelectArgs &a, const T *src, const float *sg, float *s_q,
                                               int *s_max) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = a.head_dim;
    const bool active = lane * EPL < d;
    if (threadIdx.x < 2) s_max[threadIdx.x] = 0;
    __syncthreads();
    float x[EPL];
    float top = 0.0f;
    if (warp < a.group) {
#pragma unroll
        for (int r = 0; r < EPL; r++) {
            x[r] = active ? grid_value(ld_f32(src + (int64_t)warp * d + lane * EPL + r)) : 0.0f;
            top = fmaxf(top, fabsf(x[r]));
        }
        top = warp_max(top);
        if (lane == 0) atomicMax(&s_max[0], __float_as_int(top));  // non-negative floats order as their bits
    }
    __syncthreads();
    if (warp < a.group) {
        const float f = power_of_two(12 - grid_exponent(__int_as_float(s_max[0])));
#pragma unroll
        for (int r = 0; r < EPL; r++) x[r] = active ? rintf(x[r] * f) * sg[lane * EPL + r] : 0.0f;
        warp_wht_butterfly<EPL>(x, lane, d);
        top = 0.0f;
#pragma unroll
        for (int r = 0; r < EPL; r++) top = fmaxf(top, active ? fabsf(x[r]) : 0.0f);
        top = warp_max(top);
        if (lane == 0) atomicMax(&s_max[1], __float_as_int(top));
    }
    __syncthreads();
    if (warp < a.group && active) {
        const int sh = max(0, grid_exponent(__int_as_float(s_max[1])) - 7);
        const float f = power_of_two(-sh);
#pragma unroll
        for (int r = 0; r < EPL; r++)
            s_q[warp * d + lane * EPL + r] = fminf(fmaxf(rintf(x[r] * f), -127.0f), 127.0f);
    }
    __syncthreads();
}

// grid = (heads, seq_len, batch): one CTA per query token and KV head.
template <typename T, int EPL>
__global__ void __launch_bounds__(kSelectThreads) select_blocks_kernel(SelectArgs a) {
    extern __shared__ int s_key[];  // one key per candidate block
    __shared__ float s_q[8 * 256];
    __shared__ int s_max[2], s_hist[256], s_scan[kSelectThreads / 32], s_pick[3];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, d = a.head_dim;
    const int h = blockIdx.x, s = blockIdx.y, b = blockIdx.z;
    const int64_t row = (int64_t)b * a.seq_len + s;
    const T *src = static_cast<const T *>(a.query) + (row * a.heads + h) * a.group * d;
    int32_t *out = a.block_ids + (row * a.heads + h) * a.max_blocks;
    const int own = (int)((a.pos0 + s) / kBlockTokens), nb = own + 1, k = a.max_blocks;
    if (nb <= k) {  // every block
        for (int i = tid; i < k; i += kSelectThreads) out[i] = i < nb ? i : -1;
        return;
    }
    select_queries<T, EPL>(a, src, a.signs + (int64_t)h * d, s_q, s_max);

    // ---- scores as order-preserving integers; the forced blocks above all ----
    const __nv_bfloat16 *means = static_cast<const __nv_bfloat16 *>(a.means) + ((int64_t)b * a.heads + h) * a.row_stride;
    const bool active = lane * EPL < d;
    for (int i = warp; i < nb; i += kSelectThreads / 32) {
        int key = 0x7fffffff;
        if (i >= a.sink && i <= own - a.local) {
            float m[EPL], best = -INFINITY;
#pragma unroll
            for (int r = 0; r < EPL; r++)
                m[r] = active ? __bfloat162float(means[(int64_t)i * d + lane * EPL + r]) : 0.0f;
            for (int g = 0; g < a.group; g++) {
                float dot = 0.0f;
#pragma unroll
                for (int r = 0; r < EPL; r++) dot = fmaf(m[r], active ? s_q[g * d + lane * EPL + r] : 0.0f, dot);
                best = fmaxf(best, warp_sum(dot));
            }
            key = order_key(best + 0.0f);
        }
        if (lane == 0) s_key[i] = key;
    }
    __syncthreads();

    // ---- the k-th largest key, byte by byte from the top ----
    uint32_t prefix = 0;  // of the keys with the sign bit flipped (unsigned order)
    int left = k;         // keys still to take among those that share the prefix
    for (int byte = 3; byte >= 0; byte--) {
        s_hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < nb; i += kSelectThreads) {
            const uint32_t u = (uint32_t)s_key[i] ^ 0x80000000u;
            if (byte == 3 || (u >> (8 * byte + 8)) == prefix) atomicAdd(&s_hist[(u >> (8 * byte)) & 255u], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int digit = 255, n = left;
            while (s_hist[digit] < n) n -= s_hist[digit--];
            s_pick[0] = digit;
            s_pick[1] = n;
        }
        __syncthreads();
        prefix = (prefix << 8) | (uint32_t)s_pick[0];
        left = s_pick[1];
        __syncthreads();
    }

    // ---- ascending ids of the keys above it, and of the `left` lowest blocks that equal it ----
    int above = 0, equal = 0;  // counts before this round of blocks
    for (int i0 = 0; i0 < nb; i0 += kSelectThreads) {
        const int i = i0 + tid;
        const uint32_t u = i < nb ? (uint32_t)s_key[i] ^ 0x80000000u : 0u;
        const bool gt = i < nb && u > prefix, eq = i < nb && u == prefix;
        // warp and block counts of both, packed (at most 256 a round)
        const unsigned mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq);
        if (lane == 0) s_scan[warp] = __popc(mg) | (__popc(me) << 16);
        __syncthreads();
        int before = 0, all = 0;
        for (int w = 0; w < kSelectThreads / 32; w++) {
            if (w < warp) before += s_scan[w];
            all += s_scan[w];
        }
        const unsigned below = (1u << lane) - 1u;
        const int ng = above + (before & 0xffff) + __popc(mg & below);
        const int ne = equal + (before >> 16) + __popc(me & below);
        if (gt || (eq && ne < left)) out[ng + min(ne, left)] = i;
        above += all & 0xffff;
        equal += all >> 16;
        __syncthreads();
    }
}

template <typename T, int EPL>
int launch_select_t(const SelectArgs &a, cudaStream_t stream) {
    auto kern = select_blocks_kernel<T, EPL>;
    const int64_t blocks = (a.pos0 + a.seq_len - 1) / kBlockTokens + 1;
    const size_t smem = (size_t)blocks * sizeof(int);
    if (smem > 192 * 1024)
        return set_error(SA_ERR_UNSUPPORTED, "gqa_select_blocks: %lld blocks, at most 49152", (long long)blocks);
    if (a.seq_len > 65535 || a.batch > 65535)
        return set_error(SA_ERR_UNSUPPORTED, "gqa_select_blocks: %d x %d query rows, at most 65535 each", a.batch,
                         a.seq_len);
    if (smem > 32 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return check_cuda(e, "gqa_select_blocks smem attribute");
    }
    kern<<<dim3(a.heads, a.seq_len, a.batch), kSelectThreads, smem, stream>>>(a);
    count_launch();
    return check_cuda(cudaGetLastError(), "gqa_select_blocks launch");
}

template <typename T>
int launch_select_dtype(const SelectArgs &a, cudaStream_t stream) {
    switch (a.head_dim) {
        case 16:
        case 32: return launch_select_t<T, 1>(a, stream);
        case 64: return launch_select_t<T, 2>(a, stream);
        case 128: return launch_select_t<T, 4>(a, stream);
        default: return launch_select_t<T, 8>(a, stream);
    }
}

}  // namespace

int launch_block_means(const MeansArgs &a, cudaStream_t stream) {
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
