// Attention of one new token per sequence over the paged, quantised key-value cache (bw_kv_attend).
//
//     out[b][h] = sum_t w_t V[t],   w = softmax over t < lengths[b] of  alpha * q[b][h] . K[t],   K, V rows of head h / (heads / kv_heads)
//
// One pass over the cache with the running maximum and sum of the softmax; codes become values in registers.
#include "kv_attend_tiles.cuh"

namespace bw {

int attend_window_tiles(const AttendArgs &a, int64_t batch, int dtype, int bits, void *workspace, cudaStream_t st);      // kv_attend_window.cu

namespace {

// Any head dimension up to 256, any page size: one CTA a head of a sequence, its warps on every fourth token.
template <typename T, int BITS>
__global__ void __launch_bounds__(128) kv_attend_general_kernel(AttendArgs p) {
    constexpr int VPI = 32 / BITS, MOST = 8;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t b = blockIdx.x / p.heads;
    const int h = (int)(blockIdx.x - b * p.heads), kh = h / (p.heads / p.kv_heads);
    const T *q = (const T *)p.q + b * p.q_stride + h * p.q_head_stride;
    float qv[MOST], o[MOST] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < MOST; ++i) qv[i] = lane + 32 * i < p.dim ? to_f32(q[lane + 32 * i]) * p.alpha : 0.0f;
    const int64_t most = (int64_t)p.max_pages * p.page_size, n = p.lengths[b];
    bool bad = n > most;
    const int64_t len = bad ? most : n;
    // the visible tokens: `first` of the beginning, then those from `from` on
    const int64_t first = p.sinks < len ? p.sinks : len, from = n - p.window > first ? n - p.window : first, seen = first + (len > from ? len - from : 0);
    for (int64_t i = warp; i < seen; i += 4) {
        const int64_t t = i < first ? i : i - first + from, in = t / p.page_size, page = p.table[b * p.table_stride + in];
        if (page < 0 || page >= p.pages) {
            bad = true;
            continue;
        }
        const int64_t row = (page * p.kv_heads + kh) * p.page_size + (t - in * p.page_size);
        const float2 kc = __half22float2(p.params[2 * row]), vc = __half22float2(p.params[2 * row + 1]);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < MOST; ++i) {
            const int d = lane + 32 * i;
            if (d < p.dim) {
                const uint32_t w = (uint32_t)p.k_codes[row * p.words + d / VPI];
                s += qv[i] * (kc.x * ((float)((w >> (d % VPI * BITS)) & ((1u << BITS) - 1)) - kc.y));
            }
        }
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        const float top = fmaxf(m, s), keep = m == -INFINITY ? 0.0f : expf(m - top), e = expf(s - top);
        m = top;
        l = l * keep + e;
#pragma unroll
        for (int i = 0; i < MOST; ++i) {
            const int d = lane + 32 * i;
            if (d < p.dim) {
                const uint32_t w = (uint32_t)p.v_codes[row * p.words + d / VPI];
                o[i] = o[i] * keep + e * (vc.x * ((float)((w >> (d % VPI * BITS)) & ((1u << BITS) - 1)) - vc.y));
            }
        }
    }
    __shared__ float sm[4], sl[4], so[4][256];
    if (bad) l = NAN;
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < MOST; ++i)
        if (lane + 32 * i < p.dim) so[warp][lane + 32 * i] = o[i];
    __syncthreads();
    const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float f[4], sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = sm[w] == -INFINITY ? 0.0f : expf(sm[w] - top);
        sum += sl[w] == sl[w] ? f[w] * sl[w] : NAN;
    }
    for (int d = threadIdx.x; d < p.dim; d += 128) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) v += f[w] * so[w][d];
        ((T *)p.out)[(b * p.heads + h) * p.dim + d] = from_f32<T>(seen <= 0 && !bad ? 0.0f : v / sum);
    }
}

template <typename T>
int attend_general(const AttendArgs &p, int64_t batch, int bits, cudaStream_t st) {
    const unsigned grid = (unsigned)(batch * p.heads);
    if (bits == 2) kv_attend_general_kernel<T, 2><<<grid, 128, 0, st>>>(p);
    else if (bits == 4) kv_attend_general_kernel<T, 4><<<grid, 128, 0, st>>>(p);
    else kv_attend_general_kernel<T, 8><<<grid, 128, 0, st>>>(p);
    return check_launch("kv_attend_general_kernel");
}

}  // namespace

size_t kv_attend_workspace_bytes(int64_t batch, int heads, int kv_heads, int dim, int page_size, int64_t max_pages, int64_t window, int64_t sinks) {
    // (what any number of bits needs; and a cache of more rows asks for scratch that it does not use)
    for (int bits : {2, 4, 8}) {
        FastArgs p;
        if (fast_args(p, batch, heads, kv_heads, dim, bits, 0, page_size, max_pages, window, sinks) && !p.cluster) return (size_t)2 * MOST_CTAS * p.cols * (dim + 2) * sizeof(float);
    }
    return 0;
}

int kv_attend(const void *q, int dtype, int64_t batch, int heads, int64_t q_stride, int64_t q_head_stride, const int32_t *kc, const int32_t *vc,
              const void *params, int bits, int64_t pages, int page_size, int kv_heads, int dim, const int32_t *table, int64_t table_stride,
              int max_pages, const int32_t *lengths, int window, int sinks, float alpha, void *out, void *workspace, cudaStream_t st) {
    FastArgs f = {};
    AttendArgs p = {q, kc, vc, (const __half2 *)params, table, lengths, out, q_stride, q_head_stride, table_stride, pages,
                    heads, kv_heads, dim, dim * bits / 32, page_size, max_pages, alpha, window, sinks};
    if (fast_args(f, batch, heads, kv_heads, dim, bits, pages, page_size, max_pages, window, sinks)) {
        if (window < INT32_MAX) return attend_window_tiles(p, batch, dtype, bits, workspace, st);
        f.a = p;
        f.slots = (float *)workspace;
        return dtype == BW_F16 ? launch_bits<false, __half>(f, bits, st) : launch_bits<false, __nv_bfloat16>(f, bits, st);
    }
    return dtype == BW_F16 ? attend_general<__half>(p, batch, bits, st) : attend_general<__nv_bfloat16>(p, batch, bits, st);
}

}  // namespace bw
