// Log probabilities of given tokens with the entropy and the largest alternatives (bw_token_log_probs), and their gradient.
//
// Of a row x with largest value m:  s = sum 2^u, w = sum 2^u u  with u = (x - m) / ln 2;
//     log p[j] = (x[j] - m) - ln s,   H = ln s - ln2 * w / s
// The gradient of g log p[t] + e H + sum g_i log p[t_i] in x[j] is  p[j] (-(g + sum g_i) - e (log p[j] + H)) + (j == t) g + sum (j == t_i) g_i.
#include "bw_common.cuh"

namespace bw {
namespace {

constexpr int MOST_TOP = 32;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// The order of the alternatives: falling value, rising index; NaN before all.  Larger is better.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0xfffffffeu;                       // (below the mark of no value yet, whatever the index)
    const uint32_t b = __float_as_uint(x + 0.0f);         // (-0 counts as 0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct LogProbs {
    const void *logits;
    const int64_t *tokens;
    float *log_probs, *entropy, *top_log_probs;
    int64_t *top_tokens;
    float4 *stats;                       // m, log2 s, H
    int64_t stride;
    int vocab, top;
};

// Any size and stride: a CTA a row, and a pass over the row for each alternative.
template <typename T>
__global__ void __launch_bounds__(256) log_probs_general_kernel(const LogProbs p) {
    const int64_t row = blockIdx.x;
    const T *x = (const T *)p.logits + row * p.stride;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    __shared__ float s_a[8], s_b[8];
    __shared__ uint64_t s_best[8];
    // the largest value; NaN if there is one
    float m = -INFINITY;
    bool nan = false;
    for (int j = tid; j < p.vocab; j += 256) {
        const float v = to_f32(x[j]);
        nan |= v != v;
        m = fmaxf(m, v);
    }
    if (nan) m = INFINITY;
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (lane == 0) s_a[warp] = m;
    __syncthreads();
    for (int i = 0; i < 8; ++i) m = fmaxf(m, s_a[i]);
    __syncthreads();
    // (a thread's sums in blocks of 32: equal values round the same way each time, and 500 of them in a row were off by 100 half steps)
    float s = 0.0f, w = 0.0f;
    for (int j0 = tid; j0 < p.vocab; j0 += 32 * 256) {
        float sb = 0.0f, wb = 0.0f;
        for (int j = j0; j < p.vocab && j < j0 + 32 * 256; j += 256) {
            const float u = (to_f32(x[j]) - m) * LOG2E, e = exp2f(u);
            sb += e;
            wb += e == 0.0f ? 0.0f : e * u;
        }
        s += sb;
        w += wb;
    }
    for (int d = 16; d; d >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, d);
        w += __shfl_xor_sync(0xffffffffu, w, d);
    }
    if (lane == 0) {
        s_a[warp] = s;
        s_b[warp] = w;
    }
    __syncthreads();
    s = w = 0.0f;
    for (int i = 0; i < 8; ++i) {
        s += s_a[i];
        w += s_b[i];
    }
    // (infinities of either sign as the largest value, and NaN: nothing is known of the row)
    const float log2s = fabsf(m) == INFINITY ? NAN : log2f(s), ln_s = LN2 * log2s, h = ln_s - LN2 * (w / s);
    if (tid == 0) {
        if (p.tokens) {
            const int64_t t = p.tokens[row];
            p.log_probs[row] = t < 0 ? 0.0f : t >= p.vocab ? NAN : (to_f32(x[t]) - m) - ln_s;
        }
        if (p.entropy) p.entropy[row] = h;
        if (p.stats) p.stats[row] = make_float4(m, log2s, h, 0.0f);
    }
    uint64_t last = ~0ull;               // (order << 32) | ~index
    for (int i = 0; i < p.top; ++i) {
        uint64_t best = 0;
        for (int j = tid; j < p.vocab; j += 256) {
            const uint64_t key = (uint64_t)order_of(to_f32(x[j])) << 32 | (uint32_t)~j;
            if (key < last && key > best) best = key;
        }
        for (int d = 16; d; d >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, d));
        __syncthreads();
        if (lane == 0) s_best[warp] = best;
        __syncthreads();
        for (int k = 0; k < 8; ++k) best = max(best, s_best[k]);
        last = best;
        const uint32_t at = ~(uint32_t)best;
        if (tid == 0 && at < (uint32_t)p.vocab) {
            p.top_tokens[row * p.top + i] = at;
            p.top_log_probs[row * p.top + i] = (to_f32(x[at]) - m) - ln_s;
        }
    }
}

struct LogProbsGrad {
    const void *logits;
    void *grad;
    const int64_t *tokens, *top_tokens;
    const float4 *stats;
    const float *g, *e, *g_top;
    int64_t stride;
    int vocab, top;
};

template <typename T>
__global__ void __launch_bounds__(256) log_probs_grad_general_kernel(const LogProbsGrad p) {
    const int64_t row = blockIdx.x;
    const T *x = (const T *)p.logits + row * p.stride;
    T *out = (T *)p.grad + row * p.vocab;
    const float4 st = p.stats[row];
    const int64_t t = p.tokens ? p.tokens[row] : -1;
    const float g = p.g && t >= 0 ? (t < p.vocab ? p.g[row] : NAN) : 0.0f, e = p.e ? p.e[row] : 0.0f;
    float all = g;
    if (p.g_top)
        for (int i = 0; i < p.top; ++i) all += p.g_top[row * p.top + i];
    const float c = -fmaf(e, st.z, all);
    for (int j = threadIdx.x; j < p.vocab; j += 256) {
        const float u = (to_f32(x[j]) - st.x) * LOG2E - st.y, prob = exp2f(u);
        float v = prob == 0.0f ? 0.0f : prob * fmaf(-e * LN2, u, c);
        if (j == t) v += g;
        if (p.g_top)
            for (int i = 0; i < p.top; ++i)
                if (p.top_tokens[row * p.top + i] == j) v += p.g_top[row * p.top + i];
        out[j] = from_f32<T>(v);
    }
}

template <typename T>
int log_probs_typed(const LogProbs &p, int64_t rows, cudaStream_t st) {
    log_probs_general_kernel<T><<<(unsigned)rows, 256, 0, st>>>(p);
    return check_launch("log_probs_general_kernel");
}
template <typename T>
int log_probs_grad_typed(const LogProbsGrad &p, int64_t rows, cudaStream_t st) {
    log_probs_grad_general_kernel<T><<<(unsigned)rows, 256, 0, st>>>(p);
    return check_launch("log_probs_grad_general_kernel");
}

}  // namespace

int token_log_probs(const void *logits, int dtype, int64_t rows, int64_t vocab, int64_t stride, const int64_t *tokens, float *log_probs, float *entropy,
                    int top, float *top_log_probs, int64_t *top_tokens, float *stats, cudaStream_t st) {
    const LogProbs p = {logits, tokens, log_probs, entropy, top_log_probs, top_tokens, (float4 *)stats, stride, (int)vocab, top};
    if (dtype == BW_F32) return log_probs_typed<float>(p, rows, st);
    if (dtype == BW_F16) return log_probs_typed<__half>(p, rows, st);
    return log_probs_typed<__nv_bfloat16>(p, rows, st);
}

int token_log_probs_grad(const void *logits, int dtype, int64_t rows, int64_t vocab, int64_t stride, const int64_t *tokens, const float *stats,
                         const float *g, const float *e, int top, const int64_t *top_tokens, const float *g_top, void *grad, cudaStream_t st) {
    const LogProbsGrad p = {logits, grad, tokens, top_tokens, (const float4 *)stats, g, e, g_top, stride, (int)vocab, top};
    if (dtype == BW_F32) return log_probs_grad_typed<float>(p, rows, st);
    if (dtype == BW_F16) return log_probs_grad_typed<__half>(p, rows, st);
    return log_probs_grad_typed<__nv_bfloat16>(p, rows, st);
}

}  // namespace bw
