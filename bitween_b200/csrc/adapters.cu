// Low-rank adapters of many requests beside a shared projection: bw_adapter_forward, bw_adapter_backward.
//
//     h[t] = down[i] x[t],  y[t] = base[t] + f_i up[i]^T h[t],  i = index[t]  (none below 0)
//     dh[t] = up[i] dy[t],  dx[t] = f_i down[i]^T dh[t],  d_down[i] = f_i sum dh[t] x[t]^T,  d_up[i] = f_i sum h[t] dy[t]^T
//
// Both matrices of an adapter are stored rank-major, down [n][rank][K] and up [n][rank][N], so that forward and backward are the
// same three passes: "shrink" (rows times a matrix of long rows -> rank values), "expand" (the reverse) and "outer" (sums of
// products over an adapter's tokens).
#include "bw_common.cuh"

namespace bw {
namespace {

template <typename T>
__global__ void __launch_bounds__(128) adapter_shrink_general_kernel(const T *__restrict__ x, int64_t M, int64_t K, const T *__restrict__ w, int n, int r,
                                                                     const int32_t *__restrict__ index, float *h) {
    const int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / 32, t = i / r;
    const int j = (int)(i - t * r), lane = threadIdx.x % 32;
    if (t >= M) return;
    const int a = index[t];
    float s = 0.0f;
    if (a >= 0 && a < n)
        for (int64_t k = lane; k < K; k += 32) s += to_f32(x[t * K + k]) * to_f32(w[((int64_t)a * r + j) * K + k]);
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (lane == 0) h[i] = a < n ? s : NAN;
}

template <typename T>
__global__ void __launch_bounds__(256) adapter_expand_general_kernel(const float *__restrict__ h, int64_t M, int64_t N, const T *__restrict__ w, int n, int r,
                                                                     const int32_t *__restrict__ index, const float *__restrict__ scaling, const T *base, T *out) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= N) return;
    for (int64_t t = blockIdx.y; t < M; t += gridDim.y) {
        const int a = index[t];
        float s = a < n ? 0.0f : NAN;
        if (a >= 0 && a < n) {
            for (int j = 0; j < r; ++j) s += h[t * r + j] * to_f32(w[((int64_t)a * r + j) * N + c]);
            if (scaling) s *= scaling[a];
        }
        out[t * N + c] = from_f32<T>(base ? to_f32(base[t * N + c]) + s : s);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) adapter_outer_general_kernel(const float *__restrict__ h, const T *__restrict__ x, int64_t M, int64_t N, int r,
                                                                    const int32_t *__restrict__ index, const float *__restrict__ scaling, T *dw) {
    const int64_t c = (int64_t)blockIdx.y * 256 + threadIdx.x;
    const int a = blockIdx.x / r, j = blockIdx.x % r;
    if (c >= N) return;
    float s = 0.0f;
    for (int64_t t = 0; t < M; ++t)
        if (index[t] == a) s += h[t * r + j] * to_f32(x[t * N + c]);
    dw[(int64_t)blockIdx.x * N + c] = from_f32<T>(scaling ? s * scaling[a] : s);
}

template <typename T>
int shrink(const void *x, int64_t M, int64_t K, const void *w, int n, int r, const int32_t *index, float *h, cudaStream_t st) {
    adapter_shrink_general_kernel<T><<<(unsigned)((M * r + 3) / 4), 128, 0, st>>>((const T *)x, M, K, (const T *)w, n, r, index, h);
    return check_launch("adapter_shrink_general_kernel");
}
template <typename T>
int expand(const float *h, int64_t M, int64_t N, const void *w, int n, int r, const int32_t *index, const float *scaling, const void *base, void *out,
           cudaStream_t st) {
    adapter_expand_general_kernel<T><<<dim3((unsigned)((N + 255) / 256), (unsigned)(M < 16384 ? M : 16384)), 256, 0, st>>>(
        h, M, N, (const T *)w, n, r, index, scaling, (const T *)base, (T *)out);
    return check_launch("adapter_expand_general_kernel");
}
template <typename T>
int outer(const float *h, const void *x, int64_t M, int64_t N, int n, int r, const int32_t *index, const float *scaling, void *dw, cudaStream_t st) {
    adapter_outer_general_kernel<T><<<dim3((unsigned)(n * r), (unsigned)((N + 255) / 256)), 256, 0, st>>>(h, (const T *)x, M, N, r, index, scaling, (T *)dw);
    return check_launch("adapter_outer_general_kernel");
}

template <typename T>
int forward(const void *x, int64_t M, int64_t N, int64_t K, const void *down, const void *up, int n, int r, const int32_t *index, const float *scaling,
            const void *base, void *out, float *h, cudaStream_t st) {
    int rc = shrink<T>(x, M, K, down, n, r, index, h, st);
    return rc != BW_OK ? rc : expand<T>(h, M, N, up, n, r, index, scaling, base, out, st);
}
template <typename T>
int backward(const void *dy, const void *x, int64_t M, int64_t N, int64_t K, const void *down, const void *up, int n, int r, const int32_t *index,
             const float *scaling, const float *h, void *dx, void *d_down, void *d_up, float *dh, cudaStream_t st) {
    int rc = BW_OK;
    if (M > 0 && (dx || d_down)) rc = shrink<T>(dy, M, N, up, n, r, index, dh, st);
    if (rc == BW_OK && M > 0 && dx) rc = expand<T>(dh, M, K, down, n, r, index, scaling, nullptr, dx, st);
    if (rc == BW_OK && d_down) rc = outer<T>(dh, x, M, K, n, r, index, scaling, d_down, st);
    if (rc == BW_OK && d_up) rc = outer<T>(h, dy, M, N, n, r, index, scaling, d_up, st);
    return rc;
}

}  // namespace

size_t adapter_hidden_bytes(int64_t M, int64_t, int, int r) { return (size_t)M * r * sizeof(float); }
size_t adapter_backward_bytes(int64_t M, int64_t, int64_t, int, int r) { return (size_t)M * r * sizeof(float); }

int adapter_forward(const void *x, int dtype, int64_t M, int64_t N, int64_t K, const void *down, const void *up, int n, int r, const int32_t *index,
                    const float *scaling, const void *base, void *out, float *h, cudaStream_t st) {
    if (dtype == BW_F16) return forward<__half>(x, M, N, K, down, up, n, r, index, scaling, base, out, h, st);
    return forward<__nv_bfloat16>(x, M, N, K, down, up, n, r, index, scaling, base, out, h, st);
}
int adapter_backward(const void *dy, int dtype, const void *x, int64_t M, int64_t N, int64_t K, const void *down, const void *up, int n, int r,
                     const int32_t *index, const float *scaling, const float *h, void *dx, void *d_down, void *d_up, void *workspace, cudaStream_t st) {
    if (dtype == BW_F16) return backward<__half>(dy, x, M, N, K, down, up, n, r, index, scaling, h, dx, d_down, d_up, (float *)workspace, st);
    return backward<__nv_bfloat16>(dy, x, M, N, K, down, up, n, r, index, scaling, h, dx, d_down, d_up, (float *)workspace, st);
}

}  // namespace bw
