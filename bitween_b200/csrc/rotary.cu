// Rotary positions (bw_rotate) and appends to the quantised cache with the rotation on the way (bw_kv_append_rotated).
//
// Pair j of a row's first R values, at (j, j + R/2) or (2j, 2j+1), is turned by the angle of its axis's position:
//     (a, b) -> (a c - b s, b c + a s),   (c, s) = table[position][j]
// The transposed rotation, which the gradient needs, has -s.
#include "kv_rows.cuh"
#include "rotary.cuh"

namespace bw {
namespace {

struct RotateRows {
    const void *x[2];
    void *out[2];
    int64_t stride[2], head_stride[2], tokens;
    int heads[2], dim;
};

// Any size and stride: a warp a row.
template <typename T>
__global__ void __launch_bounds__(256) rotate_general_kernel(const RotateRows p, const Rotary r) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int all = p.heads[0] + p.heads[1];
    const int64_t row = (int64_t)blockIdx.x * 8 + warp, token = row / all;
    if (token >= p.tokens) return;
    int h = (int)(row - token * all);
    const int i = h >= p.heads[0];
    if (i) h -= p.heads[0];
    const T *x = (const T *)p.x[i] + token * p.stride[i] + h * p.head_stride[i];
    T *out = (T *)p.out[i] + (token * p.heads[i] + h) * p.dim;
    for (int d = lane; d < p.dim; d += 32) out[d] = from_f32<T>(turned_value(r, x, token, d));
}

struct AppendRotated {
    RotateRows q;                        // one tensor, or none (no heads)
    const void *k, *v;
    const int64_t *slots;
    int32_t *codes[2];
    __half2 *params;
    KvRows rows;
};

// Any size and stride: a warp a row of q, k or v.
template <typename T, int BITS>
__global__ void __launch_bounds__(256) kv_append_rotated_general_kernel(const AppendRotated p, const Rotary r) {
    constexpr float Q = (1 << BITS) - 1, RQ = 1.0f / Q;
    __shared__ uint8_t s_codes[8][256];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, kv = p.rows.heads, all = p.q.heads[0] + 2 * kv;
    const int64_t row = (int64_t)blockIdx.x * 8 + warp, token = row / all;
    if (token >= p.rows.tokens) return;
    int h = (int)(row - token * all);
    if (h >= 2 * kv) {
        h -= 2 * kv;
        const T *x = (const T *)p.q.x[0] + token * p.q.stride[0] + h * p.q.head_stride[0];
        T *out = (T *)p.q.out[0] + (token * p.q.heads[0] + h) * p.q.dim;
        for (int d = lane; d < p.q.dim; d += 32) out[d] = from_f32<T>(turned_value(r, x, token, d));
        return;
    }
    const int j = h >= kv;
    if (j) h -= kv;
    const int64_t slot = p.slots[token];
    if (slot < 0 || slot >= p.rows.slots) return;
    const T *x = (const T *)(j ? p.v : p.k) + token * p.rows.stride[j] + h * p.rows.head_stride[j];
    float v[8], lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        v[i] = d >= p.rows.dim ? 0.0f : j ? to_f32(x[d]) : turned_value(r, x, token, d);
        lo = min_nan(lo, v[i]);
        hi = max_nan(hi, v[i]);
    }
    for (int d = 16; d; d >>= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, d));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, d));
    }
    const float span = div_by_recip(__fsub_rn(hi, lo), Q, RQ);
    const bool ok = span <= 65504.0f;
    const __half scale = scale_up(span);
    const float s = __half2float(scale), rs = __frcp_rn(s), z = rintf(div_by_recip(-lo, s, rs));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        if (d < p.rows.dim) s_codes[warp][d] = ok ? (uint8_t)fminf(rintf(__fadd_rn(div_by_recip(v[i], s, rs), z)), Q) : 0;
    }
    __syncwarp();
    const int64_t to = cache_row(p.rows, slot, h);
    for (int w = lane; w < p.rows.words; w += 32) {
        uint32_t word = 0;
        for (int i = 0; i < 32 / BITS; ++i) word |= (uint32_t)s_codes[warp][w * (32 / BITS) + i] << (i * BITS);
        p.codes[j][to * p.rows.words + w] = (int32_t)word;
    }
    if (lane == 0) p.params[2 * to + j] = ok ? __halves2half2(scale, __float2half_rn(z)) : __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0));
}

Rotary rotary_of(const bw_rotary &r, bool inverse) {
    Rotary p = {};
    p.table = (const float2 *)r.table;
    p.positions = r.positions;
    p.max_positions = r.max_positions;
    p.axis_stride = r.axis_stride;
    p.pairs = r.rotary_dim / 2;
    p.interleaved = r.interleaved != 0;
    p.sign = inverse ? -1.0f : 1.0f;
    for (int i = 0; i < p.pairs; ++i) p.axis[i] = r.axes ? r.axes[i] : 0;
    return p;
}

template <typename T>
int rotate_typed(const RotateRows &p, const Rotary &r, cudaStream_t st) {
    const int64_t rows = p.tokens * (p.heads[0] + p.heads[1]);
    rotate_general_kernel<T><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(p, r);
    return check_launch("rotate_general_kernel");
}

template <typename T, int BITS>
int append_rotated_typed(const AppendRotated &p, const Rotary &r, cudaStream_t st) {
    const int64_t rows = p.rows.tokens * (p.q.heads[0] + 2 * p.rows.heads);
    kv_append_rotated_general_kernel<T, BITS><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(p, r);
    return check_launch("kv_append_rotated_general_kernel");
}
template <typename T>
int append_rotated_bits(const AppendRotated &p, const Rotary &r, int bits, cudaStream_t st) {
    return bits == 2 ? append_rotated_typed<T, 2>(p, r, st) : bits == 4 ? append_rotated_typed<T, 4>(p, r, st) : append_rotated_typed<T, 8>(p, r, st);
}

}  // namespace

int rotate(const bw_rotary &rotary, int64_t tokens, int dim, int dtype, bool inverse, const void *const *x, const int *heads, const int64_t *strides,
           void *const *out, cudaStream_t st) {
    RotateRows p = {};
    p.tokens = tokens;
    p.dim = dim;
    for (int i = 0; i < 2; ++i) {
        p.x[i] = x[i];
        p.out[i] = out[i];
        p.heads[i] = heads[i];
        p.stride[i] = strides[2 * i];
        p.head_stride[i] = strides[2 * i + 1];
    }
    const Rotary r = rotary_of(rotary, inverse);
    if (dtype == BW_F32) return rotate_typed<float>(p, r, st);
    if (dtype == BW_F16) return rotate_typed<__half>(p, r, st);
    return rotate_typed<__nv_bfloat16>(p, r, st);
}

int kv_append_rotated(const bw_rotary &rotary, const void *q, int q_heads, int64_t q_stride, int64_t q_head_stride, void *q_out, const void *k, const void *v,
                      int dtype, int64_t tokens, const int64_t *strides, const int64_t *slots, int heads, int dim, int bits, int64_t pages, int page_size,
                      int32_t *kc, int32_t *vc, void *params, cudaStream_t st) {
    AppendRotated p = {};
    p.q.x[0] = q;
    p.q.out[0] = q_out;
    p.q.heads[0] = q_heads;
    p.q.stride[0] = q_stride;
    p.q.head_stride[0] = q_head_stride;
    p.q.tokens = tokens;
    p.q.dim = dim;
    p.k = k;
    p.v = v;
    p.slots = slots;
    p.codes[0] = kc;
    p.codes[1] = vc;
    p.params = (__half2 *)params;
    p.rows = kv_rows(tokens, heads, dim, bits, pages, page_size);
    for (int i = 0; i < 2; ++i) {
        p.rows.stride[i] = strides[2 * i];
        p.rows.head_stride[i] = strides[2 * i + 1];
    }
    const Rotary r = rotary_of(rotary, false);
    if (dtype == BW_F32) return append_rotated_bits<float>(p, r, bits, st);
    if (dtype == BW_F16) return append_rotated_bits<__half>(p, r, bits, st);
    return append_rotated_bits<__nv_bfloat16>(p, r, bits, st);
}

}  // namespace bw
