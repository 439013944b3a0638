// The quantised key-value cache: rows written (bw_kv_append) and read back (bw_kv_read).
//
// A row is one token's D values of one head.  With Q = 2^bits - 1, lo = min(row, 0), hi = max(row, 0):
//     scale = (hi - lo) / Q rounded UP to fp16, at least 2^-24;  zero = rne(-lo / scale);  code = clamp(rne(x / scale + zero), 0, Q)
// which is quantize_rtn's rounding of a group whose range holds zero, with the scale that is stored: rounded up so that the
// largest values of the row stay inside the codes, and never zero.  Every step is one correctly rounded fp32 operation, so the codes
// are those of the same steps in any IEEE arithmetic.  A row with a NaN or an infinity, or of more than fp16's range, gets scale NaN:
// it reads back as NaN instead of as wrong numbers.
//
// Layout: codes [pages][heads][page_size][D * bits / 32] words, packed like weights; constants [pages][heads][page_size][4]
// fp16: (scale, zero) of the key, then of the value: what an attention step needs of one token lies in 8 bytes.
#include "bw_common.cuh"

namespace bw {
namespace {

struct KvRows {
    int64_t tokens, slots;      // rows of tokens in the call; pages * page_size
    int64_t stride[2], head_stride[2];   // of k and v, in elements
    int heads, dim, words, page_size;
    int lanes;                  // of a row: the power of two that holds its words, at most 32
};

// Where a slot's row of a head lies, in rows of the cache.
__device__ __forceinline__ int64_t cache_row(const KvRows &p, int64_t slot, int head) {
    const int64_t page = slot / p.page_size;
    return (page * p.heads + head) * p.page_size + (slot - page * p.page_size);
}

// fp16 not below s (finite, positive), at least 2^-24; infinity beyond fp16's range.
__device__ __forceinline__ __half scale_up(float s) { return __float2half_ru(fmaxf(s, 0x1p-24f)); }

// One group of lanes a row; a lane holds whole words, so that it packs them by itself.
template <typename T, int BITS>
__global__ void __launch_bounds__(256) kv_append_kernel(const T *__restrict__ k, const T *__restrict__ v, const int64_t *__restrict__ slots,
                                                        KvRows p, int32_t *k_codes, int32_t *v_codes, __half2 *params) {
    constexpr int VPI = 32 / BITS, WORDS = BITS == 8 ? 2 : 1;      // words a lane: 256 values of 8 bits are 64 words
    constexpr float Q = (1 << BITS) - 1;
    const int64_t row = (int64_t)blockIdx.x * (256 / p.lanes) + threadIdx.x / p.lanes;
    const int lane = threadIdx.x % p.lanes;
    const bool is_v = blockIdx.y;
    const int64_t token = row / p.heads;
    const int head = (int)(row - token * p.heads);
    const int64_t slot = token < p.tokens ? slots[token] : -1;
    const bool live = slot >= 0 && slot < p.slots;
    const T *src = (is_v ? v : k) + (live ? token * p.stride[is_v] + head * p.head_stride[is_v] : 0);

    float x[WORDS][VPI], lo = 0.0f, hi = 0.0f;
    bool fine = true;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
        const int at = (lane + w * p.lanes) * VPI;
#pragma unroll
        for (int i = 0; i < VPI; ++i) {
            x[w][i] = live && at < p.dim ? to_f32(src[at + i]) : 0.0f;
            lo = fminf(lo, x[w][i]);
            hi = fmaxf(hi, x[w][i]);
            fine &= isfinite(x[w][i]);
        }
    }
    for (int d = p.lanes / 2; d; d >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        fine &= (bool)__shfl_xor_sync(0xffffffffu, (int)fine, d);
    }
    const __half scale = scale_up(__fdiv_rn(__fsub_rn(hi, lo), Q));
    fine &= !__hisinf(scale);
    const float s = __half2float(scale), z = fminf(rintf(__fdiv_rn(-lo, s)), Q);
    if (!live) return;
    const int64_t at = cache_row(p, slot, head);
    int32_t *dst = (is_v ? v_codes : k_codes) + at * p.words;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < VPI; ++i) {
            const float c = fminf(fmaxf(rintf(__fadd_rn(__fdiv_rn(x[w][i], s), z)), 0.0f), Q);
            word |= (fine ? (uint32_t)c : 0u) << (i * BITS);
        }
        if (lane + w * p.lanes < p.words) dst[lane + w * p.lanes] = (int32_t)word;
    }
    if (lane == 0) params[2 * at + is_v] = fine ? __halves2half2(scale, __float2half_rn(z)) : __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0));
}

template <typename T, int BITS>
__global__ void __launch_bounds__(256) kv_read_kernel(const int32_t *__restrict__ k_codes, const int32_t *__restrict__ v_codes,
                                                      const __half2 *__restrict__ params, const int64_t *__restrict__ slots, KvRows p, T *k, T *v) {
    constexpr int VPI = 32 / BITS;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;       // a word of the output, both tensors' rows dense
    const int64_t row = i / p.words;
    const int word = (int)(i - row * p.words);
    const bool is_v = blockIdx.y;
    const int64_t token = row / p.heads;
    if (token >= p.tokens) return;
    const int64_t slot = slots[token];
    T *dst = (is_v ? v : k) + row * p.dim + word * VPI;
    if (slot < 0 || slot >= p.slots) {
#pragma unroll
        for (int j = 0; j < VPI; ++j) dst[j] = from_f32<T>(0.0f);
        return;
    }
    const int64_t at = cache_row(p, slot, (int)(row - token * p.heads));
    const uint32_t w = (uint32_t)(is_v ? v_codes : k_codes)[at * p.words + word];
    const float2 c = __half22float2(params[2 * at + is_v]);
#pragma unroll
    for (int j = 0; j < VPI; ++j) dst[j] = from_f32<T>(c.x * ((float)((w >> (j * BITS)) & ((1u << BITS) - 1)) - c.y));
}

KvRows kv_rows(int64_t tokens, int heads, int dim, int bits, int64_t pages, int page_size) {
    KvRows p = {};
    p.tokens = tokens;
    p.slots = pages * page_size;
    p.heads = heads;
    p.dim = dim;
    p.words = dim * bits / 32;
    p.page_size = page_size;
    p.lanes = 1;
    while (p.lanes < p.words && p.lanes < 32) p.lanes *= 2;
    return p;
}

template <typename T>
int append_bits(const void *k, const void *v, const int64_t *slots, const KvRows &p, int bits, int32_t *kc, int32_t *vc, void *params, cudaStream_t st) {
    const int64_t rows = p.tokens * p.heads, per = 256 / p.lanes;
    const dim3 grid((unsigned)((rows + per - 1) / per), 2);
    if (bits == 2) kv_append_kernel<T, 2><<<grid, 256, 0, st>>>((const T *)k, (const T *)v, slots, p, kc, vc, (__half2 *)params);
    else if (bits == 4) kv_append_kernel<T, 4><<<grid, 256, 0, st>>>((const T *)k, (const T *)v, slots, p, kc, vc, (__half2 *)params);
    else kv_append_kernel<T, 8><<<grid, 256, 0, st>>>((const T *)k, (const T *)v, slots, p, kc, vc, (__half2 *)params);
    return check_launch("kv_append_kernel");
}

template <typename T>
int read_bits(const int32_t *kc, const int32_t *vc, const void *params, const int64_t *slots, const KvRows &p, int bits, void *k, void *v, cudaStream_t st) {
    const dim3 grid((unsigned)((p.tokens * p.heads * p.words + 255) / 256), 2);
    if (bits == 2) kv_read_kernel<T, 2><<<grid, 256, 0, st>>>(kc, vc, (const __half2 *)params, slots, p, (T *)k, (T *)v);
    else if (bits == 4) kv_read_kernel<T, 4><<<grid, 256, 0, st>>>(kc, vc, (const __half2 *)params, slots, p, (T *)k, (T *)v);
    else kv_read_kernel<T, 8><<<grid, 256, 0, st>>>(kc, vc, (const __half2 *)params, slots, p, (T *)k, (T *)v);
    return check_launch("kv_read_kernel");
}

}  // namespace

int kv_append(const void *k, const void *v, int dtype, int64_t tokens, const int64_t *strides, const int64_t *slots, int heads, int dim, int bits,
              int64_t pages, int page_size, int32_t *kc, int32_t *vc, void *params, cudaStream_t st) {
    KvRows p = kv_rows(tokens, heads, dim, bits, pages, page_size);
    for (int i = 0; i < 2; ++i) {
        p.stride[i] = strides[2 * i];
        p.head_stride[i] = strides[2 * i + 1];
    }
    if (dtype == BW_F32) return append_bits<float>(k, v, slots, p, bits, kc, vc, params, st);
    if (dtype == BW_F16) return append_bits<__half>(k, v, slots, p, bits, kc, vc, params, st);
    return append_bits<__nv_bfloat16>(k, v, slots, p, bits, kc, vc, params, st);
}

int kv_read(const int32_t *kc, const int32_t *vc, const void *params, int heads, int dim, int bits, int64_t pages, int page_size,
            const int64_t *slots, int64_t tokens, void *k, void *v, int dtype, cudaStream_t st) {
    const KvRows p = kv_rows(tokens, heads, dim, bits, pages, page_size);
    if (dtype == BW_F32) return read_bits<float>(kc, vc, params, slots, p, bits, k, v, st);
    if (dtype == BW_F16) return read_bits<__half>(kc, vc, params, slots, p, bits, k, v, st);
    return read_bits<__nv_bfloat16>(kc, vc, params, slots, p, bits, k, v, st);
}

}  // namespace bw
