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
#include <type_traits>

#include "early_launch.cuh"

namespace bw {
namespace {

// Division of 32-bit numbers by one that is known on the host: the high half of a product, and shifts (Granlund and Montgomery).
struct Divisor {
    uint32_t d, m;
    int sh1, sh2;
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
        const uint32_t t = __umulhi(m, n);
        return (t + ((n - t) >> sh1)) >> sh2;
    }
};
Divisor divisor(uint32_t d) {
    int l = 0;
    while (l < 32 && ((uint64_t)1 << l) < d) ++l;
    return {d, (uint32_t)((((uint64_t)1 << l) - d) * ((uint64_t)1 << 32) / d + 1), l < 1 ? l : 1, l < 1 ? 0 : l - 1};
}

struct KvRows {
    int64_t tokens, slots;      // rows of tokens in the call; pages * page_size
    int64_t stride[2], head_stride[2];   // of k and v, in elements
    Divisor by_heads, by_page;
    int heads, dim, words, page_size;
    int lanes;                  // of a row: the power of two that holds its pieces
};

// Where a slot's row of a head lies, in rows of the cache.
__device__ __forceinline__ int64_t cache_row(const KvRows &p, int64_t slot, int head) {
    const int64_t page = slot >> 32 ? slot / p.page_size : (int64_t)p.by_page((uint32_t)slot);
    return (page * p.heads + head) * p.page_size + (slot - page * p.page_size);
}

// fp16 not below s (finite, positive), at least 2^-24; infinity beyond fp16's range.
__device__ __forceinline__ __half scale_up(float s) { return __float2half_ru(fmaxf(s, 0x1p-24f)); }

constexpr float MAGIC = 12582912.0f;                         // 1.5 * 2^23: the sum of 0 <= t <= 255 and this has rint(t) in its low bits
constexpr uint32_t MAGIC_BITS = 0x4B400000u;

// Values that a thread takes of a row: whole words of codes at any width.  (Of 8 the work on a row's ends, scale and place was most of it.)
constexpr int E = 16;

// (From L2, as all that a kernel before may have written: the SM's L1 may hold lines from before this kernel's start, at which they were still being written.)
__device__ __forceinline__ float ld_l2(const float *p) { return __ldcg(p); }
__device__ __forceinline__ __half ld_l2(const __half *p) { return __ldcg(p); }
__device__ __forceinline__ __nv_bfloat16 ld_l2(const __nv_bfloat16 *p) { return __ldcg(p); }

// min and max that keep NaN
__device__ __forceinline__ float min_nan(float a, float b) {
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// E values of a row at `at` (fewer than E are left only at the end of a row that is no multiple of E: zeros), and their ends together with 0:
// of 16-bit values in pairs.
template <typename T, bool VEC>
__device__ __forceinline__ void load_values(const T *row, int at, int dim, bool live, float (&x)[E], float &lo, float &hi) {
    lo = hi = 0.0f;
    if constexpr (VEC) {
        uint4 raw[E * sizeof(T) / 16];
#pragma unroll
        for (int i = 0; i < (int)(E * sizeof(T) / 16); ++i) raw[i] = live ? __ldcg(reinterpret_cast<const uint4 *>(row + at) + i) : make_uint4(0, 0, 0, 0);
        const T *v = reinterpret_cast<const T *>(raw);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = to_f32(v[i]);
        if constexpr (sizeof(T) == 2) {
            using T2 = typename std::conditional<__is_same(T, __half), __half2, __nv_bfloat162>::type;
            const T2 *p = reinterpret_cast<const T2 *>(raw);
            T2 a = p[0], b = p[0];
#pragma unroll
            for (int i = 1; i < E / 2; ++i) {
                a = __hmin2_nan(a, p[i]);
                b = __hmax2_nan(b, p[i]);
            }
            lo = min_nan(0.0f, min_nan(to_f32(a.x), to_f32(a.y)));
            hi = max_nan(0.0f, max_nan(to_f32(b.x), to_f32(b.y)));
            return;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = live && at + i < dim ? to_f32(ld_l2(row + at + i)) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        lo = min_nan(lo, x[i]);
        hi = max_nan(hi, x[i]);
    }
}

// One group of lanes a row, each with whole words of codes; a thread has its piece of the key and of the value.  Bound by instruction issue: 16384 tokens
// of 8 heads of 128, fp16 to 8 bits, 27 us, 3.8 TB/s, 66 % of the issue slots (the division in four FMAs and the packed adds of rtn_quantize.cu; one element a
// load and a hardware division each: 174 us).
template <typename T, int BITS, bool VEC>
__global__ void __launch_bounds__(256) kv_append_kernel(const T *__restrict__ k, const T *__restrict__ v, const int64_t *__restrict__ slots,
                                                        const KvRows p, int32_t *k_codes, int32_t *v_codes, __half2 *params) {
    constexpr int WORDS = E * BITS / 32, VPI = 32 / BITS;
    constexpr float Q = (1 << BITS) - 1, RQ = 1.0f / Q;
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t row = blockIdx.x * (256 / p.lanes) + threadIdx.x / p.lanes, token = p.by_heads(row);
    const int head = (int)(row - token * (uint32_t)p.heads), lane = threadIdx.x % p.lanes, at = lane * E;
    const int64_t slot = token < p.tokens ? __ldcg(slots + token) : -1;
    const bool in = slot >= 0 && slot < p.slots, live = in && at < p.dim;
    float x[2][E], lo[2], hi[2];
    // (strides that are read 16 bytes at a time are known to fit 32 bits: a product of 64 bits is three operations)
    const auto offset = [&](int j) {
        if (!in) return (int64_t)0;
        if constexpr (VEC) return (int64_t)((uint64_t)token * (uint32_t)p.stride[j] + (uint64_t)(uint32_t)head * (uint32_t)p.head_stride[j]);
        return token * p.stride[j] + head * p.head_stride[j];
    };
    load_values<T, VEC>(k + offset(0), at, p.dim, live, x[0], lo[0], hi[0]);
    load_values<T, VEC>(v + offset(1), at, p.dim, live, x[1], lo[1], hi[1]);
    for (int d = p.lanes / 2; d; d >>= 1)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            lo[j] = min_nan(lo[j], __shfl_xor_sync(0xffffffffu, lo[j], d));
            hi[j] = max_nan(hi[j], __shfl_xor_sync(0xffffffffu, hi[j], d));
        }
    if (!live) return;
    const int64_t to = cache_row(p, slot, head);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        // (a NaN or an infinity in the row, and what leaves fp16's range, fails the comparison)
        const float span = div_by_recip(__fsub_rn(hi[j], lo[j]), Q, RQ);
        const bool ok = span <= 65504.0f;
        const __half scale = scale_up(span);
        const float s = __half2float(scale), r = __frcp_rn(s), z = rintf(div_by_recip(-lo[j], s, r));      // (at most Q: scale * Q >= hi - lo >= -lo)
        uint32_t words[WORDS] = {};
        if (ok) {
            float c[E];
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                // x / s + z >= -1/2, which is 0 rounded: only the upper end has to be clamped
                const float2 t = fadd2(div_by_recip2(make_float2(x[j][i], x[j][i + 1]), s, r), make_float2(z, z));
                const float2 y = fadd2(make_float2(fminf(t.x, Q), fminf(t.y, Q)), make_float2(MAGIC, MAGIC));
                c[i] = y.x;
                c[i + 1] = y.y;
            }
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                // one shift and add a code; what the magic number adds on the way is a constant
                uint32_t word = 0, extra = 0;
#pragma unroll
                for (int i = VPI - 1; i >= 0; --i) {
                    word = (word << BITS) + __float_as_uint(c[w * VPI + i]);
                    extra = (extra << BITS) + MAGIC_BITS;
                }
                words[w] = word - extra;
            }
        }
        int32_t *dst = (j ? v_codes : k_codes) + to * p.words + lane * WORDS;
        if constexpr (VEC && WORDS == 4) *reinterpret_cast<int4 *>(dst) = make_int4((int)words[0], (int)words[1], (int)words[2], (int)words[3]);
        else if constexpr (VEC && WORDS == 2) *reinterpret_cast<int2 *>(dst) = make_int2((int)words[0], (int)words[1]);
        else {
#pragma unroll
            for (int w = 0; w < WORDS; ++w)
                if (lane * WORDS + w < p.words) dst[w] = (int32_t)words[w];
        }
        if (lane == 0) params[2 * to + j] = ok ? __halves2half2(scale, __float2half_rn(z)) : __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0));
    }
}

// E values of a row: code + 2^23 by one OR, minus 2^23, exact; then scale * code - scale * zero, whose second product is exact (22 bits), in one rounding to fp32
// (none where the zero point is an integer as append writes it: 19 bits); then the result's rounding.
template <typename T, int BITS, bool VEC>
__device__ __forceinline__ void read_piece(const int32_t *codes, uint32_t constants, int lane, int words, int dim, T *dst) {
    constexpr int WORDS = E * BITS / 32, VPI = 32 / BITS;
    const float2 c = __half22float2(*reinterpret_cast<const __half2 *>(&constants));
    const float zero = -c.x * c.y;
    uint32_t w[WORDS] = {};
    if constexpr (WORDS == 4 && VEC) {
        const uint4 u = __ldcg(reinterpret_cast<const uint4 *>(codes) + lane);
        w[0] = u.x;
        w[1] = u.y;
        w[2] = u.z;
        w[3] = u.w;
    } else if constexpr (WORDS == 2 && VEC) {
        const uint2 u = __ldcg(reinterpret_cast<const uint2 *>(codes) + lane);
        w[0] = u.x;
        w[1] = u.y;
    } else {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = lane * WORDS + i < words ? (uint32_t)__ldcg(codes + lane * WORDS + i) : 0u;
    }
    __align__(16) T out[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const uint32_t code = w[i / VPI] >> (i % VPI * BITS) & ((1u << BITS) - 1);
        out[i] = from_f32<T>(__fmaf_rn(c.x, __uint_as_float(0x4B000000u | code) - 8388608.0f, zero));
    }
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)(E * sizeof(T) / 16); ++i) __stcs(reinterpret_cast<uint4 *>(dst) + i, reinterpret_cast<const uint4 *>(out)[i]);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (lane * E + i < dim) dst[i] = out[i];
    }
}

template <typename T, int BITS, bool VEC>
__global__ void __launch_bounds__(256) kv_read_kernel(const int32_t *__restrict__ k_codes, const int32_t *__restrict__ v_codes,
                                                      const uint2 *__restrict__ params, const int64_t *__restrict__ slots, const KvRows p, T *k, T *v) {
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t row = blockIdx.x * (256 / p.lanes) + threadIdx.x / p.lanes, token = p.by_heads(row);
    const int lane = threadIdx.x % p.lanes;
    if (token >= p.tokens || lane * E >= p.dim) return;
    const int64_t slot = __ldcg(slots + token), to = (int64_t)row * p.dim + lane * E;
    if (slot < 0 || slot >= p.slots) {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (lane * E + i < p.dim) k[to + i] = v[to + i] = from_f32<T>(0.0f);
        return;
    }
    const int64_t at = cache_row(p, slot, (int)(row - token * (uint32_t)p.heads));
    const uint2 c = __ldcg(params + at);
    read_piece<T, BITS, VEC>(k_codes + at * p.words, c.x, lane, p.words, p.dim, k + to);
    read_piece<T, BITS, VEC>(v_codes + at * p.words, c.y, lane, p.words, p.dim, v + to);
}

KvRows kv_rows(int64_t tokens, int heads, int dim, int bits, int64_t pages, int page_size) {
    KvRows p = {};
    p.tokens = tokens;
    p.slots = pages * page_size;
    p.heads = heads;
    p.dim = dim;
    p.words = dim * bits / 32;
    p.page_size = page_size;
    p.by_heads = divisor((uint32_t)heads);
    p.by_page = divisor((uint32_t)page_size);
    const int pieces = (dim + E - 1) / E;
    p.lanes = 1;
    while (p.lanes < pieces) p.lanes *= 2;
    return p;
}

unsigned kv_grid(const KvRows &p) {
    const int64_t per = 256 / p.lanes;
    return (unsigned)((p.tokens * p.heads + per - 1) / per);
}

template <typename T, int BITS>
int append_typed(const void *kv, const void *vv, const int64_t *slots, const KvRows &p, int32_t *kc, int32_t *vc, void *params, cudaStream_t st) {
    const T *k = (const T *)kv, *v = (const T *)vv;
    constexpr int V = 16 / sizeof(T);
    bool vec = p.dim % E == 0 && aligned_to(k, 16) && aligned_to(v, 16);
    for (int i = 0; i < 2; ++i)
        for (int64_t stride : {p.stride[i], p.head_stride[i]}) vec = vec && stride % V == 0 && stride >= 0 && stride <= UINT32_MAX;
    return launch_early("kv_append_kernel", vec ? kv_append_kernel<T, BITS, true> : kv_append_kernel<T, BITS, false>, dim3(kv_grid(p)), 256, 0, st, dim3(1), k, v, slots, p,
                        kc, vc, (__half2 *)params);
}
template <typename T>
int append_bits(const void *k, const void *v, const int64_t *slots, const KvRows &p, int bits, int32_t *kc, int32_t *vc, void *params, cudaStream_t st) {
    return bits == 2 ? append_typed<T, 2>(k, v, slots, p, kc, vc, params, st) : bits == 4 ? append_typed<T, 4>(k, v, slots, p, kc, vc, params, st)
                                                                                          : append_typed<T, 8>(k, v, slots, p, kc, vc, params, st);
}

template <typename T, int BITS>
int read_typed(const int32_t *kc, const int32_t *vc, const void *params, const int64_t *slots, const KvRows &p, void *k, void *v, cudaStream_t st) {
    // (k and v are dense and start on 16 bytes: so do all pieces of rows that are whole pieces)
    return launch_early("kv_read_kernel", p.dim % E == 0 ? kv_read_kernel<T, BITS, true> : kv_read_kernel<T, BITS, false>, dim3(kv_grid(p)), 256, 0, st, dim3(1), kc, vc,
                        (const uint2 *)params, slots, p, (T *)k, (T *)v);
}
template <typename T>
int read_bits(const int32_t *kc, const int32_t *vc, const void *params, const int64_t *slots, const KvRows &p, int bits, void *k, void *v, cudaStream_t st) {
    return bits == 2 ? read_typed<T, 2>(kc, vc, params, slots, p, k, v, st) : bits == 4 ? read_typed<T, 4>(kc, vc, params, slots, p, k, v, st)
                                                                                      : read_typed<T, 8>(kc, vc, params, slots, p, k, v, st);
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
