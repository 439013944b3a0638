// Rows of the quantised key-value cache: where they lie, and the rounding of their constants (kv_cache.cu has the definition).
#pragma once
#include "bw_common.cuh"

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
inline Divisor divisor(uint32_t d) {
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

// Values that a thread takes of a row: whole words of codes at any width.  (Of 8 the work on a row's ends, scale and place was most of it.)
constexpr int E = 16;

inline KvRows kv_rows(int64_t tokens, int heads, int dim, int bits, int64_t pages, int page_size) {
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

}  // namespace
}  // namespace bw
