// Rotary positions, as the kernels that rotate take them (bw_rotary of the C ABI, by value).
#pragma once
#include "bw_common.cuh"

namespace bw {

struct Rotary {
    const float2 *table;                 // [max_positions][pairs]: cosine, sine
    const int64_t *positions;
    int64_t max_positions, axis_stride;
    int pairs, interleaved;
    float sign;                          // of the sines: -1 turns back
    uint8_t axis[128];                   // of each pair
};

// (From L2, as all that a kernel before may have written.)  A position outside the table gives NaN.
__device__ __forceinline__ float2 turn_of(const Rotary &p, int64_t token, int pair) {
    const int64_t at = __ldcg(p.positions + p.axis[pair] * p.axis_stride + token);
    if (at < 0 || at >= p.max_positions) return make_float2(NAN, NAN);
    const float2 t = __ldcg(p.table + at * p.pairs + pair);
    return make_float2(t.x, p.sign * t.y);
}

// Each operation rounded once: what rows of the cache hold is defined to the bit.
__device__ __forceinline__ float turned_first(float a, float b, float2 t) { return __fsub_rn(__fmul_rn(a, t.x), __fmul_rn(b, t.y)); }
__device__ __forceinline__ float turned_second(float a, float b, float2 t) { return __fadd_rn(__fmul_rn(b, t.x), __fmul_rn(a, t.y)); }

// Value d of a rotated row.
template <typename T>
__device__ __forceinline__ float turned_value(const Rotary &p, const T *row, int64_t token, int d) {
    if (d >= 2 * p.pairs) return to_f32(row[d]);
    const int pair = p.interleaved ? d / 2 : d % p.pairs, first = p.interleaved ? 2 * pair : pair, second = p.interleaved ? first + 1 : pair + p.pairs;
    const float a = to_f32(row[first]), b = to_f32(row[second]);
    const float2 t = turn_of(p, token, pair);
    return d == first ? turned_first(a, b, t) : turned_second(a, b, t);
}

}  // namespace bw
