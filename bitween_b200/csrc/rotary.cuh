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
    uint32_t whole;                      // of eight pairs in a row: whether they have one axis
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

// The pieces of a row that are rotated, 16 values each: eight neighbours of the first half with their partners of the second, or 16 neighbours where interleaved;
// behind them 16 neighbours that stay.  `piece` has eight pairs from pair 8 * piece on.  (For rotary dimensions that are multiples of 16.)
struct Turn {
    float2 t[8];                         // cosines and sines
    int at0, at1;                        // where its values begin, eight each
    bool turns;

    __device__ __forceinline__ Turn(const Rotary &p, int64_t token, int piece, bool live) {
        turns = 8 * piece < p.pairs;
        at0 = turns && !p.interleaved ? 8 * piece : 16 * piece;
        at1 = turns && !p.interleaved ? p.pairs + 8 * piece : 16 * piece + 8;
        if (!live || !turns) return;
        if (p.whole >> piece & 1) {
            const int64_t at = __ldcg(p.positions + p.axis[8 * piece] * p.axis_stride + token);
            const bool there = at >= 0 && at < p.max_positions;
            const float4 *from = reinterpret_cast<const float4 *>(p.table + (there ? at : 0) * p.pairs + 8 * piece);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 two = there ? __ldcg(from + i) : make_float4(NAN, NAN, NAN, NAN);
                t[2 * i] = make_float2(two.x, p.sign * two.y);
                t[2 * i + 1] = make_float2(two.z, p.sign * two.w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = turn_of(p, token, 8 * piece + i);
        }
    }
    // Products two an instruction, sums by themselves: packed sums behind packed products came out fused, rounded once for both.
    __device__ __forceinline__ void operator()(const Rotary &p, float (&x)[16]) const {
        if (!turns) return;
        if (p.interleaved) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a = x[2 * i], b = x[2 * i + 1];
                const float2 u = fmul2(make_float2(a, b), make_float2(t[i].x, t[i].x)), v = fmul2(make_float2(b, a), make_float2(t[i].y, t[i].y));
                x[2 * i] = __fsub_rn(u.x, v.x);
                x[2 * i + 1] = __fadd_rn(u.y, v.y);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float2 a = make_float2(x[i], x[i + 1]), b = make_float2(x[8 + i], x[9 + i]), c = make_float2(t[i].x, t[i + 1].x), s = make_float2(t[i].y, t[i + 1].y);
                const float2 ac = fmul2(a, c), bs = fmul2(b, s), bc = fmul2(b, c), as = fmul2(a, s);
                x[i] = __fsub_rn(ac.x, bs.x);
                x[i + 1] = __fsub_rn(ac.y, bs.y);
                x[8 + i] = __fadd_rn(bc.x, as.x);
                x[9 + i] = __fadd_rn(bc.y, as.y);
            }
        }
    }
};

// Eight values, 16-byte aligned.
template <typename T> struct Eight {
    uint4 raw[8 * sizeof(T) / 16];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i) raw[i] = __ldcg(reinterpret_cast<const uint4 *>(p) + i);
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i) reinterpret_cast<uint4 *>(p)[i] = raw[i];
    }
    __device__ __forceinline__ void get(float *x) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(reinterpret_cast<const T *>(raw)[i]);
    }
    __device__ __forceinline__ void put(const float *x) {
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<T *>(raw)[i] = from_f32<T>(x[i]);
    }
};

}  // namespace bw
