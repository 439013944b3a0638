// The tiled kernels of attention over the quantised cache: all tokens (kv_attend.cu) or those of a window and the sinks (kv_attend_window.cu).
#pragma once
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "early_launch.cuh"

namespace bw {

struct AttendArgs {
    const void *q;
    const int32_t *k_codes, *v_codes;
    const __half2 *params;                     // [row][2]: (scale, zero) of the key, of the value
    const int32_t *table, *lengths;
    void *out;
    int64_t q_stride, q_head_stride, table_stride, pages;
    int heads, kv_heads, dim, words, page_size, max_pages;
    float alpha;
    int window, sinks;                         // tokens t < sinks or t >= length - window are visible
};

namespace {

// ---- head dimensions of 64, 128 and 256, pages of whole tiles of 16 tokens --------------------------------------------
//
// A warp takes steps of one or two tiles of 16 tokens; K and V codes are the A operand of mma.sync.m16n8k16 (16 tokens, then 16 values, by
// 8 heads of the group), so that one read of the cache serves all heads that share it:
//   scores   S[t][h] = scale_t * (sum_d code[t][d] q[h][d] - zero_t * sum_d q[h][d]).  A code, masked out of its word, IS an fp16 number:
//            the subnormal code * 2^-24 (tensor cores take subnormals exactly), so expanding two codes costs one AND.  Codes that stand in
//            higher bits of their byte (`planes`) are larger by a power of two and get accumulators of their own.  Scale and zero point
//            are applied to the sums, in fp32: nothing is rounded.
//   weights  p = 2^(x - m); p * (value's scale) goes to fp16 for the second product.  m covers p * scale, so that this stays in fp16's
//            range whatever the scales are; it moves only when some p * scale is about to leave that range (one vote a step), and then the largest of the step becomes 2^12: a
//            weight counts to within 2^-37 of the largest.  (With 1 at the top weights below 2^-25 of it left the numerator and stayed in the sum of weights: many of them
//            beside a token that dominates were lost.)  The
//            rest p - fp16(p) is multiplied as well: 22 bits of a weight count, for bf16 results too (without, they were off by up to 2^-12 of sum w |v|,
//            an eighth of their own rounding).
//   values   O[d][h] += (code - zero_t)[d][t] * p[t][h]: 1024 + code by one OR, minus (1024 + the zero point's nearest code), exact.  What the zero point is off that code
//            (nothing where append wrote it) is the same for all d: sum_t p * (nearest code - zero_t), in fp32 beside the sum of weights, is added at the end.  ldmatrix.trans puts
//            16 bits (2 to 8 codes) of two tokens beside each other, as the operand wants them.
// Groups of up to 4 heads fill half of the eight columns: their steps are two tiles, whose scores share one set of registers (columns 0 to 3
// the first tile's, 4 to 7 the second's), which halves the work on weights; the columns' sums meet at the end, and where one tile's values are
// multiplied the other's columns take the rests of its weights: they cost no MMA (both columns of a head go by one maximum).
//
// Bound by the bytes of the cache up to here, and by instruction issue at 2 and 4 bits.  Each warp has a ring of steps in shared memory, filled by
// 16-byte cp.async and read by it alone: no block-wide barrier in the loop, and the loads in flight cost no registers.
//
// Work: all steps of all sequences and heads in one line, an equal share of it to each CTA, whatever the lengths are; a part of a sequence
// counts START steps more, which is what its start and end cost.  What a share has of a sequence that others have too goes to scratch (running
// maximum, sum, unnormalised output), and kv_attend_join_kernel joins it.  Where tables are short enough for a cluster of CTAs to take a
// sequence and head, it does, and joins its parts through shared memory: no scratch, no second launch.
constexpr int WARPS = 4, TILE = 16, START = 16;
constexpr int MOST_CTAS = 592;              // shares of a call: four CTAs on each of 148 SMs
constexpr int CLUSTER_ROUNDS = 5;           // tables of up to so many steps a warp: clusters

struct FastArgs {
    AttendArgs a;
    int64_t batch;
    float *slots;                           // [2 * MOST_CTAS][cols] x ([dim] output; then [2]: maximum, sum)
    int units;                              // of a sequence: cache heads x blocks of query heads
    int blocks, cols;                       // blocks of query heads of a cache head; heads of a block
    int ctas, most_tiles, tiles_per_page;
    int pair;                               // tiles of a step
    int cluster;                            // CTAs of a cluster, one unit each; 0: shares of the line of work, and a join
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
// (a predicate, not a branch: the loop has ten of these)
__device__ __forceinline__ void copy16_if(bool ok, uint32_t to, const uint8_t *from) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %0, 0;\n @p cp.async.cg.shared.global [%1], [%2], 16;\n}" ::"r"((int)ok), "r"(to), "l"(from) : "memory");
}
// (x & bits) | magic in one operation: the compiler, which knows both constants, makes two of it.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t bits, uint32_t magic) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(bits), "r"(magic));
    return y;
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
template <int WORDS> __device__ __forceinline__ void load_words(uint32_t at, uint32_t *w) {
    if constexpr (WORDS == 1) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
    else if constexpr (WORDS == 2) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
    else asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_transposed2(uint32_t at, uint32_t *x) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_transposed4(uint32_t at, uint32_t *x) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
}

namespace cg = cooperative_groups;

// A part's share of the sum of weights, given its maximum, its sum and the largest maximum.  (Without a finite score it has none, but for the mark of a bad
// page or length.)
__device__ __forceinline__ float part_of(float m, float l, float top) { return m == -INFINITY ? (l == l ? 0.0f : NAN) : l * ex2(m - top); }

// Tiles of a sequence within its table; its true length goes beside it.
__device__ __forceinline__ int tiles_of(int n, int most) {
    const int t = n > 0 ? (n - 1) / TILE + 1 : 0;
    return t < most ? t : most;
}
// With a window: the tiles that hold a visible token of a sequence of n, numbered on without the ones between the sinks' and the window's.  (Each of them
// holds one: without a window's token none is the window's.)
struct Visible {
    int tiles, head, skip;                     // all; the sinks'; those left out behind them
    int first;                                 // of the window's tokens
    __device__ __forceinline__ Visible(const FastArgs &p, int n) {
        const int all = tiles_of(n, p.most_tiles), sinks = p.a.sinks / TILE + (p.a.sinks % TILE != 0);
        first = n > p.a.window ? n - p.a.window : 0;
        head = sinks < all ? sinks : all;
        const int from = p.a.window ? first / TILE : all, start = from > head ? (from < all ? from : all) : head;
        skip = start - head;
        tiles = all - skip;
    }
    __device__ __forceinline__ int tile(int i) const { return i < head ? i : i + skip; }
    __device__ __forceinline__ bool operator()(const FastArgs &p, int t) const { return t < p.a.sinks || (t >= first && p.a.window); }
    __device__ __forceinline__ bool one(const FastArgs &p, int n) const {      // whether it is one token
        const int s = p.a.sinks < n ? p.a.sinks : n, f = p.a.window ? (first > s ? first : s) : n;
        return s + (n - f) == 1;
    }
};
// Tiles of a sequence's work.
template <bool WINDOW>
__device__ __forceinline__ int work_tiles(const FastArgs &p, int n) {
    if constexpr (WINDOW) return Visible(p, n).tiles;
    else return tiles_of(n, p.most_tiles);
}
// What a unit (a block of heads of a sequence) counts in the line of work; 0 for an empty sequence.
template <bool WINDOW>
__device__ __forceinline__ int weight_of(const FastArgs &p, int64_t b) {
    const int tiles = work_tiles<WINDOW>(p, __ldcg(p.a.lengths + b));
    return tiles ? (tiles + p.pair - 1) / p.pair + START : 0;
}
// The steps of one CTA's share of `total`.  Shares of less than two steps a warp are not worth another CTA.
__device__ __forceinline__ int64_t share(const FastArgs &p, int64_t total) {
    const int64_t even = (total + p.ctas - 1) / p.ctas;
    return even < 2 * WARPS ? 2 * WARPS : even;
}

// How a tile lies in shared memory: 16 rows of keys, 16 of values, 16 constants; the 16-byte pieces of a row are exchanged by row so that eight
// rows' pieces of one number (ldmatrix) lie in different banks.
template <int BITS, int DIM> struct Shape {
    static constexpr int PLANES = 8 / BITS;                 // places of a code in a byte
    static constexpr int ROW = DIM * BITS / 8, PIECES = ROW / 16;
    static constexpr int KW = ROW / 16;                     // words of a key row that a lane holds
    static constexpr int MMAS = DIM / 16;                   // of a tile's keys, and of its values
    static constexpr int BYTES = 32 * ROW + 128;
    static constexpr int STRIDE = DIM + 1;                  // of a column's sums in shared memory
    static __device__ __forceinline__ int swizzle(int row) { return ROW >= 128 ? row & 7 : ROW == 64 ? row >> 1 & 3 : ROW == 32 ? row >> 2 & 1 : 0; }
};

template <typename T, int BITS, int DIM, int NB, int PAIR>
struct Config {
    static constexpr int COLS = 8 * NB, STEP = PAIR * Shape<BITS, DIM>::BYTES;
    static constexpr int STAGES = STEP <= 2304 ? 4 : STEP <= 4352 ? 3 : 2;      // of a warp's ring: 9 to 17 KB
    static constexpr int RING = WARPS * STAGES * STEP, SUMS = WARPS * COLS * Shape<BITS, DIM>::STRIDE * 4;
    static constexpr int SMEM = RING > SUMS ? RING : SUMS;
    static constexpr int CTAS = DIM == 256 ? 2 : NB == 2 ? (DIM == 64 ? 3 : 2) : BITS == 8 && DIM == 128 ? 3 : 4;      // an SM, which registers are made to fit
};

template <typename T, int BITS, int DIM, int NB, int PAIR, bool WINDOW>
__global__ void __launch_bounds__(32 * WARPS, (Config<T, BITS, DIM, NB, PAIR>::CTAS)) kv_attend_kernel(const FastArgs p) {
    using S = Shape<BITS, DIM>;
    using C = Config<T, BITS, DIM, NB, PAIR>;
    static_assert(PAIR == 1 || NB == 1, "steps of two tiles are for groups of up to four heads");
    constexpr int COLS = C::COLS, STAGES = C::STAGES, HEADS = PAIR == 2 ? 4 : COLS;
    const AttendArgs &a = p.a;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
    extern __shared__ __align__(128) uint8_t smem[];        // the warps' rings; at the end of a part, their sums
    __shared__ __align__(16) __half sq[HEADS][DIM + 8];
    __shared__ float s_factor[HEADS], s_sum[HEADS], s_m[WARPS][COLS], s_l[WARPS][COLS];
    __shared__ float2 s_total[HEADS];                       // maximum and sum of this CTA's part
    float *s_o = reinterpret_cast<float *>(smem);
    const uint32_t ring = smem_addr(smem) + warp * (STAGES * C::STEP);
    pdl_wait();
    pdl_launch_dependents();

    // this CTA's share of the line of work, and the sequence in which it starts
    int64_t at, end, b = 0, before = 0;      // `before`: work in front of sequence b, of one unit
    const int rank = p.cluster ? (int)(blockIdx.x % p.cluster) : 0;
    const int64_t item = p.cluster ? blockIdx.x / p.cluster : 0;
    if (p.cluster) {
        b = item / p.units;
        at = 0;
        end = INT64_MAX;
    } else {
        int64_t total = 0;
        int mine = 0;
        for (int64_t i = lane; i < p.batch; i += 32) total += mine = weight_of<WINDOW>(p, i);
        for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
        total *= p.units;
        const int64_t per = share(p, total);
        at = blockIdx.x * per;
        end = at + per < total ? at + per : total;
        if (at >= end) return;
        for (int64_t b0 = 0; b0 < p.batch; b0 += 32) {
            if (p.batch > 32) mine = b0 + lane < p.batch ? weight_of<WINDOW>(p, b0 + lane) : 0;
            int64_t sum = mine;
            for (int d = 1; d < 32; d *= 2) {
                const int64_t o = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += o;
            }
            const unsigned past = __ballot_sync(0xffffffffu, (before + sum) * p.units > at);
            if (past) {
                const int l = __ffs(past) - 1;
                b = b0 + l;
                before += __shfl_sync(0xffffffffu, sum - mine, l);
                break;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
            b = p.batch;
        }
    }

    while (at < end && b < p.batch) {
        // the next part of one sequence, cache head and block of query heads: steps [from, to) of `steps`
        const int n = __ldcg(a.lengths + b), tiles = work_tiles<WINDOW>(p, n), steps = (tiles + PAIR - 1) / PAIR, weight = steps + START;
        if (!p.cluster && tiles == 0) {
            ++b;
            continue;
        }
        const int64_t start = before * p.units;
        const int unit = p.cluster ? (int)(item % p.units) : (int)((at - start) / weight);
        if (unit >= p.units) return;           // (lengths that change under the call)
        int from, to;
        if (p.cluster) {
            from = (int)((int64_t)steps * rank / p.cluster);
            to = (int)((int64_t)steps * (rank + 1) / p.cluster);
        } else {
            const int64_t in = at - start - (int64_t)unit * weight, out = in + (end - at);
            from = in > START ? (int)in - START : 0;
            to = out >= weight ? steps : out > START ? (int)out - START : 0;
            at += (out < weight ? out : weight) - in;
            if (to == steps && unit == p.units - 1) before += weight;
            if (to <= from) continue;          // (only of what the part's start counts for; the sequence goes on in the next share)
        }
        const int64_t seq = b;
        if (!p.cluster && to == steps && unit == p.units - 1) ++b;
        const int kh = unit / p.blocks, group = a.heads / a.kv_heads, h0 = (unit - kh * p.blocks) * p.cols;
        const int heads = group - h0 < p.cols ? group - h0 : p.cols;      // of this block
        const int64_t head0 = (int64_t)kh * group + h0;
        __syncthreads();

        // Where the warp's tiles lie: a lane looks up one tile of the next 32, a batch ahead of its use, and hands its first row of the cache around.
        bool bad = n > p.most_tiles * TILE;          // more than the table holds (pages are whole tiles)
        const Visible seen(p, n);                    // (not used without a window)
        const bool empty = WINDOW ? tiles == 0 && !bad : n <= 0;
        const int32_t *pages = a.table + seq * a.table_stride;
        constexpr int BATCH = 32 / PAIR;              // steps
        constexpr uint32_t NONE = 0xffffffffu, BAD = 0xfffffffeu;
        auto look_up = [&](int step0) {
            const int tile = (step0 + lane / PAIR * WARPS) * PAIR + lane % PAIR;
            uint32_t row = NONE;
            if (tile < to * PAIR && tile < tiles) {
                const int place = WINDOW ? seen.tile(tile) : tile, at_page = place / p.tiles_per_page;
                const uint32_t page = (uint32_t)__ldcg(pages + at_page);
                row = page < (uint32_t)a.pages ? page * (uint32_t)(a.kv_heads * a.page_size) + (uint32_t)(kh * a.page_size + (place - at_page * p.tiles_per_page) * TILE) : BAD;
            }
            return row;
        };
        uint32_t rows = look_up(from + warp), rows_ahead = look_up(from + warp + BATCH * WARPS);
        int looked = from + warp, in_batch = 0;       // first step of `rows`; steps of it that have been copied
        const uint8_t *k_at = reinterpret_cast<const uint8_t *>(a.k_codes) + lane * 16, *v_at = reinterpret_cast<const uint8_t *>(a.v_codes) + lane * 16,
                      *c_at = reinterpret_cast<const uint8_t *>(a.params) + lane * 16;
        auto copy_step = [&](uint32_t to_smem) {      // the next step into the ring
#pragma unroll
            for (int i = 0; i < PAIR; ++i) {
                const uint32_t row0 = __shfl_sync(0xffffffffu, rows, in_batch * PAIR + i);
                const bool ok = row0 < BAD;
                bad |= row0 == BAD;
                {
                    const uint8_t *k = k_at + (uint64_t)row0 * S::ROW, *v = v_at + (uint64_t)row0 * S::ROW;
                    const uint32_t t = to_smem + i * S::BYTES;
#pragma unroll
                    for (int j = 0; j < (S::ROW + 31) / 32; ++j) {
                        const int piece = lane + 32 * j, row = piece / S::PIECES;
                        const uint32_t o = t + row * S::ROW + ((piece % S::PIECES) ^ S::swizzle(row)) * 16;
                        copy16_if(ok && (S::ROW >= 32 || lane < 16), o, k + j * 512);
                        copy16_if(ok && (S::ROW >= 32 || lane < 16), o + 16 * S::ROW, v + j * 512);
                    }
                    copy16_if(ok && lane < 8, t + 32 * S::ROW + lane * 16, c_at + (uint64_t)row0 * 8);
                }
            }
            copies_commit();
            if (++in_batch == BATCH) {
                in_batch = 0;
                looked += BATCH * WARPS;
                rows = rows_ahead;
                rows_ahead = look_up(looked + BATCH * WARPS);
            }
        };
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) copy_step(ring + i * C::STEP);

        // the queries in fp16: as they are, or (bf16) times the power of two that takes their largest value to 2^14 and more, which the scores get back: elements down
        // to 2^-30 of it keep all their bits, and below that what is lost is less than 2^-39 of it
        for (int h = warp; h < HEADS; h += WARPS) {
            float v[DIM / 32], big = 0.0f, sum = 0.0f;
#pragma unroll
            for (int i = 0; i < DIM / 32; ++i) {
                v[i] = h < heads ? to_f32(__ldcg((const T *)a.q + seq * a.q_stride + (head0 + h) * a.q_head_stride + lane + 32 * i)) : 0.0f;
                big = fmaxf(big, fabsf(v[i]));
            }
            float back = 1.0f;
            if constexpr (__is_same(T, __nv_bfloat16)) {
                for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
                const int e = min(max((int)(__float_as_uint(big) >> 23), 16), 254);      // (a zero or infinite row: any power; infinities stay what they are)
                back = __uint_as_float((e - 14) << 23);
                const float by = __uint_as_float((268 - e) << 23);
#pragma unroll
                for (int i = 0; i < DIM / 32; ++i) v[i] *= by;
            }
#pragma unroll
            for (int i = 0; i < DIM / 32; ++i) {
                const __half q = __float2half_rn(v[i]);
                sq[h][lane + 32 * i] = q;
                sum += __half2float(q);
            }
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (lane == 0) {
                // scores in powers of two; of one visible token (whose weight is 1) zero: its value comes out exactly as read gives it
                s_factor[h] = (WINDOW ? seen.one(p, n) : n == 1) ? 0.0f : a.alpha * 1.4426950408889634f * back;
                s_sum[h] = sum;
            }
        }
        __syncthreads();
        uint32_t q[NB][S::MMAS][2];
        float f[NB][2], fsum[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const __half *row = sq[(nb * 8 + r) % HEADS] + c * (DIM / 4);
#pragma unroll
            for (int i = 0; i < S::KW; ++i)
#pragma unroll
                for (int pl = 0; pl < S::PLANES; ++pl) {
                    const __half *d = row + i * (32 / BITS) + pl;
                    q[nb][i * S::PLANES + pl][0] = as_u32(__halves2half2(d[0], d[16 / BITS]));
                    q[nb][i * S::PLANES + pl][1] = as_u32(__halves2half2(d[S::PLANES], d[S::PLANES + 16 / BITS]));
                }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                f[nb][j] = s_factor[(nb * 8 + 2 * c + j) % HEADS];
                fsum[nb][j] = f[nb][j] * s_sum[(nb * 8 + 2 * c + j) % HEADS];
            }
        }

        uint32_t magic;                                       // 1024 in both halves
        asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));
        float o[NB][S::MMAS][4] = {}, m[NB][2], l[NB][2] = {}, off[NB][2] = {};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) m[nb][0] = m[nb][1] = -INFINITY;
        const int half_tile = PAIR == 2 ? c / 2 : 0;         // the tile whose scores this lane's columns are
        int stage = 0, next = STAGES - 1;
#pragma unroll 1
        for (int now = from + warp; now < to; now += WARPS) {
            copies_wait<STAGES - 2>();
            __syncwarp();                                     // all lanes' copies are there, and all have used the stage that is filled next
            copy_step(ring + next * C::STEP);
            const uint32_t buf = ring + stage * C::STEP;
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            next = next + 1 == STAGES ? 0 : next + 1;

            // scores
            float acc[NB][S::PLANES][4];
#pragma unroll
            for (int i = 0; i < PAIR; ++i) {
                float sum[NB][S::PLANES][4] = {};
                uint32_t w[2][S::KW];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int row = r + 8 * j;
                    constexpr int WORDS = S::KW < 4 ? S::KW : 4;
#pragma unroll
                    for (int x = 0; x < S::KW; x += WORDS) {
                        const int byte = (c * S::KW + x) * 4;
                        load_words<WORDS>(buf + i * S::BYTES + row * S::ROW + (((byte / 16) ^ S::swizzle(row)) * 16 + byte % 16), w[j] + x);
                    }
                }
#pragma unroll
                for (int x = 0; x < S::KW; ++x) {
                    const uint32_t u0 = w[0][x] >> 8, u1 = w[1][x] >> 8;
#pragma unroll
                    for (int pl = 0; pl < S::PLANES; ++pl) {
                        const uint32_t bits = ((1u << BITS) - 1) * 0x00010001u << (pl * BITS);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
                            mma(sum[nb][pl], w[0][x] & bits, w[1][x] & bits, u0 & bits, u1 & bits, q[nb][x * S::PLANES + pl][0], q[nb][x * S::PLANES + pl][1]);
                    }
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int pl = 0; pl < S::PLANES; ++pl)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[nb][pl][e] = i == 0 || half_tile == 1 ? sum[nb][pl][e] : acc[nb][pl][e];
            }
            const int at_tile = now * PAIR + half_tile, t0 = (WINDOW ? seen.tile(at_tile) : at_tile) * TILE + r;
            float ks[2], kz[2], vs[2], vr[2];
            uint32_t vz[2];
            bool live[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t constants[2];
                load_words<2>(buf + half_tile * S::BYTES + 32 * S::ROW + (r + 8 * j) * 8, constants);
                const float2 kc = __half22float2(as_half2(constants[0]));
                live[j] = t0 + 8 * j < n && (PAIR == 1 || at_tile < tiles) && (!WINDOW || seen(p, t0 + 8 * j));      // rows that are not seen may hold anything
                ks[j] = kc.x;
                kz[j] = kc.y;
                const __half2 vc = as_half2(constants[1]);
                const __half2 z = __high2half2(vc), code = __hmin2(__hmax2(h2rint(z), __float2half2_rn(0.0f)), __float2half2_rn((float)((1 << BITS) - 1)));
                vs[j] = live[j] ? __low2float(vc) : 0.0f;
                vr[j] = live[j] ? __low2float(code) - __low2float(z) : 0.0f;
                vz[j] = live[j] ? as_u32(code) : 0u;
            }
            float u[NB][4];                           // [j * 2 + column]
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float dot = acc[nb][0][e];
#pragma unroll
                    for (int pl = 1; pl < S::PLANES; ++pl) dot = fmaf(acc[nb][pl][e], 1.0f / (1 << (pl * BITS)), dot);
                    u[nb][e] = ks[e / 2] * fmaf(dot, f[nb][e % 2] * 0x1p24f, -kz[e / 2] * fsum[nb][e % 2]);
                }
            float pv[NB][4], pw[NB][4];
            bool over = false;
            auto weights = [&]() {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        pw[nb][e] = live[e / 2] ? ex2(u[nb][e] - m[nb][e % 2]) : 0.0f;
                        pv[nb][e] = pw[nb][e] * vs[e / 2];
                        over |= pw[nb][e] > 0x1p40f || fabsf(pv[nb][e]) > 65000.0f;      // (scales may be negative)
                    }
            };
            weights();
            if (__any_sync(0xffffffffu, over)) {
                // the maximum moves: the largest p * scale of this step becomes 2^12 or more, by the power of two under the scale (scales are 2^-24 at least; of rows that are zero
                // p stays below 2^40)
                float lv[2];
#pragma unroll
                for (int row = 0; row < 2; ++row) lv[row] = (float)(max((int)(__float_as_uint(vs[row]) >> 23 & 255) - 127, -27) - 12);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float top = m[nb][j];
#pragma unroll
                        for (int row = 0; row < 2; ++row)
                            if (live[row]) top = fmaxf(top, u[nb][2 * row + j] + lv[row]);
                        for (int d = PAIR == 2 ? 2 : 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));      // (of a head's two columns as well)
                        const float keep = m[nb][j] == -INFINITY ? 0.0f : ex2(m[nb][j] - top);
                        m[nb][j] = top;
                        l[nb][j] *= keep;
                        off[nb][j] *= keep;
#pragma unroll
                        for (int i = 0; i < S::MMAS; ++i) {
                            o[nb][i][j] *= keep;
                            o[nb][i][2 + j] *= keep;
                        }
                    }
                weights();
            }
            uint32_t w[NB][2][2];                     // [j][weights, rests]
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l[nb][0] += pw[nb][2 * j];
                    l[nb][1] += pw[nb][2 * j + 1];
                    off[nb][0] = fmaf(pv[nb][2 * j], vr[j], off[nb][0]);
                    off[nb][1] = fmaf(pv[nb][2 * j + 1], vr[j], off[nb][1]);
                    const __half2 top = __floats2half2_rn(pv[nb][2 * j], pv[nb][2 * j + 1]);
                    const float2 t = __half22float2(top);
                    w[nb][j][0] = transpose8x8(as_u32(top));
                    w[nb][j][1] = transpose8x8(as_u32(__floats2half2_rn(pv[nb][2 * j] - t.x, pv[nb][2 * j + 1] - t.y)));
                    if constexpr (PAIR == 2) w[nb][j][1] = __shfl_xor_sync(0xffffffffu, w[nb][j][1], 16);      // to the head's other column
                }
            // Zero points of two tokens beside each other.  (The transposed matrix has every column of a row alike where a step is one tile; of two tiles
            // columns 0 to 3, now rows, have the first one's and 4 to 7 the second one's.)
            uint32_t zt[2] = {transpose8x8(vz[0]), transpose8x8(vz[1])};

            // values
#pragma unroll
            for (int i = 0; i < PAIR; ++i) {
                __half2 zero[S::PLANES][2];
                uint32_t b0[NB][3 - PAIR], b1[NB][3 - PAIR];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t z = zt[j];
                    if constexpr (PAIR == 2) z = __shfl_sync(0xffffffffu, z, c + 16 * i);
#pragma unroll
                    for (int pl = 0; pl < S::PLANES; ++pl) zero[pl][j] = __hfma2(as_half2(z), __float2half2_rn((float)(1 << (pl * BITS))), __float2half2_rn(1024.0f));
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int k = 0; k < 3 - PAIR; ++k) {
                        const int part = PAIR == 1 ? k : r / 4 != i;      // (of two tiles the columns of the other one's weights take this one's rests)
                        b0[nb][k] = part ? w[nb][0][1] : w[nb][0][0];
                        b1[nb][k] = part ? w[nb][1][1] : w[nb][1][0];
                    }
                const uint32_t values = buf + i * S::BYTES + 16 * S::ROW;
#pragma unroll
                for (int piece = 0; piece < S::PIECES; piece += 2) {
                    uint32_t x[4];                    // [piece][tokens 0 to 7, 8 to 15]
                    const int row = lane % 16;
                    if constexpr (S::PIECES == 1) load_transposed2(values + row * S::ROW, x);
                    else load_transposed4(values + row * S::ROW + ((piece + lane / 16) ^ S::swizzle(row)) * 16, x);
#pragma unroll
                    for (int h = 0; h < (S::PIECES == 1 ? 1 : 2); ++h) {
                        const uint32_t x0 = x[2 * h], x1 = x[2 * h + 1], y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
                        for (int pl = 0; pl < S::PLANES; ++pl) {
                            const uint32_t bits = ((1u << BITS) - 1) * 0x00010001u << (pl * BITS);
                            const uint32_t a0 = as_u32(__hsub2(as_half2(and_or(x0, bits, magic)), zero[pl][0]));
                            const uint32_t a1 = as_u32(__hsub2(as_half2(and_or(y0, bits, magic)), zero[pl][0]));
                            const uint32_t a2 = as_u32(__hsub2(as_half2(and_or(x1, bits, magic)), zero[pl][1]));
                            const uint32_t a3 = as_u32(__hsub2(as_half2(and_or(y1, bits, magic)), zero[pl][1]));
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                mma(o[nb][(piece + h) * S::PLANES + pl], a0, a1, a2, a3, b0[nb][0], b1[nb][0]);
                                if constexpr (PAIR == 1) mma(o[nb][(piece + h) * S::PLANES + pl], a0, a1, a2, a3, b0[nb][2 - PAIR], b1[nb][2 - PAIR]);
                            }
                        }
                    }
                }
            }
        }

        // the warps' parts become one
        copies_wait<0>();
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                for (int d = 4; d < 32; d *= 2) {
                    l[nb][j] += __shfl_xor_sync(0xffffffffu, l[nb][j], d);
                    off[nb][j] += __shfl_xor_sync(0xffffffffu, off[nb][j], d);
                }
                if (r == 0) {
                    s_m[warp][nb * 8 + 2 * c + j] = m[nb][j];
                    s_l[warp][nb * 8 + 2 * c + j] = bad ? NAN : l[nb][j];
                }
            }
        __syncthreads();
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int col = nb * 8 + 2 * c + j;
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < WARPS * PAIR; ++i) top = fmaxf(top, s_m[i / PAIR][PAIR == 2 ? col % 4 + i % 2 * 4 : col]);
                const float by = m[nb][j] == -INFINITY ? 0.0f : ex2(m[nb][j] - top);
#pragma unroll
                for (int i = 0; i < S::MMAS; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int pl = i % S::PLANES, d = (i / S::PLANES * 8 + r) * (16 / BITS) + pl + k * S::PLANES;
                        s_o[(warp * COLS + col) * S::STRIDE + d] = fmaf(o[nb][i][2 * k + j], by / (1 << (pl * BITS)), off[nb][j] * by);
                    }
            }
        if (threadIdx.x < heads) {
            const int col = threadIdx.x;
            float total = 0.0f, top = -INFINITY;
#pragma unroll
            for (int k = 0; k < WARPS * PAIR; ++k) top = fmaxf(top, s_m[k / PAIR][col + k % PAIR * 4]);
#pragma unroll
            for (int k = 0; k < WARPS * PAIR; ++k) total += part_of(s_m[k / PAIR][col + k % PAIR * 4], s_l[k / PAIR][col + k % PAIR * 4], top);
            s_total[col] = make_float2(top, total);
        }
        __syncthreads();
        auto sum_of = [&](int col, int d) {
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < WARPS * PAIR; ++k) sum += s_o[(k / PAIR * COLS + col + k % PAIR * 4) * S::STRIDE + d];
            return sum;
        };
        if (p.cluster > 1) {
            // the CTAs' parts become one: each CTA adds up its own first, then takes its share of the values from all
            cg::cluster_group cluster = cg::this_cluster();
            for (int i = threadIdx.x; i < heads * DIM; i += 32 * WARPS) s_o[i / DIM * S::STRIDE + i % DIM] = sum_of(i / DIM, i % DIM);
            cluster.sync();
            for (int i = rank * 32 * WARPS + threadIdx.x; i < heads * DIM; i += p.cluster * 32 * WARPS) {
                const int col = i / DIM, d = i % DIM;
                float top = -INFINITY, sum = 0.0f, total = 0.0f;
                for (int k = 0; k < p.cluster; ++k) top = fmaxf(top, cluster.map_shared_rank(s_total, k)[col].x);
                for (int k = 0; k < p.cluster; ++k) {
                    const float2 t = cluster.map_shared_rank(s_total, k)[col];
                    total += part_of(t.x, t.y, top);
                    sum += t.x == -INFINITY ? 0.0f : cluster.map_shared_rank(s_o, k)[col * S::STRIDE + d] * ex2(t.x - top);
                }
                ((T *)a.out)[(seq * a.heads + head0) * DIM + i] = from_f32<T>(empty ? 0.0f : sum / total);
            }
            cluster.sync();
            return;
        }
        const bool whole = from == 0 && to == steps;
        float *slot = p.slots + (int64_t)(2 * blockIdx.x + (from == 0)) * p.cols * (DIM + 2);
        for (int i = threadIdx.x; i < heads * DIM; i += 32 * WARPS) {
            const int col = i / DIM, d = i % DIM;
            const float sum = sum_of(col, d);
            if (whole) ((T *)a.out)[(seq * a.heads + head0) * DIM + i] = from_f32<T>(empty ? 0.0f : sum / s_total[col].y);
            else {
                slot[i] = sum;
                if (d == 0) *reinterpret_cast<float2 *>(slot + p.cols * DIM + 2 * col) = s_total[col];
            }
        }
        if (p.cluster) return;
    }
}

// One CTA a head of a sequence: zeros for an empty sequence, and the parts of one that several CTAs share.
template <typename T, int DIM, bool WINDOW>
__global__ void __launch_bounds__(128) kv_attend_join_kernel(const FastArgs p) {
    const AttendArgs &a = p.a;
    const int64_t b = blockIdx.x / a.heads;
    const int h = (int)(blockIdx.x - b * a.heads), group = a.heads / a.kv_heads, kh = h / group, block = (h - kh * group) / p.cols,
              col = h - kh * group - block * p.cols, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    T *out = (T *)a.out + (int64_t)blockIdx.x * DIM;
    // (the lengths were there when the launch before this one began its work, which then is all that is waited for)
    const int n = __ldcg(a.lengths + b), weight = weight_of<WINDOW>(p, b);
    int64_t total = 0, before = 0;
    for (int64_t i = lane; i < p.batch; i += 32) {
        const int w = weight_of<WINDOW>(p, i);
        total += w;
        before += i < b ? w : 0;
    }
    for (int d = 16; d; d >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, d);
        before += __shfl_xor_sync(0xffffffffu, before, d);
    }
    const int64_t per = share(p, total * p.units), from = before * p.units + (int64_t)(kh * p.blocks + block) * weight + START;
    const int first = (int)(from / per), last = (int)((from + weight - START - 1) / per), parts = last - first + 1;
    pdl_wait();
    if (weight == 0) {
        for (int d = threadIdx.x; d < DIM; d += 128) out[d] = from_f32<T>((WINDOW ? n > p.most_tiles * TILE : n > 0) ? NAN : 0.0f);
        return;
    }
    if (parts == 1) return;
    const int64_t size = (int64_t)p.cols * (DIM + 2);             // of a slot; the first CTA's part is in its second one, the others' in their first
    auto slot = [&](int i) { return p.slots + (2 * (int64_t)(first + i) + (i == 0)) * size; };
    __shared__ float s_f[MOST_CTAS], s_l[MOST_CTAS], s_part[4], s_o[4][DIM];
    // A warp takes every fourth part; the first of them are asked for before their factors are known.
    constexpr int V = DIM / 32, AHEAD = 32 / V;
    float ahead[AHEAD][V];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (warp + 4 * i < parts) {
            const float *from = slot(warp + 4 * i) + (int64_t)col * DIM + lane;
#pragma unroll
            for (int k = 0; k < V; ++k) ahead[i][k] = __ldcg(from + 32 * k);
        }
    // factors of the parts: 2^(m - largest m)
    float top = -INFINITY;
    for (int i = threadIdx.x; i < parts; i += 128) {
        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(slot(i) + p.cols * DIM + 2 * col));
        s_f[i] = ml.x;
        s_l[i] = ml.y;
        top = fmaxf(top, ml.x);
    }
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (lane == 0) s_part[warp] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_part[0], s_part[1]), fmaxf(s_part[2], s_part[3]));
    float l = 0.0f;
    for (int i = threadIdx.x; i < parts; i += 128) {
        const float f = s_f[i] == -INFINITY ? 0.0f : ex2(s_f[i] - top), sum = s_l[i];
        s_f[i] = f;
        l += sum == sum ? f * sum : NAN;
    }
    for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    __syncthreads();
    if (lane == 0) s_part[warp] = l;
    float o[V] = {};
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (warp + 4 * i < parts) {
#pragma unroll
            for (int k = 0; k < V; ++k) o[k] += s_f[warp + 4 * i] * ahead[i][k];
        }
#pragma unroll 4
    for (int i = warp + 4 * AHEAD; i < parts; i += 4) {
        const float f = s_f[i], *from = slot(i) + (int64_t)col * DIM + lane;
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] += f * __ldcg(from + 32 * k);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) s_o[warp][lane + 32 * k] = o[k];
    __syncthreads();
    for (int d = threadIdx.x; d < DIM; d += 128)
        out[d] = from_f32<T>((s_o[0][d] + s_o[1][d] + s_o[2][d] + s_o[3][d]) / (s_part[0] + s_part[1] + s_part[2] + s_part[3]));
}

// CTAs of a cluster that takes a unit of a window of `steps`; 0: the line of work.  A window's sequences are alike, so that CTAs need no equal shares, and without a join one CTA a unit is
// as fast as the chip goes from some hundred units on.  Times in steps of a warp (0.75 us of 32 tokens of 128 values): a part's own, two more for a cluster's join; or what
// the chip needs for all, each CTA's start and end counting 13 steps, and a third of what its last wave leaves idle; the line's parts and join count 30.  Measured, 4 bits, line / 1 / 2 / 4 / 8 CTAs:
// 64 units of 17 steps 10.7 / 8.2 / 8.9 / 8.1 / 8.6 us, 64 of 129 17.7 / 29.1 / 19.1 / 15.2 / 15.8, 512 of 17 25.7 / 15.2 / 23.0 / 34.6 / 58.3, 1536 of 129 205 / 172 / 181 / 216 / 290; 8 bits, 512 of 129 97 / 121 /
// 113 / 110 / 150.
int window_cluster(int64_t units, int64_t steps, int dim, int cols, int pair, int bits) {
    const double slots = 148 * (dim == 256 ? 2 : cols == 16 ? (dim == 64 ? 3 : 2) : bits == 8 && dim == 128 ? 3 : 4);
    const double rate = 600.0 * 128 / dim * (pair == 2 ? 1 : 2) * (bits == 8 ? 1.0 : 1.6);      // steps of all SMs in a warp's
    double best = std::max(12.0, units * (steps + 30) / rate);
    int found = 0;
    for (int c = 1; c <= 8 && (c == 1 || steps > c / 2 * WARPS); c *= 2) {
        const double waves = units * c / slots, idle = waves > 1 ? (std::ceil(waves) / waves - 1) / 3 : 0;
        const double own = (double)((steps + WARPS * c - 1) / (WARPS * c)) + (c > 1 ? 2 : 0), all = units * (13 * c + steps) / rate * (1 + idle);
        if (std::max(own, all) < best) {
            best = std::max(own, all);
            found = c;
        }
    }
    return found;
}

// Whether the tiled kernel takes this cache, and how it divides a call.
// `window`, `sinks`: INT32_MAX and 0 where everything is seen.  (Without a window `bits` does not matter.)
bool fast_args(FastArgs &p, int64_t batch, int heads, int kv_heads, int dim, int bits, int64_t pages, int page_size, int64_t max_pages, int64_t window, int64_t sinks) {
    // (rows of the cache are numbered in 32 bits)
    if ((dim != 64 && dim != 128 && dim != 256) || page_size % TILE != 0 || pages * kv_heads * page_size >= 0xfffffffell) return false;
    const int group = heads / kv_heads;
    p.batch = batch;
    p.cols = group > 8 && dim < 256 ? 16 : 8;
    p.blocks = (group + p.cols - 1) / p.cols;
    p.units = kv_heads * p.blocks;
    p.tiles_per_page = page_size / TILE;
    p.most_tiles = (int)(max_pages * p.tiles_per_page);
    p.pair = group <= 4 && dim < 256 ? 2 : 1;      // (of 256 values of 8 bits two tiles would be 16 KB a step)
    // Clusters, where one wave of them (of 444 CTAs: three an SM) goes through the longest table in CLUSTER_ROUNDS steps a warp.  8 cache heads of 128, 4 bits:
    // 4 sequences of 1000 tokens 8.0 us, in shares with a join 10.3; 16 of 600 10.9 / 13.9; 16 of up to 2048 (5.3 steps) 16.8 / 15.8: the longest is waited for.
    // (with a window: through the tiles that it and the sinks can lie on)
    int64_t tiles = p.most_tiles;
    if (window < INT32_MAX) tiles = std::min(tiles, (sinks + TILE - 1) / TILE + (window ? (window + TILE - 2) / TILE + 1 : 0));
    const int64_t items = batch * p.units, steps = (tiles + p.pair - 1) / p.pair, wide = 444 / (items < 444 ? items : 444);
    int64_t size = (steps + 2 * WARPS - 1) / (2 * WARPS);            // (a part of less than two steps a warp is not worth a CTA)
    if (size > wide) size = wide;
    size = size > 8 ? 8 : size < 1 ? 1 : size;
    p.cluster = steps <= size * WARPS * (size > 1 ? CLUSTER_ROUNDS : 2) ? (int)size : 0;
    // (a long window of more than half of the longest sequence meets lengths as ragged as attention without one does)
    if (window < INT32_MAX && (steps <= 64 || 2 * tiles <= p.most_tiles)) p.cluster = window_cluster(items, steps, dim, p.cols, p.pair, bits);
    return batch * p.units < (int64_t)1 << 28;
}

template <typename T, int BITS, int DIM, int NB, int PAIR, bool WINDOW>
int launch_fast(FastArgs &p, cudaStream_t st) {
    auto kern = kv_attend_kernel<T, BITS, DIM, NB, PAIR, WINDOW>;
    constexpr int SMEM = Config<T, BITS, DIM, NB, PAIR>::SMEM;
    static std::atomic<int> per_sm[64];                     // by device
    int device = 0;
    BW_CUDA_TRY(cudaGetDevice(&device));
    int n = device < 64 ? per_sm[device].load() : 0;
    if (!n) {
        BW_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        BW_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, 32 * WARPS, SMEM));
        n = n < 1 ? 1 : n > 4 ? 4 : n;
        if (device < 64) per_sm[device] = n;
    }
    p.ctas = 148 * n;
    if (p.cluster) return launch_early("kv_attend_kernel", kern, dim3((unsigned)(p.batch * p.units * p.cluster)), 32 * WARPS, SMEM, st, dim3(p.cluster), p);
    const int rc = launch_early("kv_attend_kernel", kern, dim3((unsigned)p.ctas), 32 * WARPS, SMEM, st, dim3(1), p);
    if (rc != BW_OK) return rc;
    return launch_early("kv_attend_join_kernel", kv_attend_join_kernel<T, DIM, WINDOW>, dim3((unsigned)(p.batch * p.a.heads)), 128, 0, st, dim3(1), p);
}

template <typename T, int BITS, int DIM, bool WINDOW>
int launch_group(FastArgs &p, cudaStream_t st) {
    if constexpr (DIM < 256) {
        if (p.cols == 16) return launch_fast<T, BITS, DIM, 2, 1, WINDOW>(p, st);
        if (p.pair == 2) return launch_fast<T, BITS, DIM, 1, 2, WINDOW>(p, st);
    }
    return launch_fast<T, BITS, DIM, 1, 1, WINDOW>(p, st);
}
template <typename T, int BITS, bool WINDOW>
int launch_dim(FastArgs &p, cudaStream_t st) {
    if (p.a.dim == 64) return launch_group<T, BITS, 64, WINDOW>(p, st);
    if (p.a.dim == 128) return launch_group<T, BITS, 128, WINDOW>(p, st);
    return launch_group<T, BITS, 256, WINDOW>(p, st);
}
template <bool WINDOW, typename T>
int launch_bits(FastArgs &p, int bits, cudaStream_t st) {
    return bits == 2 ? launch_dim<T, 2, WINDOW>(p, st) : bits == 4 ? launch_dim<T, 4, WINDOW>(p, st) : launch_dim<T, 8, WINDOW>(p, st);
}

}  // namespace
}  // namespace bw
