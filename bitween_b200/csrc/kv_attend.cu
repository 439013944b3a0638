// Attention of one new token per sequence over the paged, quantised key-value cache (bw_kv_attend).
//
//     out[b][h] = sum_t w_t V[t],   w = softmax over t < lengths[b] of  alpha * q[b][h] . K[t],   K, V rows of head h / (heads / kv_heads)
//
// One pass over the cache with the running maximum and sum of the softmax; codes become values in registers.
#include "bw_common.cuh"

namespace bw {
namespace {

struct AttendArgs {
    const void *q;
    const int32_t *k_codes, *v_codes;
    const __half2 *params;                     // [row][2]: (scale, zero) of the key, of the value
    const int32_t *table, *lengths;
    void *out;
    int64_t q_stride, q_head_stride, table_stride, pages;
    int heads, kv_heads, dim, words, page_size, max_pages;
    float alpha;
};

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
    for (int64_t t = warp; t < len; t += 4) {
        const int64_t in = t / p.page_size, page = p.table[b * p.table_stride + in];
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
        ((T *)p.out)[(b * p.heads + h) * p.dim + d] = from_f32<T>(n <= 0 ? 0.0f : v / sum);
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


// ---- head dimensions of 64, 128 and 256, pages of whole tiles of 16 tokens --------------------------------------------
//
// A warp takes tiles of 16 tokens; K and V codes are the A operand of mma.sync.m16n8k16 (16 tokens, then 16 values, by 8 heads of the
// group), so that one read of the cache serves all heads that share it:
//   scores   S[t][h] = scale_t * (sum_d code[t][d] q[h][d] - zero_t * sum_d q[h][d]).  A code, masked out of its word, IS an fp16 number:
//            the subnormal code * 2^-24 (tensor cores take subnormals exactly), so expanding two codes costs one AND.  Codes that stand in
//            higher bits of their byte (`planes`) are larger by a power of two and get accumulators of their own.  Scale and zero point
//            are applied to the sums, in fp32: nothing is rounded.
//   weights  p = 2^(x - m); p * (value's scale) goes to fp16 for the second product.  m covers p * scale, so that this stays in fp16's
//            range whatever the scales are; it moves only when some p * scale leaves [0, 1024] (one vote a tile).  For fp16 results the
//            rest p - fp16(p) is a second operand, in the unused columns of groups of up to 4 heads or by second MMAs: one rounding
//            of 2^-11 less in the result.  For bf16 results that rounding is an eighth of the result's own.
//   values   O[d][h] += (code - zero_t)[d][t] * p[t][h]: 1024 + code by one OR, minus (1024 + zero), exact.  Codes of two tokens are put
//            beside each other by one byte permutation a word.
//
// Work: all tiles of all sequences and heads in one line, an equal share of it to each CTA, whatever the lengths are.  What
// a share has of a sequence that others have too goes to scratch (running maximum, sum, unnormalised output), and
// kv_attend_join_kernel joins it.  Tables of few tiles go without: one CTA a sequence and head.
constexpr int WARPS = 4, TILE = 16;
constexpr int MOST_CTAS = 592;              // shares of a call: four CTAs on each of 148 SMs
constexpr int SINGLE_TILES = 16;            // tables of up to so many tiles (256 tokens): one CTA, four tiles a warp

struct FastArgs {
    AttendArgs a;
    int64_t batch;
    float *slots;                           // [2 * MOST_CTAS][cols][dim + 2]
    int units;                              // of a sequence: cache heads x blocks of query heads
    int blocks, cols;                       // blocks of query heads of a cache head; heads of a block
    int ctas, most_tiles, tiles_per_page;
    bool single;
};

__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
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

template <int BYTES> __device__ __forceinline__ void load_bytes(const uint8_t *p, uint32_t *w) {
    if constexpr (BYTES == 2) w[0] = __ldg(reinterpret_cast<const unsigned short *>(p));
    else if constexpr (BYTES == 4) w[0] = __ldg(reinterpret_cast<const uint32_t *>(p));
    else if constexpr (BYTES == 8) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
        w[0] = v.x; w[1] = v.y;
    } else {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    }
}

// Tiles of a sequence within its table; its true length goes beside it.
__device__ __forceinline__ int tiles_of(int n, int most) {
    const int t = n > 0 ? (n - 1) / TILE + 1 : 0;
    return t < most ? t : most;
}

// Tiles of all sequences together (every warp by itself: a step of 32 sequences).
__device__ __forceinline__ int64_t tiles_of_all(const FastArgs &p) {
    const int lane = threadIdx.x % 32;
    int64_t sum = 0;
    for (int64_t b = lane; b < p.batch; b += 32) sum += tiles_of(__ldcg(p.a.lengths + b), p.most_tiles);
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return sum;
}

// The tiles of one CTA's share.  Shares of less than two tiles a warp are not worth another CTA.
__device__ __forceinline__ int64_t share(const FastArgs &p, int64_t total) {
    const int64_t even = (total + p.ctas - 1) / p.ctas;
    return even < 2 * WARPS ? 2 * WARPS : even;
}

template <int BITS, int DIM> struct Shape {
    static constexpr int PLANES = 8 / BITS;                 // places of a code in a byte
    static constexpr int KW = DIM * BITS / 128;             // words of a key row that a lane holds (of two rows)
    static constexpr int VH = DIM * BITS / 128;             // 16-bit halves of a value row that a lane holds (of four rows)
    static constexpr int VW = (VH + 1) / 2;
    static constexpr int KMMAS = KW * PLANES, VMMAS = VH * PLANES;   // DIM / 16 each
    static constexpr uint32_t MASK = ((1u << BITS) - 1) * 0x00010001u;
    static constexpr bool AHEAD = KW <= 4;                  // the next tile is loaded before the present one is used: else registers run out
    static constexpr int STRIDE = DIM + DIM / 16 + (36 - (DIM + DIM / 16) % 32) % 32;   // of a head's sums in shared memory: 4 mod 32, values padded by one in 16
    // Byte of a lane's word i of a key row (quarter c), and of a value row (eighth r): 16-byte pieces side by side.
    static __device__ __forceinline__ int key_byte(int i, int c) { return KW <= 4 ? (c * KW + i) * 4 : (i / 4) * 64 + c * 16 + (i % 4) * 4; }
    static __device__ __forceinline__ int value_byte(int half, int r) { return VH <= 8 ? (r * VH + half) * 2 : (half / 8) * 128 + r * 16 + (half % 8) * 2; }
};

template <int BITS, int DIM>
struct Tile {
    using S = Shape<BITS, DIM>;
    uint32_t k[2][S::KW], v[4][S::VW];
    uint2 c[2];                             // constants of the lane's two key rows: (scale, zero) of key and value
};

template <int BITS, int DIM>
__device__ __forceinline__ void load_keys(Tile<BITS, DIM> &t, const AttendArgs &a, int64_t row0, int r, int c) {
    using S = Shape<BITS, DIM>;
    constexpr int BYTES = S::KW >= 4 ? 16 : S::KW * 4;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t row = row0 + (r >> 1) + 4 * (r & 1) + 8 * j;
        const uint8_t *p = reinterpret_cast<const uint8_t *>(a.k_codes) + row * (DIM * BITS / 8);
#pragma unroll
        for (int i = 0; i < S::KW; i += BYTES / 4) load_bytes<BYTES>(p + S::key_byte(i, c), t.k[j] + i);
        t.c[j] = __ldg(reinterpret_cast<const uint2 *>(a.params) + row);
    }
}
template <int BITS, int DIM>
__device__ __forceinline__ void load_values(Tile<BITS, DIM> &t, const AttendArgs &a, int64_t row0, int r, int c) {
    using S = Shape<BITS, DIM>;
    constexpr int BYTES = S::VH >= 8 ? 16 : S::VH * 2;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint8_t *p = reinterpret_cast<const uint8_t *>(a.v_codes) + (row0 + c + 4 * j) * (DIM * BITS / 8);
#pragma unroll
        for (int h = 0; h < S::VH; h += BYTES / 2) load_bytes<BYTES>(p + S::value_byte(h, r), t.v[j] + h / 2);
    }
}

// REST: how the rests of the weights' rounding enter.  0: not (bf16 results); 1: columns 4 to 7 repeat columns 0 to 3 and carry the rests
// (groups of up to 4); 2: MMAs of their own.
template <typename T, int BITS, int DIM, int NB, int REST>
__global__ void __launch_bounds__(32 * WARPS) kv_attend_kernel(const FastArgs p) {
    using S = Shape<BITS, DIM>;
    constexpr int COLS = 8 * NB;
    const AttendArgs &a = p.a;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
    __shared__ __align__(16) __half sq[COLS][DIM + 8];
    __shared__ float s_factor[COLS], s_sum[COLS], s_m[WARPS][COLS], s_l[WARPS][COLS];
    __shared__ __align__(16) float s_o[WARPS][COLS * S::STRIDE];
    pdl_launch_dependents();

    // this CTA's share of the line of tiles, and the sequence in which it starts
    int64_t at, end, b = 0, before = 0;      // `before`: tiles in front of sequence b
    if (p.single) {
        b = blockIdx.x / p.units;
        at = 0;
        end = INT64_MAX;
    } else {
        const int64_t total = tiles_of_all(p) * p.units, per = share(p, total);
        at = blockIdx.x * per;
        end = at + per < total ? at + per : total;
        if (at >= end) return;
        for (int64_t b0 = 0; b0 < p.batch; b0 += 32) {
            const int mine = b0 + lane < p.batch ? tiles_of(__ldcg(a.lengths + b0 + lane), p.most_tiles) : 0;
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
        // the next part of one sequence, cache head and block of query heads: tiles [from, to) of `tiles`
        const int n = __ldcg(a.lengths + b), tiles = tiles_of(n, p.most_tiles);
        if (!p.single && tiles == 0) {
            ++b;
            continue;
        }
        const int64_t start = before * p.units;
        const int unit = p.single ? (int)(blockIdx.x % p.units) : (int)((at - start) / tiles);
        const int from = p.single ? 0 : (int)(at - start - (int64_t)unit * tiles);
        const int to = p.single || end - at > tiles - from ? tiles : from + (int)(end - at);
        if (unit >= p.units) return;           // (lengths that change under the call)
        const int kh = unit / p.blocks, group = a.heads / a.kv_heads, h0 = (unit - kh * p.blocks) * p.cols;
        const int heads = group - h0 < p.cols ? group - h0 : p.cols;      // of this block
        const int64_t out0 = (b * a.heads + (int64_t)kh * group + h0) * DIM;

        // the queries in fp16: as they are, or (bf16) divided by a power of two near their largest value, which the scores get back
        __syncthreads();
        for (int h = warp; h < COLS; h += WARPS) {
            const int head = REST == 1 ? h % 4 : h;
            float v[DIM / 32], big = 0.0f, sum = 0.0f;
#pragma unroll
            for (int i = 0; i < DIM / 32; ++i) {
                v[i] = head < heads ? to_f32(((const T *)a.q)[b * a.q_stride + (int64_t)(kh * group + h0 + head) * a.q_head_stride + lane + 32 * i]) : 0.0f;
                big = fmaxf(big, fabsf(v[i]));
            }
            float back = 1.0f;
            if constexpr (__is_same(T, __nv_bfloat16)) {
                for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
                const int e = min(max((int)(__float_as_uint(big) >> 23), 2), 252);       // (a zero or infinite row: any power; infinities stay what they are)
                back = __uint_as_float(e << 23);
                const float by = __uint_as_float((254 - e) << 23);
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
                s_factor[h] = a.alpha * 1.4426950408889634f * back;       // scores in powers of two
                s_sum[h] = sum;
            }
        }
        __syncthreads();
        uint32_t q[NB][S::KMMAS][2];
        float f[NB][2], fsum[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const __half *row = sq[nb * 8 + r];
#pragma unroll
            for (int i = 0; i < S::KW; ++i) {
                const int d0 = S::key_byte(i, c) * 8 / BITS;
#pragma unroll
                for (int pl = 0; pl < S::PLANES; ++pl) {
                    const int d = d0 + pl;
                    q[nb][i * S::PLANES + pl][0] = as_u32(__halves2half2(row[d], row[d + 16 / BITS]));
                    q[nb][i * S::PLANES + pl][1] = as_u32(__halves2half2(row[d + S::PLANES], row[d + S::PLANES + 16 / BITS]));
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                f[nb][j] = s_factor[nb * 8 + 2 * c + j];
                fsum[nb][j] = f[nb][j] * s_sum[nb * 8 + 2 * c + j];
            }
        }

        float o[NB][S::VMMAS][4] = {}, m[NB][2], l[NB][2] = {};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) m[nb][0] = m[nb][1] = -INFINITY;
        bool bad = n > p.most_tiles * TILE;          // more than the table holds (pages are whole tiles)

        // pages: the tile's place in its page goes forward with the tiles
        int tile = from + warp, page_at = tile / p.tiles_per_page, in = tile - page_at * p.tiles_per_page;
        const int step_pages = WARPS / p.tiles_per_page, step_in = WARPS - step_pages * p.tiles_per_page;
        const int32_t *pages = a.table + b * a.table_stride;
        int page = tile < to ? __ldg(pages + page_at) : 0, place = in;
        auto forward = [&](int next) {               // `page` and `place` of tile `next`
            page_at += step_pages;
            in += step_in;
            if (in >= p.tiles_per_page) {
                in -= p.tiles_per_page;
                ++page_at;
            }
            if (next < to) page = __ldg(pages + page_at);
            place = in;
        };
        Tile<BITS, DIM> cur = {}, ahead = {};
        auto row_of = [&]() { return ((int64_t)page * a.kv_heads + kh) * a.page_size + place * TILE; };
        auto valid = [&]() { return page >= 0 && page < a.pages; };
        if (S::AHEAD && tile < to) {
            if (valid()) {
                load_keys(cur, a, row_of(), r, c);
                load_values(cur, a, row_of(), r, c);
            } else bad = true;
            forward(tile + WARPS);
        }
#pragma unroll 2
        for (; tile < to; tile += WARPS) {
            if constexpr (S::AHEAD) {
                if (tile + WARPS < to) {
                    if (valid()) {
                        load_keys(ahead, a, row_of(), r, c);
                        load_values(ahead, a, row_of(), r, c);
                    } else bad = true;
                    forward(tile + 2 * WARPS);
                }
            } else {
                if (valid()) {
                    load_keys(cur, a, row_of(), r, c);
                    load_values(cur, a, row_of(), r, c);
                } else bad = true;
                forward(tile + WARPS);
            }

            // scores
            float acc[NB][S::PLANES][4] = {};
#pragma unroll
            for (int i = 0; i < S::KW; ++i) {
                const uint32_t w0 = cur.k[0][i], w1 = cur.k[1][i], u0 = w0 >> 8, u1 = w1 >> 8;
#pragma unroll
                for (int pl = 0; pl < S::PLANES; ++pl) {
                    constexpr uint32_t MASK = S::MASK;
                    const uint32_t bits = MASK << (pl * BITS);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
                        mma(acc[nb][pl], w0 & bits, w1 & bits, u0 & bits, u1 & bits, q[nb][i * S::PLANES + pl][0], q[nb][i * S::PLANES + pl][1]);
                }
            }
            const int t0 = tile * TILE + (r >> 1) + 4 * (r & 1);
            float ks[2], kz[2], vs[2];
            uint32_t vz[2];
            bool live[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 kc = __half22float2(as_half2(cur.c[j].x));
                live[j] = t0 + 8 * j < n;             // rows behind the sequence may hold anything
                ks[j] = kc.x;
                kz[j] = kc.y;
                const __half2 vc = as_half2(cur.c[j].y);
                vs[j] = live[j] ? __low2float(vc) : 0.0f;
                vz[j] = live[j] ? as_u32(__high2half2(vc)) : 0u;
            }
            float u[NB][4];                           // [j * 2 + column]
            uint32_t w[NB][2][2];                     // [j][weights, rests]
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float dot = acc[nb][0][e] * 0x1p24f;
#pragma unroll
                    for (int pl = 1; pl < S::PLANES; ++pl) dot = fmaf(acc[nb][pl][e], 0x1p24f / (1 << (pl * BITS)), dot);
                    u[nb][e] = ks[e / 2] * fmaf(dot, f[nb][e % 2], -kz[e / 2] * fsum[nb][e % 2]);
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
                        over |= pw[nb][e] > 0x1p40f || pv[nb][e] > 1024.0f;
                    }
            };
            weights();
            if (__any_sync(0xffffffffu, over)) {
                // the maximum moves: the largest of this tile's p and p * scale becomes at most 1
                const float lv[2] = {fmaxf(__log2f(vs[0]), -40.0f), fmaxf(__log2f(vs[1]), -40.0f)};
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float top = m[nb][j];
#pragma unroll
                        for (int row = 0; row < 2; ++row)
                            if (live[row]) top = fmaxf(top, u[nb][2 * row + j] + lv[row]);
                        for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        const float keep = m[nb][j] == -INFINITY ? 0.0f : ex2(m[nb][j] - top);
                        m[nb][j] = top;
                        l[nb][j] *= keep;
#pragma unroll
                        for (int i = 0; i < S::VMMAS; ++i) {
                            o[nb][i][j] *= keep;
                            o[nb][i][2 + j] *= keep;
                        }
                    }
                weights();
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l[nb][0] += pw[nb][2 * j];
                    l[nb][1] += pw[nb][2 * j + 1];
                    const __half2 top = __floats2half2_rn(pv[nb][2 * j], pv[nb][2 * j + 1]);
                    w[nb][j][0] = as_u32(top);
                    if constexpr (REST != 0) {
                        const float2 t = __half22float2(top);
                        const uint32_t rest = as_u32(__floats2half2_rn(pv[nb][2 * j] - t.x, pv[nb][2 * j + 1] - t.y));
                        if constexpr (REST == 1) w[nb][j][0] = c >= 2 ? rest : w[nb][j][0];
                        else w[nb][j][1] = transpose8x8(rest);
                    }
                    w[nb][j][0] = transpose8x8(w[nb][j][0]);
                }

            // values
            __half2 zero[S::PLANES][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const __half2 z = as_half2(transpose8x8(vz[j]));
#pragma unroll
                for (int pl = 0; pl < S::PLANES; ++pl) zero[pl][j] = __hfma2(z, __float2half2_rn((float)(1 << (pl * BITS))), __float2half2_rn(1024.0f));
            }
#pragma unroll
            for (int h = 0; h < S::VH; ++h) {
                const uint32_t sel = h % 2 ? 0x7632 : 0x5410;
                const uint32_t x0 = __byte_perm(cur.v[0][h / 2], cur.v[1][h / 2], sel), x1 = __byte_perm(cur.v[2][h / 2], cur.v[3][h / 2], sel);
                const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
                for (int pl = 0; pl < S::PLANES; ++pl) {
                    constexpr uint32_t MASK = S::MASK;
                    const uint32_t bits = MASK << (pl * BITS);
                    const uint32_t a0 = as_u32(__hsub2(as_half2((x0 & bits) | 0x64006400u), zero[pl][0]));
                    const uint32_t a1 = as_u32(__hsub2(as_half2((y0 & bits) | 0x64006400u), zero[pl][0]));
                    const uint32_t a2 = as_u32(__hsub2(as_half2((x1 & bits) | 0x64006400u), zero[pl][1]));
                    const uint32_t a3 = as_u32(__hsub2(as_half2((y1 & bits) | 0x64006400u), zero[pl][1]));
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        mma(o[nb][h * S::PLANES + pl], a0, a1, a2, a3, w[nb][0][0], w[nb][1][0]);
                        if constexpr (REST == 2) mma(o[nb][h * S::PLANES + pl], a0, a1, a2, a3, w[nb][0][1], w[nb][1][1]);
                    }
                }
            }
            if constexpr (S::AHEAD) cur = ahead;
        }

        // the four warps' parts become one
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                for (int d = 4; d < 32; d *= 2) l[nb][j] += __shfl_xor_sync(0xffffffffu, l[nb][j], d);
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
                float top = s_m[0][col];
#pragma unroll
                for (int w2 = 1; w2 < WARPS; ++w2) top = fmaxf(top, s_m[w2][col]);
                const float by = m[nb][j] == -INFINITY ? 0.0f : ex2(m[nb][j] - top);
#pragma unroll
                for (int h = 0; h < S::VH; ++h)
#pragma unroll
                    for (int pl = 0; pl < S::PLANES; ++pl)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int d = S::value_byte(h, r) * 8 / BITS + pl + k * S::PLANES;
                            s_o[warp][col * S::STRIDE + d + d / 16] = o[nb][h * S::PLANES + pl][2 * k + j] * (by / (1 << (pl * BITS)));
                        }
            }
        __syncthreads();
        const bool whole = from == 0 && to == tiles;
        float *slot = p.slots + (int64_t)(2 * blockIdx.x + (from == 0)) * p.cols * (DIM + 2);
        for (int i = threadIdx.x; i < heads * DIM; i += 32 * WARPS) {
            const int col = i / DIM, d = i % DIM;
            float sum = 0.0f, total = 0.0f, top = s_m[0][col];
#pragma unroll
            for (int w2 = 1; w2 < WARPS; ++w2) top = fmaxf(top, s_m[w2][col]);
#pragma unroll
            for (int w2 = 0; w2 < WARPS; ++w2) {
                sum += s_o[w2][col * S::STRIDE + d + d / 16];
                if constexpr (REST == 1) sum += s_o[w2][(col + 4) * S::STRIDE + d + d / 16];
                total += s_m[w2][col] == -INFINITY ? (s_l[w2][col] == s_l[w2][col] ? 0.0f : NAN) : s_l[w2][col] * ex2(s_m[w2][col] - top);
            }
            if (whole) ((T *)a.out)[out0 + i] = from_f32<T>(n <= 0 ? 0.0f : sum / total);
            else {
                slot[col * (DIM + 2) + d] = sum;
                if (d == 0) {
                    slot[col * (DIM + 2) + DIM] = top;
                    slot[col * (DIM + 2) + DIM + 1] = total;
                }
            }
        }
        if (p.single) return;
        at += to - from;
        if (to == tiles && unit == p.units - 1) {
            before += tiles;
            ++b;
        }
    }
}

// One CTA a head of a sequence: zeros for an empty sequence, and the parts of one that several CTAs share.
template <typename T>
__global__ void __launch_bounds__(128) kv_attend_join_kernel(const FastArgs p, int dim) {
    pdl_wait();
    const AttendArgs &a = p.a;
    const int64_t b = blockIdx.x / a.heads;
    const int h = (int)(blockIdx.x - b * a.heads), group = a.heads / a.kv_heads, kh = h / group, block = (h - kh * group) / p.cols,
              col = h - kh * group - block * p.cols, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    T *out = (T *)a.out + (int64_t)blockIdx.x * dim;
    const int n = __ldcg(a.lengths + b), tiles = tiles_of(n, p.most_tiles);
    if (tiles == 0) {
        for (int d = threadIdx.x; d < dim; d += 128) out[d] = from_f32<T>(n > 0 ? NAN : 0.0f);
        return;
    }
    int64_t total = 0, before = 0;
    for (int64_t i = lane; i < p.batch; i += 32) {
        const int64_t t = tiles_of(__ldcg(a.lengths + i), p.most_tiles);
        total += t;
        before += i < b ? t : 0;
    }
    for (int d = 16; d; d >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, d);
        before += __shfl_xor_sync(0xffffffffu, before, d);
    }
    const int64_t per = share(p, total * p.units), from = before * p.units + (int64_t)(kh * p.blocks + block) * tiles;
    const int64_t first = from / per, last = (from + tiles - 1) / per;
    if (first == last) return;
    const int64_t stride = (int64_t)2 * p.cols * (dim + 2);       // of CTAs; the first one's part is in its second slot
    const float *parts = p.slots + (int64_t)col * (dim + 2);
    const float *head = parts + first * stride + stride / 2;
    __shared__ float s_o[4][256], s_l[4];
    // each warp: every fourth part
    float top = -INFINITY;
    for (int64_t i = first + lane; i <= last; i += 32) top = fmaxf(top, __ldcg((i == first ? head : parts + i * stride) + dim));
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    float o[8] = {}, l = 0.0f;
#pragma unroll 4
    for (int64_t i = first + warp; i <= last; i += 4) {
        const float *s = i == first ? head : parts + i * stride;
        const float m = __ldcg(s + dim), sum = __ldcg(s + dim + 1), f = m == -INFINITY ? 0.0f : ex2(m - top);
        l += sum == sum ? f * sum : NAN;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (lane + 32 * k < dim) o[k] += f * __ldcg(s + lane + 32 * k);
    }
    if (lane == 0) s_l[warp] = l;
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (lane + 32 * k < dim) s_o[warp][lane + 32 * k] = o[k];
    __syncthreads();
    for (int d = threadIdx.x; d < dim; d += 128)
        out[d] = from_f32<T>((s_o[0][d] + s_o[1][d] + s_o[2][d] + s_o[3][d]) / (s_l[0] + s_l[1] + s_l[2] + s_l[3]));
}

// Whether the tiled kernel takes this cache, and how it divides a call.
bool fast_args(FastArgs &p, int64_t batch, int heads, int kv_heads, int dim, int page_size, int64_t max_pages) {
    if ((dim != 64 && dim != 128 && dim != 256) || page_size % TILE != 0) return false;
    const int group = heads / kv_heads;
    p.batch = batch;
    p.cols = group > 8 && dim < 256 ? 16 : 8;
    p.blocks = (group + p.cols - 1) / p.cols;
    p.units = kv_heads * p.blocks;
    p.tiles_per_page = page_size / TILE;
    p.most_tiles = (int)(max_pages * p.tiles_per_page);
    p.single = p.most_tiles <= SINGLE_TILES;
    return batch * p.units < (int64_t)1 << 31;
}

template <typename T, int BITS, int DIM, int NB, int REST>
int launch_fast(FastArgs &p, cudaStream_t st) {
    static int per_sm = 0;
    if (!per_sm) {
        int n = 0;
        BW_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kv_attend_kernel<T, BITS, DIM, NB, REST>, 32 * WARPS, 0));
        per_sm = n < 1 ? 1 : n > 4 ? 4 : n;
    }
    p.ctas = 148 * per_sm;
    const int64_t grid = p.single ? p.batch * p.units : p.ctas;
    kv_attend_kernel<T, BITS, DIM, NB, REST><<<(unsigned)grid, 32 * WARPS, 0, st>>>(p);
    int rc = check_launch("kv_attend_kernel");
    if (rc != BW_OK || p.single) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.batch * p.a.heads));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    BW_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv_attend_join_kernel<T>, p, DIM));
    return BW_OK;
}

template <typename T, int BITS, int DIM>
int launch_rest(FastArgs &p, cudaStream_t st) {
    constexpr bool EXACT = __is_same(T, __half);
    if constexpr (DIM < 256)
        if (p.cols == 16) return launch_fast<T, BITS, DIM, 2, EXACT ? 2 : 0>(p, st);
    if constexpr (EXACT)
        if (p.a.heads / p.a.kv_heads <= 4) return launch_fast<T, BITS, DIM, 1, 1>(p, st);
    return launch_fast<T, BITS, DIM, 1, EXACT ? 2 : 0>(p, st);
}
template <typename T, int BITS>
int launch_dim(FastArgs &p, cudaStream_t st) {
    if (p.a.dim == 64) return launch_rest<T, BITS, 64>(p, st);
    if (p.a.dim == 128) return launch_rest<T, BITS, 128>(p, st);
    return launch_rest<T, BITS, 256>(p, st);
}
template <typename T>
int launch_bits(FastArgs &p, int bits, cudaStream_t st) {
    return bits == 2 ? launch_dim<T, 2>(p, st) : bits == 4 ? launch_dim<T, 4>(p, st) : launch_dim<T, 8>(p, st);
}

}  // namespace

size_t kv_attend_workspace_bytes(int64_t batch, int heads, int kv_heads, int dim, int page_size, int64_t max_pages) {
    FastArgs p;
    if (!fast_args(p, batch, heads, kv_heads, dim, page_size, max_pages) || p.single) return 0;
    return (size_t)2 * MOST_CTAS * p.cols * (dim + 2) * sizeof(float);
}

int kv_attend(const void *q, int dtype, int64_t batch, int heads, int64_t q_stride, int64_t q_head_stride, const int32_t *kc, const int32_t *vc,
              const void *params, int bits, int64_t pages, int page_size, int kv_heads, int dim, const int32_t *table, int64_t table_stride,
              int max_pages, const int32_t *lengths, float alpha, void *out, void *workspace, cudaStream_t st) {
    FastArgs f = {};
    AttendArgs p = {q, kc, vc, (const __half2 *)params, table, lengths, out, q_stride, q_head_stride, table_stride, pages,
                    heads, kv_heads, dim, dim * bits / 32, page_size, max_pages, alpha};
    if (fast_args(f, batch, heads, kv_heads, dim, page_size, max_pages)) {
        f.a = p;
        f.slots = (float *)workspace;
        return dtype == BW_F16 ? launch_bits<__half>(f, bits, st) : launch_bits<__nv_bfloat16>(f, bits, st);
    }
    return dtype == BW_F16 ? attend_general<__half>(p, batch, bits, st) : attend_general<__nv_bfloat16>(p, batch, bits, st);
}

}  // namespace bw
