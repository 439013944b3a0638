// Low-rank adapters of many requests beside a shared projection: bw_adapter_forward, bw_adapter_backward.
//
//     h[t] = down[i] x[t],  y[t] = base[t] + f_i up[i]^T h[t],  i = index[t]  (none below 0)
//     dh[t] = up[i] dy[t],  dx[t] = f_i down[i]^T dh[t],  d_down[i] = f_i sum dh[t] x[t]^T,  d_up[i] = f_i sum h[t] dy[t]^T
//
// Both matrices of an adapter are stored rank-major, down [n][rank][K] and up [n][rank][N], so that forward and backward are the
// same three passes: "shrink" (rows times a matrix of long rows -> rank values), "expand" (the reverse) and "outer" (sums of
// products over an adapter's tokens).  All three are bound by the bytes of x, base, y and their gradients; the products run on
// mma.sync.m16n8k16, whose fragments come straight from 16-byte loads:
//   * the reduced index of a product may be permuted at will, if both operands are: where rows are long in it (shrink), a lane's 16 bytes
//     of a row serve two MMAs, k pairs (0, 1), (2, 3) and (4, 5), (6, 7);
//   * where it runs over rows (expand over ranks, outer over tokens), a lane takes 16 bytes of four rows, eight columns of its own, and
//     pairs the rows by byte permutations: MMA j of eight has column j of every lane.  A lane's results are then 16 neighbours of a row.
// Rank values stay in 32 bits between the passes and enter the second product as two 16-bit parts (value and rest), which keeps 16 (bf16) or 22
// (fp16) of their bits.  fp16 parts are taken of h * 2^-e, e of the row's largest (expand) or of the largest so far (outer): gradients
// without loss scaling would be lost below 2^-14, and large rank values beyond 65504.
//
// Tokens of one adapter need not be neighbours: a tile of tokens goes through the adapters that occur in it, one after the other or (a few
// tokens, many adapters) a CTA each; outer gathers the tokens of its adapter first.  Rows of other adapters enter no product.
#include <cooperative_groups.h>

#include "bw_common.cuh"

namespace bw {
namespace {

// ---- any sizes and alignments -------------------------------------------------------------------------------------------
// Rank values may be in parts (splits of their sums): the tensor-core forms write them so, and either form may read them.
__device__ __forceinline__ float rank_value(const float *h, int64_t part, int64_t i, int parts) {
    float s = h[i];
    for (int k = 1; k < parts; ++k) s += h[k * part + i];
    return s;
}

template <typename T>
__global__ void __launch_bounds__(128) adapter_shrink_general_kernel(const T *__restrict__ x, int64_t M, int64_t K, const T *__restrict__ w, int n, int r,
                                                                     const int32_t *__restrict__ index, float *h, int parts) {
    const int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / 32, t = i / r;
    const int j = (int)(i - t * r), lane = threadIdx.x % 32;
    if (t >= M) return;
    const int a = index[t];
    float s = 0.0f;
    if (a >= 0 && a < n)
        for (int64_t k = lane; k < K; k += 32) s += to_f32(x[t * K + k]) * to_f32(w[((int64_t)a * r + j) * K + k]);
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (lane == 0)
        for (int k = 0; k < parts; ++k) h[k * M * r + i] = k ? 0.0f : s;
}

template <typename T>
__global__ void __launch_bounds__(256) adapter_expand_general_kernel(const float *__restrict__ h, int64_t M, int64_t N, const T *__restrict__ w, int n, int r,
                                                                     const int32_t *__restrict__ index, const float *__restrict__ scaling, const T *base, T *out, int parts) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= N) return;
    for (int64_t t = blockIdx.y; t < M; t += gridDim.y) {
        const int a = index[t];
        float s = a < n ? 0.0f : NAN;
        if (a >= 0 && a < n) {
            for (int j = 0; j < r; ++j) s += rank_value(h, M * r, t * r + j, parts) * to_f32(w[((int64_t)a * r + j) * N + c]);
            if (scaling) s *= scaling[a];
        }
        out[t * N + c] = from_f32<T>(base ? to_f32(base[t * N + c]) + s : s);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) adapter_outer_general_kernel(const float *__restrict__ h, const T *__restrict__ x, int64_t M, int64_t N, int r,
                                                                    const int32_t *__restrict__ index, const float *__restrict__ scaling, T *dw, int parts) {
    const int64_t c = (int64_t)blockIdx.y * 256 + threadIdx.x;
    const int a = blockIdx.x / r, j = blockIdx.x % r;
    if (c >= N) return;
    float s = 0.0f;
    for (int64_t t = 0; t < M; ++t)
        if (index[t] == a) s += rank_value(h, M * r, t * r + j, parts) * to_f32(x[t * N + c]);
    dw[(int64_t)blockIdx.x * N + c] = from_f32<T>(scaling ? s * scaling[a] : s);
}

// ---- tensor-core forms: K and N multiples of 8, rows on 16-byte boundaries, rank a multiple of 8 up to 128 -----------------

template <typename T> struct Pair;
template <> struct Pair<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
__device__ __forceinline__ uint4 load16_if(const void *p, bool ok) { return ok ? __ldg(reinterpret_cast<const uint4 *>(p)) : make_uint4(0, 0, 0, 0); }
// Column j (of a lane's eight) of two rows beside each other.
__device__ __forceinline__ uint32_t column_pair(const uint4 &even, const uint4 &odd, int j) {
    const uint32_t *a = reinterpret_cast<const uint32_t *>(&even), *b = reinterpret_cast<const uint32_t *>(&odd);
    return __byte_perm(a[j / 2], b[j / 2], j % 2 ? 0x7632 : 0x5410);
}
// The power of two under a positive number (and of what is too small or too large to divide by, one that can be).
__device__ __forceinline__ int exponent_of(float big) { return min(max((int)(__float_as_uint(big) >> 23) - 127, -100), 100); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// The adapters that occur in a tile of up to 64 tokens, in the order of their first token; every warp goes through them alike.  Tokens behind the
// last are in no group.
struct TileAdapters {
    int lo, hi;               // of tokens lane and lane + 32
    unsigned long long todo;
    __device__ __forceinline__ TileAdapters(const int32_t *index, int64_t t0, int64_t M, int tokens) {
        const int lane = threadIdx.x % 32;
        const bool a = lane < tokens && t0 + lane < M, b = lane + 32 < tokens && t0 + lane + 32 < M;
        lo = a ? __ldg(index + t0 + lane) : 0;
        hi = b ? __ldg(index + t0 + lane + 32) : 0;
        todo = __ballot_sync(0xffffffffu, a) | (unsigned long long)__ballot_sync(0xffffffffu, b) << 32;
    }
    // The next adapter and its tokens; false when there is none.
    __device__ __forceinline__ bool next(int &adapter, unsigned long long &tokens) {
        if (!todo) return false;
        const int first = __ffsll((long long)todo) - 1;
        adapter = first < 32 ? __shfl_sync(0xffffffffu, lo, first) : __shfl_sync(0xffffffffu, hi, first - 32);
        tokens = todo & (__ballot_sync(0xffffffffu, lo == adapter) | (unsigned long long)__ballot_sync(0xffffffffu, hi == adapter) << 32);
        todo &= ~tokens;
        return true;
    }
};

struct AdapterArgs {
    int64_t M, cols;            // tokens; length of a row of w (K of down, N of up)
    const int32_t *index;
    const float *scaling;
    int adapters, rank;
    int splits;                 // of the rank values' sums
    int slots;                  // CTAs among which the adapters of a tile of tokens are dealt
};

// Rank values of MW * 16 tokens, one split of the columns: MW warps of 16 tokens, KW parts of the split's columns, NBR * 8 ranks.
template <typename T, int MW, int KW, int NBR>
__global__ void __launch_bounds__(32 * MW * KW) adapter_shrink_kernel(const T *__restrict__ x, const T *__restrict__ w, const AdapterArgs p, int64_t per_split, float *h) {
    constexpr int RANKS = 8 * NBR, UNROLL = NBR <= 2 ? 4 : 2;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32, r = lane / 4, c = lane % 4, wm = warp % MW, wk = warp / MW;
    const int slot = blockIdx.z % p.slots, rank0 = blockIdx.z / p.slots * RANKS;
    const int64_t t0 = (int64_t)blockIdx.x * (16 * MW);
    __shared__ float red[KW > 1 ? KW - 1 : 1][MW * 16][RANKS + 1];
    const int64_t begin = blockIdx.y * per_split, end = begin + per_split < p.cols ? begin + per_split : p.cols;
    const int64_t per_warp = (per_split / 32 + KW - 1) / KW * 32, k0 = begin + wk * per_warp, k1 = k0 + per_warp < end ? k0 + per_warp : end;
    const int64_t ta = t0 + wm * 16 + r, tb = ta + 8;

    TileAdapters in_tile(p.index, t0, p.M, 16 * MW);
    int a;
    unsigned long long tokens;
    for (int i = 0; in_tile.next(a, tokens); ++i) {
        if (i % p.slots != slot || a < 0 || a >= p.adapters) continue;
        const unsigned mine = (unsigned)(tokens >> (16 * wm)) & 0xffffu;
        const bool has_a = mine >> r & 1, has_b = mine >> (r + 8) & 1;
        float acc[NBR][4] = {};
        if (mine) {
            const T *xa = x + ta * p.cols + c * 8, *xb = x + tb * p.cols + c * 8, *wr = w + ((int64_t)a * p.rank + rank0 + r) * p.cols + c * 8;
#pragma unroll UNROLL
            for (int64_t k = k0; k < k1; k += 32) {
                const bool in = k + c * 8 < k1;
                const uint4 va = load16_if(xa + k, in && has_a), vb = load16_if(xb + k, in && has_b);
                const uint32_t lo[4] = {va.x, vb.x, va.y, vb.y}, hi[4] = {va.z, vb.z, va.w, vb.w};
#pragma unroll
                for (int nb = 0; nb < NBR; ++nb) {
                    const uint4 b = load16_if(wr + nb * 8 * p.cols + k, in && rank0 + nb * 8 < p.rank);
                    Pair<T>::mma(acc[nb], lo, b.x, b.y);
                    Pair<T>::mma(acc[nb], hi, b.z, b.w);
                }
            }
        }
        if constexpr (KW > 1) {
            if (wk > 0) {
#pragma unroll
                for (int nb = 0; nb < NBR; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) red[wk - 1][wm * 16 + r + 8 * (e / 2)][nb * 8 + 2 * c + e % 2] = acc[nb][e];
            }
            __syncthreads();
            if (wk == 0) {
#pragma unroll
                for (int nb = 0; nb < NBR; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int o = 0; o < KW - 1; ++o) acc[nb][e] += red[o][wm * 16 + r + 8 * (e / 2)][nb * 8 + 2 * c + e % 2];
            }
        }
        if (wk == 0) {
#pragma unroll
            for (int nb = 0; nb < NBR; ++nb)
                if (rank0 + nb * 8 < p.rank) {
                    float *to = h + ((int64_t)blockIdx.y * p.M + ta) * p.rank + rank0 + nb * 8 + 2 * c;
                    if (has_a) *reinterpret_cast<float2 *>(to) = make_float2(acc[nb][0], acc[nb][1]);
                    if (has_b) *reinterpret_cast<float2 *>(to + 8 * p.rank) = make_float2(acc[nb][2], acc[nb][3]);
                }
        }
        if constexpr (KW > 1) __syncthreads();
    }
}

// Two neighbouring rank values of a token, summed over the splits.
__device__ __forceinline__ float2 rank_pair(const float *h, const AdapterArgs &p, int64_t t, int j) {
    float2 v = __ldg(reinterpret_cast<const float2 *>(h + t * p.rank + j));
    for (int s = 1; s < p.splits; ++s) {
        const float2 o = __ldg(reinterpret_cast<const float2 *>(h + (s * p.M + t) * p.rank + j));
        v.x += o.x;
        v.y += o.y;
    }
    return v;
}

// out[t] = base[t] + f * (h[t] times w) of SUB * 16 tokens, eight warps with 64 columns each at a time; KS steps of 16 ranks at once.
template <typename T, int SUB, int KS>
__global__ void __launch_bounds__(256) adapter_expand_kernel(const float *__restrict__ h, const T *__restrict__ w, const AdapterArgs p, const T *base, T *out) {
    constexpr bool F16 = __is_same(T, __half);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
    const int64_t t0 = (int64_t)blockIdx.x * (16 * SUB);
    const int steps = (p.rank + 15) / 16;
    extern __shared__ uint4 frag[];                              // [SUB][steps][2 (value, rest)][32]
    __shared__ float s_factor[16 * SUB];

    TileAdapters in_tile(p.index, t0, p.M, 16 * SUB);
    // rank values as fragments; rows without an adapter hold zeros
    for (int row = warp; row < 16 * SUB; row += 8) {
        const int64_t t = t0 + row;
        const int a = row < 32 ? __shfl_sync(0xffffffffu, in_tile.lo, row) : __shfl_sync(0xffffffffu, in_tile.hi, row - 32);
        const bool has = t < p.M && a >= 0 && a < p.adapters;
        float2 v[2];
        float big = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int j = 2 * (lane + 32 * i);
            v[i] = has && j < p.rank ? rank_pair(h, p, t, j) : make_float2(0.0f, 0.0f);
            big = fmaxf(big, fmaxf(fabsf(v[i].x), fabsf(v[i].y)));
        }
        float by = 1.0f, back = 1.0f;
        if constexpr (F16) {
            for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
            const int e = exponent_of(big);
            by = power_of_two(-e);
            back = power_of_two(e);
        }
        if (lane == 0) s_factor[row] = has && p.scaling ? back * __ldg(p.scaling + a) : back;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int j = 2 * (lane + 32 * i);
            if (j < 16 * steps) {
                const uint32_t top = Pair<T>::pack(v[i].x * by, v[i].y * by);
                const float2 f = Pair<T>::unpack(top);
                const uint32_t rest = Pair<T>::pack(v[i].x * by - f.x, v[i].y * by - f.y);
                uint32_t *to = reinterpret_cast<uint32_t *>(frag + (size_t)(row / 16 * steps + j / 16) * 64) + ((row % 8) * 4 + j % 8 / 2) * 4 + j % 16 / 8 * 2 + row % 16 / 8;
                to[0] = top;
                to[128] = rest;
            }
        }
    }
    __syncthreads();

    const int64_t first = ((int64_t)blockIdx.y * 8 + warp) * 64, step = (int64_t)gridDim.y * 512;
    int a;
    unsigned long long tokens;
    for (int i = 0; in_tile.next(a, tokens); ++i) {
        if (i % p.slots != (int)blockIdx.z) continue;
        const bool has = a >= 0 && a < p.adapters;
        if (a < 0 && base == out) continue;
        for (int64_t cb = first; cb < p.cols; cb += step) {
            const int64_t col = cb + r * 8;                       // of the lane's columns of w; its results: cb + 16 c and on
            uint32_t b[KS][8][2];
            auto load_w = [&](int k0) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const int j = k0 + 16 * ks + 2 * c;
                    const T *from = w + ((int64_t)a * p.rank + j) * p.cols + col;
                    const bool in = has && col < p.cols;
                    const uint4 w0 = load16_if(from, in && j < p.rank), w1 = load16_if(from + p.cols, in && j < p.rank),
                                w2 = load16_if(from + 8 * p.cols, in && j + 8 < p.rank), w3 = load16_if(from + 9 * p.cols, in && j + 8 < p.rank);
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        b[ks][n][0] = column_pair(w0, w1, n);
                        b[ks][n][1] = column_pair(w2, w3, n);
                    }
                }
            };
            if (has) load_w(0);
#pragma unroll 1
            for (int sub = 0; sub < SUB; ++sub) {
                const unsigned mine = (unsigned)(tokens >> (16 * sub)) & 0xffffu;
                if (!mine) continue;
                const int64_t at = (t0 + sub * 16 + r) * p.cols + cb + 16 * c;
                const bool live[2] = {(bool)(mine >> r & 1), (bool)(mine >> (r + 8) & 1)};
                uint4 old[2][2];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    old[j / 2][j % 2] = base && live[j / 2] && cb + 16 * c + j % 2 * 8 < p.cols
                                            ? *reinterpret_cast<const uint4 *>(base + at + j / 2 * 8 * p.cols + j % 2 * 8) : make_uint4(0, 0, 0, 0);
                float acc[8][4] = {};
                if (has)
                    for (int k = 0; k < steps; k += KS) {
                        if (k > 0 || (steps > KS && sub > 0)) load_w(16 * k);
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks) {
                            if (k + ks >= steps) break;
                            const uint4 *f = frag + (size_t)(sub * steps + k + ks) * 64 + lane;
                            const uint4 top = f[0], rest = f[32];
                            const uint32_t at4[4] = {top.x, top.y, top.z, top.w}, ar[4] = {rest.x, rest.y, rest.z, rest.w};
#pragma unroll
                            for (int n = 0; n < 8; ++n) {
                                Pair<T>::mma(acc[n], at4, b[ks][n][0], b[ks][n][1]);
                                Pair<T>::mma(acc[n], ar, b[ks][n][0], b[ks][n][1]);
                            }
                        }
                    }
#pragma unroll
                for (int j = 0; j < 4; ++j) {                      // row r or r + 8, columns 0 to 7 or 8 to 15 of the lane's
                    if (!live[j / 2] || cb + 16 * c + j % 2 * 8 >= p.cols) continue;
                    const float f = a >= p.adapters ? NAN : s_factor[sub * 16 + r + j / 2 * 8];
                    const uint32_t *o = reinterpret_cast<const uint32_t *>(&old[j / 2][j % 2]);
                    uint32_t y[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const float2 v = Pair<T>::unpack(o[n]);
                        y[n] = a < 0 ? o[n] : Pair<T>::pack(fmaf(acc[2 * n][j], f, v.x), fmaf(acc[2 * n + 1][j], f, v.y));
                    }
                    *reinterpret_cast<uint4 *>(out + at + j / 2 * 8 * p.cols + j % 2 * 8) = make_uint4(y[0], y[1], y[2], y[3]);
                }
            }
        }
    }
}

constexpr int OUTER_LIST = 2048, OUTER_TOKENS = 64;

// dw[a][rank0 .. + 16 RB][256 columns] = f_a * sum over the adapter's tokens of h[t] x[t]^T.  The CTAs of a cluster (blockIdx.z) take equal shares of
// the tokens and add their sums through each other's shared memory.
template <typename T, int RB>
__global__ void __launch_bounds__(128) adapter_outer_kernel(const float *__restrict__ h, const T *__restrict__ x, const AdapterArgs p, T *dw) {
    namespace cg = cooperative_groups;
    constexpr bool F16 = __is_same(T, __half);
    constexpr int RANKS = 16 * RB;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
    const int rank_blocks = (p.rank + RANKS - 1) / RANKS, a = blockIdx.y / rank_blocks, rank0 = blockIdx.y % rank_blocks * RANKS;
    const int64_t cb = (int64_t)blockIdx.x * 256 + warp * 64, col = cb + r * 8;
    extern __shared__ uint4 outer_smem[];
    uint4 *frag = outer_smem;                                    // [4 token steps][RB][2 (value, rest)][32]
    float *sums = reinterpret_cast<float *>(outer_smem);         // [RANKS][256], at the end
    __shared__ int list[OUTER_LIST], s_count[4], s_big[4];

    // the adapter's tokens before this warp's quarter of all, and in all
    const int64_t quarter = (p.M + 127) / 128 * 32, q0 = warp * quarter, q1 = q0 + quarter < p.M ? q0 + quarter : p.M;
    int count = 0;
    for (int64_t t = q0; t < q1; t += 32) count += __popc(__ballot_sync(0xffffffffu, t + lane < q1 && __ldg(p.index + t + lane) == a));
    if (lane == 0) s_count[warp] = count;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < 4; ++i) {
        before += i < warp ? s_count[i] : 0;
        all += s_count[i];
    }
    const int share = (all + gridDim.z - 1) / gridDim.z, lo = blockIdx.z * share, hi = lo + share < all ? lo + share : all;

    float acc[RB][8][4] = {};
    int e = -100;                                                // fp16: the sums are of h * 2^-e
    for (int from = lo; from < hi; from += OUTER_LIST) {
        const int n = hi - from < OUTER_LIST ? hi - from : OUTER_LIST;
        __syncthreads();
        int at = before;
        for (int64_t t = q0; t < q1 && at < from + n; t += 32) {
            const bool mine = t + lane < q1 && __ldg(p.index + t + lane) == a;
            const unsigned m = __ballot_sync(0xffffffffu, mine);
            const int place = at + __popc(m & ((1u << lane) - 1)) - from;
            if (mine && place >= 0 && place < n) list[place] = (int)(t + lane);
            at += __popc(m);
        }
        __syncthreads();
        for (int chunk = 0; chunk < n; chunk += OUTER_TOKENS) {
            // rank values of 64 tokens as fragments (rows are ranks here): a thread takes pairs of tokens of one rank pair
            constexpr int ITEMS = OUTER_TOKENS / 2 * RANKS / 2 / 128;
            float2 v[ITEMS][2];
            float big = 0.0f;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int item = threadIdx.x + 128 * i, j = rank0 + item % (RANKS / 2) * 2, tp = chunk + item / (RANKS / 2) * 2;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    v[i][k] = tp + k < n && j < p.rank ? rank_pair(h, p, list[tp + k], j) : make_float2(0.0f, 0.0f);
                    big = fmaxf(big, fmaxf(fabsf(v[i][k].x), fabsf(v[i][k].y)));
                }
            }
            float by = 1.0f;
            if constexpr (F16) {
                for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
                if (lane == 0) s_big[warp] = exponent_of(big);
            }
            __syncthreads();                                     // (and the fragments before have been used)
            if constexpr (F16) {
                const int now = max(max(s_big[0], s_big[1]), max(s_big[2], s_big[3]));
                if (now > e) {
                    const float down = power_of_two(max(e - now, -126));
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                        for (int j = 0; j < 8; ++j)
#pragma unroll
                            for (int k = 0; k < 4; ++k) acc[rb][j][k] *= down;
                    e = now;
                }
                by = power_of_two(-e);
            }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int item = threadIdx.x + 128 * i, j = item % (RANKS / 2) * 2, tp = item / (RANKS / 2) * 2;
#pragma unroll
                for (int k = 0; k < 2; ++k) {                     // rank j + k, tokens tp and tp + 1
                    const float v0 = (k ? v[i][0].y : v[i][0].x) * by, v1 = (k ? v[i][1].y : v[i][1].x) * by;
                    const uint32_t top = Pair<T>::pack(v0, v1);
                    const float2 f = Pair<T>::unpack(top);
                    uint32_t *to = reinterpret_cast<uint32_t *>(frag + (size_t)(tp / 16 * RB + j / 16) * 64) + (((j + k) % 8) * 4 + tp % 8 / 2) * 4 + tp % 16 / 8 * 2 + j % 16 / 8;
                    to[0] = top;
                    to[128] = Pair<T>::pack(v0 - f.x, v1 - f.y);
                }
            }
            __syncthreads();
            if (cb < p.cols) {
#pragma unroll 2
                for (int step = 0; step < OUTER_TOKENS / 16; ++step) {
                    if (chunk + step * 16 >= n) break;
                    uint4 rows[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int i = chunk + step * 16 + 2 * c + k % 2 + k / 2 * 8;
                        const bool in = i < n && col < p.cols;
                        rows[k] = load16_if(x + (in ? (int64_t)list[i] * p.cols + col : 0), in);
                    }
                    uint32_t b[8][2];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        b[j][0] = column_pair(rows[0], rows[1], j);
                        b[j][1] = column_pair(rows[2], rows[3], j);
                    }
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        const uint4 *f = frag + (size_t)(step * RB + rb) * 64 + lane;
                        const uint4 top = f[0], rest = f[32];
                        const uint32_t at4[4] = {top.x, top.y, top.z, top.w}, ar[4] = {rest.x, rest.y, rest.z, rest.w};
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            Pair<T>::mma(acc[rb][j], at4, b[j][0], b[j][1]);
                            Pair<T>::mma(acc[rb][j], ar, b[j][0], b[j][1]);
                        }
                    }
                }
            }
        }
    }

    // sums of this CTA, in 16 neighbouring columns a lane; then those of the cluster
    const float f = (F16 ? power_of_two(e) : 1.0f) * (p.scaling ? __ldg(p.scaling + a) : 1.0f);
    __syncthreads();
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) sums[(rb * 16 + r + k / 2 * 8) * 256 + warp * 64 + c * 16 + k % 2 * 8 + j] = acc[rb][j][k] * f;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int parts = gridDim.z, mine = blockIdx.z;
    for (int i = mine * 128 + threadIdx.x; i < RANKS * 32; i += parts * 128) {        // eight columns of a rank
        const int rank = rank0 + i / 32;
        const int64_t at = (int64_t)blockIdx.x * 256 + i % 32 * 8;
        if (rank >= p.rank || at >= p.cols) continue;
        float4 s0 = make_float4(0, 0, 0, 0), s1 = s0;
        for (int o = 0; o < parts; ++o) {
            const float4 *from = reinterpret_cast<const float4 *>(cluster.map_shared_rank(sums, o) + i * 8);
            const float4 u = from[0], v = from[1];
            s0.x += u.x; s0.y += u.y; s0.z += u.z; s0.w += u.w;
            s1.x += v.x; s1.y += v.y; s1.z += v.z; s1.w += v.w;
        }
        *reinterpret_cast<uint4 *>(dw + ((int64_t)a * p.rank + rank) * p.cols + at) =
            make_uint4(Pair<T>::pack(s0.x, s0.y), Pair<T>::pack(s0.z, s0.w), Pair<T>::pack(s1.x, s1.y), Pair<T>::pack(s1.z, s1.w));
    }
    cluster.sync();                                              // a CTA's sums stay until the others have read them
}

// ---- host side -------------------------------------------------------------------------------------------------------

bool fast_rank(int r) { return r % 8 == 0 && r <= 128; }

// Splits of a shrink pass's columns.  They go by sizes alone, so that whoever reads the rank values knows how many parts they have.
int shrink_splits(int64_t M, int64_t cols, int r) {
    if (!fast_rank(r) || cols % 8 != 0) return 1;
    const int64_t tiles = M <= 64 ? (M + 15) / 16 : (M + 31) / 32;
    int64_t s = 256 / (tiles > 0 ? tiles : 1), most = (cols + 511) / 512;
    if (s > most) s = most;
    if (s > 8) s = 8;
    return s < 1 ? 1 : (int)s;
}

template <typename T, int NBR>
int shrink_fast(const T *x, const T *w, AdapterArgs p, float *h, cudaStream_t st) {
    const int64_t per_split = ((p.cols + p.splits - 1) / p.splits + 31) / 32 * 32;
    const int rank_blocks = (p.rank + 8 * NBR - 1) / (8 * NBR);
    if (p.M <= 64) {
        p.slots = p.adapters + 1 < 16 ? p.adapters + 1 : 16;
        adapter_shrink_kernel<T, 1, 8, NBR><<<dim3((unsigned)((p.M + 15) / 16), p.splits, p.slots * rank_blocks), 256, 0, st>>>(x, w, p, per_split, h);
    } else {
        p.slots = 1;
        adapter_shrink_kernel<T, 2, 4, NBR><<<dim3((unsigned)((p.M + 31) / 32), p.splits, rank_blocks), 256, 0, st>>>(x, w, p, per_split, h);
    }
    return check_launch("adapter_shrink_kernel");
}

template <typename T>
int shrink(const void *xv, const void *wv, const AdapterArgs &p, float *h, cudaStream_t st) {
    const T *x = (const T *)xv, *w = (const T *)wv;
    if (fast_rank(p.rank) && p.cols % 8 == 0 && aligned_to(x, 16) && aligned_to(w, 16)) {
        if (p.rank <= 8) return shrink_fast<T, 1>(x, w, p, h, st);
        if (p.rank <= 16) return shrink_fast<T, 2>(x, w, p, h, st);
        if (p.rank <= 32) return shrink_fast<T, 4>(x, w, p, h, st);
        return shrink_fast<T, 8>(x, w, p, h, st);
    }
    adapter_shrink_general_kernel<T><<<(unsigned)((p.M * p.rank + 3) / 4), 128, 0, st>>>(x, p.M, p.cols, w, p.adapters, p.rank, p.index, h, p.splits);
    return check_launch("adapter_shrink_general_kernel");
}

template <typename T, int SUB, int KS>
int expand_fast(const float *h, const T *w, const AdapterArgs &p, const T *base, T *out, cudaStream_t st) {
    const int64_t tiles = (p.M + 16 * SUB - 1) / (16 * SUB), most = (p.cols + 511) / 512;
    int64_t groups = SUB == 1 ? most : (592 + tiles - 1) / tiles;
    if (groups > most) groups = most;
    const size_t smem = (size_t)SUB * ((p.rank + 15) / 16) * 1024;
    adapter_expand_kernel<T, SUB, KS><<<dim3((unsigned)tiles, (unsigned)groups, p.slots), 256, smem, st>>>(h, w, p, base, out);
    return check_launch("adapter_expand_kernel");
}

template <typename T>
int expand(const float *h, const void *wv, AdapterArgs p, const void *base, void *out, cudaStream_t st) {
    const T *w = (const T *)wv, *b = (const T *)base;
    T *o = (T *)out;
    if (fast_rank(p.rank) && p.cols % 8 == 0 && aligned_to(w, 16) && aligned_to(b, 16) && aligned_to(o, 16)) {
        if (p.M <= 64) {
            p.slots = p.adapters + 1 < 16 ? p.adapters + 1 : 16;
            if (p.rank <= 16) return expand_fast<T, 1, 1>(h, w, p, b, o, st);
            if (p.rank <= 32) return expand_fast<T, 1, 2>(h, w, p, b, o, st);
            return expand_fast<T, 1, 4>(h, w, p, b, o, st);
        }
        p.slots = 1;
        if (p.rank <= 16) return expand_fast<T, 4, 1>(h, w, p, b, o, st);
        if (p.rank <= 32) return expand_fast<T, 4, 2>(h, w, p, b, o, st);
        return expand_fast<T, 4, 4>(h, w, p, b, o, st);
    }
    adapter_expand_general_kernel<T><<<dim3((unsigned)((p.cols + 255) / 256), (unsigned)(p.M < 16384 ? p.M : 16384)), 256, 0, st>>>(
        h, p.M, p.cols, w, p.adapters, p.rank, p.index, p.scaling, b, o, p.splits);
    return check_launch("adapter_expand_general_kernel");
}

template <typename T, int RB>
int outer_fast(const float *h, const T *x, const AdapterArgs &p, T *dw, cudaStream_t st) {
    const int64_t blocks = (p.cols + 255) / 256, rows = (int64_t)p.adapters * ((p.rank + 16 * RB - 1) / (16 * RB));
    int parts = 1;
    while (parts < 8 && blocks * rows * parts < 296 && p.M > (int64_t)parts * OUTER_TOKENS) parts *= 2;
    const size_t sums = (size_t)RB * 16 * 256 * sizeof(float);      // (the fragments, RB * 4 KB, are less)
    auto kern = adapter_outer_kernel<T, RB>;
    if (sums > 48 * 1024) BW_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sums));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks, (unsigned)rows, parts);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = sums;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = parts;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    BW_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, h, x, p, dw));
    return check_launch("adapter_outer_kernel");
}

template <typename T>
int outer(const float *h, const void *xv, const AdapterArgs &p, void *dwv, cudaStream_t st) {
    const T *x = (const T *)xv;
    T *dw = (T *)dwv;
    const int rb = p.rank <= 16 ? 1 : p.rank <= 32 ? 2 : 4;
    if (fast_rank(p.rank) && p.cols % 8 == 0 && aligned_to(x, 16) && aligned_to(dw, 16) && p.M < INT32_MAX &&
        (int64_t)p.adapters * ((p.rank + 16 * rb - 1) / (16 * rb)) <= 65535) {
        if (rb == 1) return outer_fast<T, 1>(h, x, p, dw, st);
        if (rb == 2) return outer_fast<T, 2>(h, x, p, dw, st);
        return outer_fast<T, 4>(h, x, p, dw, st);
    }
    adapter_outer_general_kernel<T><<<dim3((unsigned)(p.adapters * p.rank), (unsigned)((p.cols + 255) / 256)), 256, 0, st>>>(
        h, x, p.M, p.cols, p.rank, p.index, p.scaling, dw, p.splits);
    return check_launch("adapter_outer_general_kernel");
}

AdapterArgs args_of(int64_t M, int64_t cols, const int32_t *index, const float *scaling, int n, int r, int splits) {
    return {M, cols, index, scaling, n, r, splits, 1};
}

template <typename T>
int forward(const void *x, int64_t M, int64_t N, int64_t K, const void *down, const void *up, int n, int r, const int32_t *index, const float *scaling,
            const void *base, void *out, float *h, cudaStream_t st) {
    const int splits = shrink_splits(M, K, r);
    const int rc = shrink<T>(x, down, args_of(M, K, index, nullptr, n, r, splits), h, st);
    return rc != BW_OK ? rc : expand<T>(h, up, args_of(M, N, index, scaling, n, r, splits), base, out, st);
}
template <typename T>
int backward(const void *dy, const void *x, int64_t M, int64_t N, int64_t K, const void *down, const void *up, int n, int r, const int32_t *index,
             const float *scaling, const float *h, void *dx, void *d_down, void *d_up, float *dh, cudaStream_t st) {
    const int splits = shrink_splits(M, N, r);
    int rc = BW_OK;
    if (M > 0 && (dx || d_down)) rc = shrink<T>(dy, up, args_of(M, N, index, nullptr, n, r, splits), dh, st);
    if (rc == BW_OK && M > 0 && dx) rc = expand<T>(dh, down, args_of(M, K, index, scaling, n, r, splits), nullptr, dx, st);
    if (rc == BW_OK && d_down) rc = outer<T>(dh, x, args_of(M, K, index, scaling, n, r, splits), d_down, st);
    if (rc == BW_OK && d_up) rc = outer<T>(h, dy, args_of(M, N, index, scaling, n, r, shrink_splits(M, K, r)), d_up, st);
    return rc;
}

}  // namespace

size_t adapter_hidden_bytes(int64_t M, int64_t K, int, int r) { return (size_t)M * r * shrink_splits(M, K, r) * sizeof(float); }
size_t adapter_backward_bytes(int64_t M, int64_t N, int64_t, int, int r) { return (size_t)M * r * shrink_splits(M, N, r) * sizeof(float); }

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
