// Low-rank adapters of many requests beside a shared projection: bw_adapter_forward, bw_adapter_backward.
//
//     h[t] = down[i] x[t],  y[t] = base[t] + f_i up[i]^T h[t],  i = index[t]  (none below 0)
//     dh[t] = up[i] dy[t],  dx[t] = f_i down[i]^T dh[t],  d_down[i] = f_i sum dh[t] x[t]^T,  d_up[i] = f_i sum h[t] dy[t]^T
//
// Both matrices of an adapter are stored rank-major, down [n][rank][K] and up [n][rank][N], so that forward and backward are the
// same three passes: "shrink" (rows times a matrix of long rows -> rank values), "expand" (the reverse) and "outer" (sums of
// products over an adapter's tokens).  What they cannot do without are the bytes of x, base, y and their gradients; what bounds each in fact is said at the kernels.  Products of few
// tokens or ranks run on mma.sync.m16n8k16, whose fragments come from 16-byte loads:
//   * the reduced index of a product may be permuted at will, if both operands are: where rows are long in it (shrink of a few tokens), a
//     lane's 16 bytes of a row serve two MMAs, k pairs (0, 1), (2, 3) and (4, 5), (6, 7);
//   * where it runs over rows (expand over ranks, outer over tokens), a lane takes 16 bytes of four rows, eight columns of its own, and
//     pairs the rows by byte permutations: MMA j of eight has column j of every lane.  A lane's results are then 16 neighbours of a row.
// Rank values are summed in 32 bits.  The second product takes them in 16-bit parts: value and rests, three of bf16, which hold all 24 bits, two of fp16, which hold 22.
// (Two of bf16 hold 16: results of bf16 were off by up to 2^-17 more than their own rounding.)  Between the launches bf16 rank values are fp32, split where they are used;
// fp16 parts are kept as such, of h * 2^(14 - e), e of the row's largest: gradients without loss scaling would be lost below 2^-14, and large rank values beyond 65504.
//
// Tokens of one adapter need not be neighbours: a tile of 64 tokens goes through the adapters that occur in it, one after the other or (few
// tokens, many adapters) a CTA each, with the rows of each gathered; outer gathers the tokens of its adapter from all.  Rows of other
// adapters enter no product.
#include <cooperative_groups.h>

#include <atomic>

#include "early_launch.cuh"
#include "umma.cuh"

namespace bw {
namespace {

// ---- any sizes and alignments -------------------------------------------------------------------------------------------
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
    if (lane == 0) h[i] = s;
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
    // sums of 64 tokens, added up with the part that the addition rounds off carried along (Kahan): one running fp32 sum of M products could be off by M * 2^-24 of them
    float s = 0.0f, carry = 0.0f;
    for (int64_t t0 = 0; t0 < M; t0 += 64) {
        float block = 0.0f;
        const int64_t end = t0 + 64 < M ? t0 + 64 : M;
#pragma unroll 8
        for (int64_t t = t0; t < end; ++t)
            if (index[t] == a) block += h[t * r + j] * to_f32(x[t * N + c]);
        const float y = __fsub_rn(block, carry), next = __fadd_rn(s, y);
        carry = isfinite(next) ? __fsub_rn(__fsub_rn(next, s), y) : 0.0f;
        s = next;
    }
    dw[(int64_t)blockIdx.x * N + c] = from_f32<T>(scaling ? s * scaling[a] : s);
}

// ---- tensor-core forms: K and N multiples of 8, rank a multiple of 8 up to 128 -----------------------------------------------

namespace cg = cooperative_groups;

template <typename T> struct Pair;
template <> struct Pair<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    // d = a * b
    static __device__ __forceinline__ void mma_new(float (&d)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    }
};
template <> struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    // d = a * b
    static __device__ __forceinline__ void mma_new(float (&d)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    }
};
// (From L2, as all that a kernel before may have written: the SM's L1 may hold lines from before this kernel's start, at which they were still being written.)
__device__ __forceinline__ uint4 load16_if(const void *p, bool ok) { return ok ? __ldcg(reinterpret_cast<const uint4 *>(p)) : make_uint4(0, 0, 0, 0); }
// Column j (of a lane's eight) of two rows beside each other.
__device__ __forceinline__ uint32_t column_pair(const uint4 &even, const uint4 &odd, int j) {
    const uint32_t *a = reinterpret_cast<const uint32_t *>(&even), *b = reinterpret_cast<const uint32_t *>(&odd);
    return __byte_perm(a[j / 2], b[j / 2], j % 2 ? 0x7632 : 0x5410);
}
// The power of two under a positive number (and of what is too small or too large to divide by, one that can be).
__device__ __forceinline__ int exponent_of(float big) { return min(max((int)(__float_as_uint(big) >> 23) - 127, -100), 100); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes to shared memory, asynchronously, or 16 zeros (`bytes` 0: nothing is read).
__device__ __forceinline__ void copy16(uint32_t to, const void *from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Arrives once this thread's copies so far have been made (counted among the barrier's arrivals).
__device__ __forceinline__ void copies_arrive(uint64_t *bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 load_shared16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void load_matrices(uint32_t at, uint32_t (&x)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t at, uint32_t (&x)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
}

constexpr int TILE = 64;          // tokens

struct AdapterArgs {
    int64_t M, cols;            // tokens; length of a row of w (K of down, N of up)
    const int32_t *index;
    const float *scaling;
    int adapters, rank;
    int slots;                  // CTAs among which the adapters of a tile of tokens are dealt
    bool behind;                // another launch of this call comes before: all that came before that is done when this one starts
};

// Rank values.  bf16: fp32 [M][rank], and of many tokens their parts [3][M][rank] as well, for outer on tcgen05.  fp16: [2][M][rank], values and their rests, and [M] powers of
// two by which both were divided.
constexpr int64_t MANY = 512;
template <typename T> constexpr int PARTS = __is_same(T, __half) ? 2 : 3;
template <typename T> struct Hidden {
    float *sum;
    T *parts;
    int64_t size;             // of a part
    __host__ __device__ Hidden(void *p, int64_t M, int r) : sum((float *)p), parts(reinterpret_cast<T *>(sum + M * r)), size(M * r) {}
};
template <> struct Hidden<__half> {
    __half *top, *rest;
    float *back;
    __host__ __device__ Hidden(void *p, int64_t M, int r) : top((__half *)p), rest(top + M * r), back(reinterpret_cast<float *>(rest + M * r)) {}
};
// Two values as pairs of 16 bits: themselves and rests.
template <typename T, int N>
__device__ __forceinline__ void split(float2 v, uint32_t (&parts)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        parts[i] = Pair<T>::pack(v.x, v.y);
        const float2 f = Pair<T>::unpack(parts[i]);
        v = make_float2(v.x - f.x, v.y - f.y);
    }
}
// Eight neighbouring fp32 values as 16 bytes of each part.
template <typename T, int N>
__device__ __forceinline__ void split8(const float4 &a, const float4 &b, uint4 (&parts)[N]) {
    const float2 v[4] = {make_float2(a.x, a.y), make_float2(a.z, a.w), make_float2(b.x, b.y), make_float2(b.z, b.w)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t u[N];
        split<T>(v[i], u);
#pragma unroll
        for (int k = 0; k < N; ++k) reinterpret_cast<uint32_t *>(&parts[k])[i] = u[k];
    }
}

// The adapters that occur in a tile of tokens, in the order of their first token, each with a list of its tokens (every warp has its own).  Tokens
// behind the last are in no group.
struct TileAdapters {
    int lo, hi;               // of tokens lane and lane + 32
    unsigned has_lo, has_hi;  // tokens there are
    bool first_lo, first_hi;  // the lane's tokens are the first of their adapters
    int rank_lo, rank_hi;     // how many adapters come before them
    uint8_t *list;            // [TILE] places in the tile
    int groups, count, adapter;
    __device__ __forceinline__ TileAdapters(const AdapterArgs &p, int64_t t0, uint8_t *list) : list(list) {
        const int lane = threadIdx.x % 32;
        const unsigned below = (1u << lane) - 1;
        const bool a = t0 + lane < p.M, b = t0 + lane + 32 < p.M;
        lo = a ? __ldcg(p.index + t0 + lane) : 0;
        hi = b ? __ldcg(p.index + t0 + lane + 32) : 0;
        has_lo = __ballot_sync(0xffffffffu, a);
        has_hi = __ballot_sync(0xffffffffu, b);
        const unsigned like_lo = __match_any_sync(0xffffffffu, lo), like_hi = __match_any_sync(0xffffffffu, hi);      // (by all lanes)
        first_lo = a && !(like_lo & has_lo & below);
        first_hi = b && !(like_hi & has_hi & below);
        if (has_hi) {         // (then all of the first 32 are there)
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (__shfl_sync(0xffffffffu, lo, i) == hi) first_hi = false;
        }
        const unsigned f = __ballot_sync(0xffffffffu, first_lo), g = __ballot_sync(0xffffffffu, first_hi);
        rank_lo = __popc(f & below);
        rank_hi = __popc(f) + __popc(g & below);
        groups = __popc(f) + __popc(g);
    }
    // Takes adapter i of `groups`.
    __device__ __forceinline__ void take(int i) {
        const int lane = threadIdx.x % 32;
        const unsigned below = (1u << lane) - 1, f = __ballot_sync(0xffffffffu, first_lo && rank_lo == i), g = __ballot_sync(0xffffffffu, first_hi && rank_hi == i);
        adapter = f ? __shfl_sync(0xffffffffu, lo, __ffs(f) - 1) : __shfl_sync(0xffffffffu, hi, (__ffs(g) - 1) & 31);
        const unsigned a = __ballot_sync(0xffffffffu, lo == adapter) & has_lo, b = __ballot_sync(0xffffffffu, hi == adapter) & has_hi;
        __syncwarp();         // (the list before has been read)
        if (a >> lane & 1) list[__popc(a & below)] = (uint8_t)lane;
        if (b >> lane & 1) list[__popc(a) + __popc(b & below)] = (uint8_t)(lane + 32);
        count = __popc(a) + __popc(b);
        __syncwarp();
    }
};

// The end of a shrink pass: the CTAs of a cluster have sums of their part of the columns in `sums` [rows][RANKS + 4]; each CTA adds up its share of
// the rows, a warp a row, and writes them.
template <typename T, int RANKS>
__device__ __forceinline__ void finish_rows(float *sums, int rows, int row0, int count, const uint8_t *list, int64_t t0, const AdapterArgs &p, const Hidden<T> &h) {
    constexpr bool F16 = __is_same(T, __half);
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32, parts = gridDim.x, mine = blockIdx.x;
    for (int row = mine + parts * warp; row < rows && row0 + row < count; row += parts * warps) {
        constexpr int PAIRS = RANKS <= 64 ? 1 : 2;
        float2 v[PAIRS];
        float big = 0.0f;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            const int j = 2 * (lane + 32 * i);
            v[i] = make_float2(0.0f, 0.0f);
            if (j < RANKS)
                for (int o = 0; o < parts; ++o) {
                    const float2 u = *reinterpret_cast<const float2 *>(cluster.map_shared_rank(sums, o) + row * (RANKS + 4) + j);
                    v[i].x += u.x;
                    v[i].y += u.y;
                }
            big = fmaxf(big, fmaxf(fabsf(v[i].x), fabsf(v[i].y)));
        }
        const int64_t t = t0 + list[row0 + row];
        if constexpr (F16) {
            for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
            const int e = exponent_of(big);
            // (the largest to 2^14 and more: a rank has 22 bits down to 2^-16 of it, and what is lost below is less than 2^-39 of it)
            const float by = power_of_two(14 - e);
            if (lane == 0) h.back[t] = power_of_two(e - 14);
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const int j = 2 * (lane + 32 * i);
                if (j < p.rank) {
                    uint32_t parts[2];
                    split<T>(make_float2(v[i].x * by, v[i].y * by), parts);
                    *reinterpret_cast<uint32_t *>(h.top + t * p.rank + j) = parts[0];
                    *reinterpret_cast<uint32_t *>(h.rest + t * p.rank + j) = parts[1];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const int j = 2 * (lane + 32 * i);
                if (j < p.rank) {
                    *reinterpret_cast<float2 *>(h.sum + t * p.rank + j) = v[i];
                    if (p.M >= MANY) {
                        uint32_t parts[3];
                        split<T>(v[i], parts);
#pragma unroll
                        for (int k = 0; k < 3; ++k) *reinterpret_cast<uint32_t *>(h.parts + k * h.size + t * p.rank + j) = parts[k];
                    }
                }
            }
        }
    }
    cluster.sync();                                          // the sums stay until the others have read them
}

// Rank values of a few tokens (up to 64): a CTA for each adapter and part of the columns, eight warps with a part of that each, fragments from global
// memory.
template <typename T, int NBR>
__global__ void __launch_bounds__(256) adapter_shrink_few_kernel(const T *__restrict__ x, const T *__restrict__ w, const AdapterArgs p, int64_t per_split, void *hidden) {
    constexpr int RANKS = 8 * NBR, UNROLL = NBR <= 4 ? 4 : 2;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
    __shared__ __align__(16) float sums[16][RANKS + 4];
    extern __shared__ float red[];                            // [7][16][RANKS + 1]
    __shared__ uint8_t lists[8][TILE];
    const Hidden<T> h(hidden, p.M, p.rank);
    pdl_wait();
    pdl_launch_dependents();
    const int64_t begin = blockIdx.x * per_split, end = begin + per_split < p.cols ? begin + per_split : p.cols;
    const int64_t per_warp = (per_split / 32 + 7) / 8 * 32, k0 = begin + warp * per_warp, k1 = k0 + per_warp < end ? k0 + per_warp : end;

    TileAdapters tile(p, 0, lists[warp]);
    for (int i = blockIdx.y; i < tile.groups; i += p.slots) {
        tile.take(i);
        const int a = tile.adapter;
        if (a < 0 || a >= p.adapters) continue;
        for (int row0 = 0; row0 < tile.count; row0 += 16) {
            const bool has_a = row0 + r < tile.count, has_b = row0 + r + 8 < tile.count;
            const T *xa = x + (has_a ? tile.list[row0 + r] : 0) * p.cols + c * 8, *xb = x + (has_b ? tile.list[row0 + r + 8] : 0) * p.cols + c * 8;
            const T *wr = w + ((int64_t)a * p.rank + r) * p.cols + c * 8;
            float acc[NBR][4] = {};
#pragma unroll UNROLL
            for (int64_t k = k0; k < k1; k += 32) {
                const bool in = k + c * 8 < k1;
                const uint4 va = load16_if(xa + k, in && has_a), vb = load16_if(xb + k, in && has_b);
                const uint32_t lo[4] = {va.x, vb.x, va.y, vb.y}, hi[4] = {va.z, vb.z, va.w, vb.w};
#pragma unroll
                for (int nb = 0; nb < NBR; ++nb) {
                    const uint4 b = load16_if(wr + nb * 8 * p.cols + k, in && nb * 8 < p.rank);
                    Pair<T>::mma(acc[nb], lo, b.x, b.y);
                    Pair<T>::mma(acc[nb], hi, b.z, b.w);
                }
            }
            if (warp > 0) {
#pragma unroll
                for (int nb = 0; nb < NBR; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) red[((warp - 1) * 16 + r + 8 * (e / 2)) * (RANKS + 1) + nb * 8 + 2 * c + e % 2] = acc[nb][e];
            } else {
#pragma unroll
                for (int nb = 0; nb < NBR; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sums[r + 8 * (e / 2)][nb * 8 + 2 * c + e % 2] = acc[nb][e];
            }
            __syncthreads();
            for (int j = threadIdx.x; j < 16 * RANKS; j += 256) {
                float s = sums[j / RANKS][j % RANKS];
#pragma unroll
                for (int o = 0; o < 7; ++o) s += red[(o * 16 + j / RANKS) * (RANKS + 1) + j % RANKS];
                sums[j / RANKS][j % RANKS] = s;
            }
            finish_rows<T, RANKS>(&sums[0][0], 16, row0, tile.count, tile.list, 0, p, h);
        }
    }
}

constexpr int SHRINK_STAGES = 3;

// Rank values of many tokens: 64 rows of one adapter, a part of the columns; rows of x and of w go through a ring in shared memory, 64 columns a
// stage, in 16-byte pieces exchanged by row so that ldmatrix meets all banks.
template <typename T, int NBR>
__global__ void __launch_bounds__(128) adapter_shrink_kernel(const T *__restrict__ x, const T *__restrict__ w, const AdapterArgs p, int64_t per_split, void *hidden) {
    constexpr int RANKS = 8 * NBR, STAGE = (TILE + RANKS) * 128, STAGES = SHRINK_STAGES;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint8_t lists[4][TILE];
    const uint32_t ring = smem_addr(smem);
    const Hidden<T> h(hidden, p.M, p.rank);
    pdl_wait();
    pdl_launch_dependents();
    const int64_t t0 = (int64_t)blockIdx.y * TILE, begin = blockIdx.x * per_split, end = begin + per_split < p.cols ? begin + per_split : p.cols;

    TileAdapters tile(p, t0, lists[warp]);
    for (int i = blockIdx.z; i < tile.groups; i += p.slots) {
        tile.take(i);
        const int a = tile.adapter;
        if (a < 0 || a >= p.adapters) continue;
        // a thread copies piece threadIdx % 8 of every 16th row
        const int piece = threadIdx.x % 8;
        constexpr int WROWS = (RANKS + 15) / 16;
        const T *rows[4], *wrows[WROWS];
        int bytes[4], wbytes[WROWS];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = threadIdx.x / 8 + 16 * j;
            bytes[j] = row < tile.count ? 16 : 0;
            rows[j] = x + (t0 + (row < tile.count ? tile.list[row] : 0)) * p.cols + piece * 8;
        }
#pragma unroll
        for (int j = 0; j < WROWS; ++j) {
            const int rank = threadIdx.x / 8 + 16 * j;
            wbytes[j] = rank < p.rank ? 16 : 0;
            wrows[j] = w + ((int64_t)a * p.rank + (rank < p.rank ? rank : 0)) * p.cols + piece * 8;
        }
        const int swizzled = threadIdx.x / 8 * 128 + ((piece ^ (threadIdx.x / 8 & 7)) * 16);
        auto copy_stage = [&](int64_t k, int stage) {
            if (k < end) {
                const bool in = k + piece * 8 < end;
                const uint32_t to = ring + stage * STAGE + swizzled;
#pragma unroll
                for (int j = 0; j < 4; ++j) copy16(to + j * 2048, rows[j] + k, in ? bytes[j] : 0);
#pragma unroll
                for (int j = 0; j < WROWS; ++j)
                    if (RANKS >= 16 || threadIdx.x / 8 < RANKS) copy16(to + TILE * 128 + j * 2048, wrows[j] + k, in ? wbytes[j] : 0);
            }
            copies_commit();
        };
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) copy_stage(begin + s * 64, s);
        float acc[NBR][4] = {};
        const bool busy = warp * 16 < tile.count;
        // a lane's places in the stage (rows of x, of w; a step of 16 columns changes bits 5 and 6)
        const uint32_t x_place = (warp * 16 + lane % 16) * 128 + ((lane / 16) ^ (lane & 7)) * 16,
                       w_place = TILE * 128 + (NBR == 1 ? lane % 8 : lane % 8 + lane / 16 * 8) * 128 + ((lane / 8 % 2) ^ (lane & 7)) * 16;
        int stage = 0;
        for (int64_t k = begin; k < end; k += 64) {
            copies_wait<STAGES - 2>();
            __syncthreads();                                 // the stage is there for all, and the one filled next has been used by all
            copy_stage(k + (STAGES - 1) * 64, stage == 0 ? STAGES - 1 : stage - 1);
            const uint32_t at = ring + stage * STAGE;
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            if (busy) {
                uint32_t xa[4][4];
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) load_matrices(at + (x_place ^ kk * 32), xa[kk]);
                // (sums of 64 columns, added up in fp32: an MMA truncates what it adds to, which is a bias of 2^-24 of the sum each time)
#pragma unroll
                for (int nb = 0; nb < NBR; nb += 2) {
                    float some[2][4];
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        uint32_t b[4];                                   // (rank 8: the second pair is the first again)
                        load_matrices(at + (w_place ^ kk * 32) + nb * 1024, b);
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            if (nb + i >= NBR) continue;
                            else if (kk == 0) Pair<T>::mma_new(some[i], xa[kk], b[2 * i], b[2 * i + 1]);
                            else Pair<T>::mma(some[i], xa[kk], b[2 * i], b[2 * i + 1]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc[nb][e] += some[0][e];
                        if (nb + 1 < NBR) acc[nb + 1 < NBR ? nb + 1 : nb][e] += some[1][e];
                    }
                }
            }
        }
        copies_wait<0>();
        __syncthreads();
        float *sums = reinterpret_cast<float *>(smem);       // [TILE][RANKS + 4]
#pragma unroll
        for (int nb = 0; nb < NBR; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[(warp * 16 + r + 8 * (e / 2)) * (RANKS + 4) + nb * 8 + 2 * c + e % 2] = acc[nb][e];
        finish_rows<T, RANKS>(sums, TILE, 0, tile.count, tile.list, t0, p, h);
    }
}

// ---- expand --------------------------------------------------------------------------------------------------------------

// Fragments of the rank values of 16 rows, from step `first` of 16 ranks on: [parts][steps].
template <typename T, int KS>
__device__ __forceinline__ void load_rank_values(const Hidden<T> &h, int rank, int first, int64_t ta, int64_t tb, bool has_a, bool has_b, int c,
                                                 uint32_t (&values)[PARTS<T>][KS][4]) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = 16 * (first + ks) + 2 * c + e / 2 * 8;
            const bool has = (e % 2 ? has_b : has_a) && j < rank;
            const int64_t at = (e % 2 ? tb : ta) * rank + j;
            if constexpr (__is_same(T, __half)) {
                values[0][ks][e] = has ? __ldcg(reinterpret_cast<const uint32_t *>(h.top + at)) : 0u;
                values[1][ks][e] = has ? __ldcg(reinterpret_cast<const uint32_t *>(h.rest + at)) : 0u;
            } else {
                uint32_t parts[3];
                split<T>(has ? __ldcg(reinterpret_cast<const float2 *>(h.sum + at)) : make_float2(0.0f, 0.0f), parts);
#pragma unroll
                for (int i = 0; i < 3; ++i) values[i][ks][e] = parts[i];
            }
        }
}
// The power of two by which a row's rank values were divided.
__device__ __forceinline__ float power_of_row(const Hidden<__half> &h, int64_t t) { return __ldcg(h.back + t); }
__device__ __forceinline__ float power_of_row(const Hidden<__nv_bfloat16> &, int64_t) { return 1.0f; }
// What a row's product is multiplied by.
template <typename T>
__device__ __forceinline__ float row_factor(const Hidden<T> &h, const AdapterArgs &p, int a, int64_t t, bool has) {
    if (a < 0 || !has) return 0.0f;
    if (a >= p.adapters) return NAN;
    return power_of_row(h, t) * (p.scaling ? __ldcg(p.scaling + a) : 1.0f);
}
// base + f * product, 16 neighbouring columns of two rows; `old` is base (zeros without one).
template <typename T>
__device__ __forceinline__ void store_rows(T *const (&to)[2], const bool (&live)[2], const bool (&in)[2], const uint4 (&old)[2][2], const float (&acc)[8][4], const float (&f)[2], bool plain) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (!live[j / 2] || !in[j % 2]) continue;
        const uint32_t *o = reinterpret_cast<const uint32_t *>(&old[j / 2][j % 2]);
        uint32_t y[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const float2 v = Pair<T>::unpack(o[n]);
            y[n] = plain ? o[n] : Pair<T>::pack(fmaf(acc[2 * n][j], f[j / 2], v.x), fmaf(acc[2 * n + 1][j], f[j / 2], v.y));
        }
        *reinterpret_cast<uint4 *>(to[j / 2] + j % 2 * 8) = make_uint4(y[0], y[1], y[2], y[3]);
    }
}

// out[t] = base[t] + f * (h[t] times w) of a few tokens: a CTA an adapter and 512 columns, a warp 64 of them; w straight from global memory, KS steps
// of 16 ranks at once.
template <typename T, int KS>
__global__ void __launch_bounds__(128) adapter_expand_few_kernel(void *hidden, const T *__restrict__ w, const AdapterArgs p, const T *base, T *out) {
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
    __shared__ uint8_t lists[4][TILE];
    const Hidden<T> h(hidden, p.M, p.rank);
    const int64_t cb = ((int64_t)blockIdx.x * 4 + warp) * 64, col = cb + r * 8;
    const bool in[2] = {cb + 16 * c < p.cols, cb + 16 * c + 8 < p.cols};
    TileAdapters tile(p, 0, lists[warp]);
    bool waited = false;
    for (int i = blockIdx.y; i < tile.groups; i += p.slots) {
        tile.take(i);
        const int a = tile.adapter;
        if (a < 0 && base == out) continue;
        const bool has = a >= 0 && a < p.adapters;
        uint4 raw[KS][4];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = 16 * ks + 2 * c + k % 2 + k / 2 * 8;
                raw[ks][k] = load16_if(w + ((int64_t)(has ? a : 0) * p.rank + j) * p.cols + col, has && col < p.cols && j < p.rank);
            }
        if (!waited) pdl_wait();                  // (what comes before is the launch that makes the rank values; all that came before that is done)
        waited = true;
        for (int row0 = 0; row0 < tile.count; row0 += 16) {
            const bool live[2] = {row0 + r < tile.count, row0 + r + 8 < tile.count};
            const int64_t t[2] = {live[0] ? tile.list[row0 + r] : 0, live[1] ? tile.list[row0 + r + 8] : 0};
            uint4 old[2][2];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                old[j / 2][j % 2] = base && live[j / 2] && in[j % 2] ? __ldcg(reinterpret_cast<const uint4 *>(base + t[j / 2] * p.cols + cb + 16 * c + j % 2 * 8))
                                                                      : make_uint4(0, 0, 0, 0);
            const float f[2] = {row_factor(h, p, a, t[0], live[0]), row_factor(h, p, a, t[1], live[1])};
            float acc[8][4] = {};
            if (has) {
                constexpr int SOME = KS < 4 ? KS : 4;             // (steps at once, which registers hold)
#pragma unroll
                for (int k0 = 0; k0 < KS; k0 += SOME) {
                    uint32_t values[PARTS<T>][SOME][4];
                    load_rank_values<T, SOME>(h, p.rank, k0, t[0], t[1], live[0], live[1], c, values);
#pragma unroll
                    for (int ks = 0; ks < SOME; ++ks)
#pragma unroll
                        for (int n = 0; n < 8; ++n) {
                            const uint32_t b0 = column_pair(raw[k0 + ks][0], raw[k0 + ks][1], n), b1 = column_pair(raw[k0 + ks][2], raw[k0 + ks][3], n);
#pragma unroll
                            for (int part = 0; part < PARTS<T>; ++part) Pair<T>::mma(acc[n], values[part][ks], b0, b1);
                        }
                }
            }
            T *const to[2] = {out + t[0] * p.cols + cb + 16 * c, out + t[1] * p.cols + cb + 16 * c};
            store_rows<T>(to, live, in, old, acc, f, a < 0);
        }
    }
    if (!waited) pdl_wait();                      // a grid that was launched early is not done before the one in front of it
}

// The same of many tokens: 64 rows of one adapter, 16 a warp with their rank values in registers; blocks of 64 columns of w and of base go through
// a ring in shared memory.
template <typename T, int KS>
__global__ void __launch_bounds__(128, KS <= 4 ? 3 : 2) adapter_expand_kernel(void *hidden, const T *__restrict__ w, const AdapterArgs p, int64_t per_group, const T *base, T *out) {
    constexpr int W_BYTES = KS * 16 * 128, STAGE = W_BYTES + TILE * 128, STAGES = KS <= 4 ? 4 : 3;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint8_t lists[4][TILE];
    const uint32_t ring = smem_addr(smem);
    const Hidden<T> h(hidden, p.M, p.rank);
    pdl_launch_dependents();
    const int64_t t0 = (int64_t)blockIdx.x * TILE, begin = blockIdx.y * per_group, end = begin + per_group < p.cols ? begin + per_group : p.cols;

    TileAdapters tile(p, t0, lists[warp]);
    pdl_wait();                                   // (what comes before is the launch that makes the rank values, or one behind it)
    for (int i = blockIdx.z; i < tile.groups; i += p.slots) {
        tile.take(i);
        const int a = tile.adapter;
        if (a < 0 && base == out) continue;
        const bool has = a >= 0 && a < p.adapters;
        // a thread copies piece threadIdx % 8 of every 16th row of w and of base
        const int piece = threadIdx.x % 8, row0 = threadIdx.x / 8;
        const T *wrow = w + ((int64_t)(has ? a : 0) * p.rank + row0) * p.cols + piece * 8, *rows[4];
        const uint32_t wstep = (uint32_t)p.cols * 16;
        int bytes[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bytes[j] = row0 + 16 * j < tile.count ? 16 : 0;
            rows[j] = base + (t0 + (row0 + 16 * j < tile.count ? tile.list[row0 + 16 * j] : 0)) * p.cols + piece * 8;
        }
        auto copy_stage = [&](int64_t cb, int stage) {
            if (cb < end) {
                const bool in = cb + piece * 8 < p.cols;
                const uint32_t to = ring + stage * STAGE + row0 * 128;
                if (has) {
#pragma unroll
                    for (int j = 0; j < KS; ++j) {
                        const bool ok = in && row0 + 16 * j < p.rank;
                        copy16(to + j * 2048 + (piece ^ (row0 >> 1 & 3) << 1) * 16, wrow + (ok ? (int64_t)(wstep * j) + cb : 0), ok ? 16 : 0);
                    }
                }
                if (base) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) copy16(to + W_BYTES + j * 2048 + (piece ^ (row0 & 7)) * 16, rows[j] + cb, in ? bytes[j] : 0);
                }
            }
            copies_commit();
        };
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) copy_stage(begin + 64 * s, s);

        const int row = warp * 16 + r;
        const bool live[2] = {row < tile.count, row + 8 < tile.count};
        const int64_t t[2] = {t0 + (live[0] ? tile.list[row] : 0), t0 + (live[1] ? tile.list[row + 8] : 0)};
        uint32_t values[PARTS<T>][KS][4];
        load_rank_values<T, KS>(h, p.rank, 0, t[0], t[1], live[0] && has, live[1] && has, c, values);
        const float f[2] = {row_factor(h, p, a, t[0], live[0]), row_factor(h, p, a, t[1], live[1])};
        int stage = 0;
        const bool busy = warp * 16 < tile.count;
        // a lane's places in the stage: row 2 c of a step of 16 ranks, piece r; piece 2 c of its row of base; and its results
        const uint32_t w_place = c * 256 + (r ^ c << 1) * 16, base_place = W_BYTES + row * 128 + ((2 * c) ^ r) * 16;
        T *const to[2] = {out + t[0] * p.cols + 16 * c, out + t[1] * p.cols + 16 * c};
        for (int64_t cb = begin; cb < end; cb += 64) {
            copies_wait<STAGES - 2>();
            __syncthreads();
            copy_stage(cb + (STAGES - 1) * 64, stage == 0 ? STAGES - 1 : stage - 1);
            const uint32_t at = ring + stage * STAGE;
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            if (!busy) continue;
            float acc[8][4] = {};
            if (has) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    uint4 raw[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) raw[k] = load_shared16(at + w_place + ks * 2048 + k % 2 * 128 + k / 2 * 1024);
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        const uint32_t b0 = column_pair(raw[0], raw[1], n), b1 = column_pair(raw[2], raw[3], n);
#pragma unroll
                        for (int part = 0; part < PARTS<T>; ++part) Pair<T>::mma(acc[n], values[part][ks], b0, b1);
                    }
                }
            }
            uint4 old[2][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) old[j / 2][j % 2] = base ? load_shared16(at + (base_place ^ j % 2 * 16) + j / 2 * 1024) : make_uint4(0, 0, 0, 0);
            const bool in[2] = {cb + 16 * c < p.cols, cb + 16 * c + 8 < p.cols};
            T *const here[2] = {to[0] + cb, to[1] + cb};
            store_rows<T>(here, live, in, old, acc, f, a < 0);
        }
        copies_wait<0>();
        __syncthreads();
    }
}

// The same on tcgen05, for many tokens: 128 rows of one adapter (M) x blocks of 128 columns (N), reduced over the ranks of values and rests.  Rank values lie
// in tensor memory, a row a lane, their parts one after the other, rows of w MN-major in shared memory.  Eight warps bring w and base into a ring, one issues the MMAs (accumulators in turn), eight
// add the products to base in the ring, a row and half of its columns a lane, and write whole rows from there.
// Bound by the bytes of base and out: 8192 tokens, 14336 columns, rank 64, bf16: 85 us (mma.sync 133 with two parts; rank values in shared memory, a stage less, 104), 5.5 TB/s, on the 128
// SMs that there are CTAs for.
constexpr int EU_TILE = 128, EU_COLS = 128, EU_JOIN = 8, EU_COPY = 8, EU_THREADS = 32 * (EU_JOIN + EU_COPY + 1);
__device__ int g_adapter_status = 0;

template <int KS> struct ExpandShape {
    static constexpr int W_BLOCK = KS * 16 * 128, STAGE = 2 * W_BLOCK + EU_TILE * EU_COLS * 2, STAGES = KS <= 4 ? 4 : 3, SMEM = STAGES * STAGE + 1024;
};

// Rank values `ks` * 16 to + 16 of a row (ranks behind the last, and no row: zeros) as pairs of 16 bits of each part.
__device__ __forceinline__ void rank_step(const Hidden<__half> &h, int rank, int64_t t, bool live, int ks, uint32_t (&parts)[2][8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool ok = live && ks * 16 + i * 8 < rank;
        const int64_t at = ok ? t * rank + ks * 16 + i * 8 : 0;
        const uint4 u[2] = {load16_if(h.top + at, ok), load16_if(h.rest + at, ok)};
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            parts[part][4 * i] = u[part].x;
            parts[part][4 * i + 1] = u[part].y;
            parts[part][4 * i + 2] = u[part].z;
            parts[part][4 * i + 3] = u[part].w;
        }
    }
}
__device__ __forceinline__ void rank_step(const Hidden<__nv_bfloat16> &h, int rank, int64_t t, bool live, int ks, uint32_t (&parts)[3][8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool ok = live && ks * 16 + i * 4 < rank;
        const uint4 u = load16_if(h.sum + (ok ? t * rank + ks * 16 + i * 4 : 0), ok);
        const float2 v[2] = {make_float2(__uint_as_float(u.x), __uint_as_float(u.y)), make_float2(__uint_as_float(u.z), __uint_as_float(u.w))};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            uint32_t s[3];
            split<__nv_bfloat16>(v[k], s);
#pragma unroll
            for (int part = 0; part < 3; ++part) parts[part][2 * i + k] = s[part];
        }
    }
}

template <typename T, int KS>
__global__ void __launch_bounds__(EU_THREADS, 1) adapter_expand_umma_kernel(void *hidden, const T *__restrict__ w, const AdapterArgs p, int64_t per_group, const T *base, T *out) {
    using S = ExpandShape<KS>;
    constexpr bool F16 = __is_same(T, __half);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid / 32, 0), lane = tid % 32;
    extern __shared__ uint8_t raw_smem[];
    uint8_t *smem = raw_smem + ((1024u - (smem_addr(raw_smem) & 1023u)) & 1023u);      // the ring: [w | base]
    __shared__ __align__(16) int s_id[EU_TILE];
    __shared__ int s_leader[EU_TILE], s_count[4], s_abort;
    __shared__ uint32_t s_tmem;
    __shared__ uint8_t list[EU_TILE];
    __shared__ __align__(8) uint64_t full[S::STAGES], empty[S::STAGES], acc_full[2], acc_empty[2], values_full;
    volatile int *abort_flag = &s_abort;
    const Hidden<T> h(hidden, p.M, p.rank);
    const int64_t t0 = (int64_t)blockIdx.x * EU_TILE, begin = blockIdx.y * per_group, end = begin + per_group < p.cols ? begin + per_group : p.cols;
    const uint32_t ring = smem_addr(smem);

    if (tid == 0) {
        for (int i = 0; i < S::STAGES; ++i) {
            umma::mbar_init(&full[i], 33 * EU_COPY);             // (copies of each thread, and each warp)
            umma::mbar_init(&empty[i], EU_JOIN);
        }
        for (int i = 0; i < 2; ++i) {
            umma::mbar_init(&acc_full[i], 1);
            umma::mbar_init(&acc_empty[i], EU_JOIN);
        }
        umma::mbar_init(&values_full, EU_JOIN);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        umma::fence_proxy_async_smem();
    }
    if (warp == EU_JOIN + EU_COPY) umma::tmem_alloc(&s_tmem, 512);
    // the adapters of the tile, in the order of their first token
    const bool has = tid < EU_TILE && t0 + tid < p.M;
    const int id = has ? __ldcg(p.index + t0 + tid) : 0;
    bool first = false;
    if (warp < 4) {
        const unsigned there = __ballot_sync(0xffffffffu, has), like = __match_any_sync(0xffffffffu, id);
        first = has && !(like & there & ((1u << lane) - 1));
        s_id[tid] = id;
    }
    umma::tc_fence_before();
    __syncthreads();
    umma::tc_fence_after();
    pdl_launch_dependents();       // (not before the tensor memory is there: the launch behind may take as much of it, and waits for this one)
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    unsigned leaders = 0;
    if (warp < 4) {
        for (int j = 0; j < warp * 32; j += 4) {
            const int4 o = *reinterpret_cast<const int4 *>(s_id + j);
            if (o.x == id || o.y == id || o.z == id || o.w == id) first = false;
        }
        leaders = __ballot_sync(0xffffffffu, first);
        if (lane == 0) s_count[warp] = __popc(leaders);
    }
    __syncthreads();
    int groups = 0;
    for (int i = 0; i < 4; ++i) {
        if (i == warp && first) s_leader[groups + __popc(leaders & ((1u << lane) - 1))] = id;
        groups += s_count[i];
    }
    pdl_wait();                                   // (what comes before is the launch that makes the rank values, or one behind it)

    bool alive = true;                            // (after a failed wait the loops go on without work: the warps meet in them)
    int it = 0, turn = 0;                         // blocks of columns so far; adapters
    for (int pass = blockIdx.z; pass < groups; pass += p.slots) {
        __syncthreads();
        const int a = s_leader[pass];
        if (a < 0 && base == out) continue;
        unsigned mine = 0;
        if (warp < 4) {
            mine = __ballot_sync(0xffffffffu, has && id == a);
            if (lane == 0) s_count[warp] = __popc(mine);
        }
        __syncthreads();
        int count = 0;
        for (int i = 0; i < 4; ++i) {
            if (i == warp && (mine >> lane & 1)) list[count + __popc(mine & ((1u << lane) - 1))] = (uint8_t)tid;
            count += s_count[i];
        }
        __syncthreads();
        if (a < 0 || a >= p.adapters) {
            // rows without an adapter are base, or zeros; of one beyond the bank NaN
            const int pieces = (int)((end - begin) / 8);
            const uint32_t nan = Pair<T>::pack(NAN, NAN);
            for (int r = warp; r < count; r += EU_THREADS / 32)
                for (int i = lane; i < pieces; i += 32) {
                    const int64_t at = (t0 + list[r]) * p.cols + begin + i * 8;
                    uint4 v = make_uint4(nan, nan, nan, nan);
                    if (a < 0) v = base ? __ldcg(reinterpret_cast<const uint4 *>(base + at)) : make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4 *>(out + at) = v;
                }
            continue;
        }
        if (warp < EU_JOIN) {
            // ---- products and base; rows of the result ----
            const int quarter = warp % 4, half = warp / 4 * (EU_COLS / 2), row = quarter * 32 + lane;
            const bool live = row < count;
            const int64_t t = t0 + (live ? list[row] : 0);
            const float f = live ? power_of_row(h, t) * (p.scaling ? __ldcg(p.scaling + a) : 1.0f) : 0.0f;
            // the row's rank values into tensor memory, behind the two accumulators: [part][step] of 16 ranks in 8 columns (the adapter's before were last read for a block
            // whose sums this warp has waited for)
#pragma unroll 2
            for (int ks = warp / 4; ks < KS; ks += 2) {
                uint32_t parts[PARTS<T>][8];
                rank_step(h, p.rank, t, live, ks, parts);
#pragma unroll
                for (int part = 0; part < PARTS<T>; ++part) umma::tmem_st_32x32b_x8(tmem + ((uint32_t)(quarter * 32) << 16) + 2 * EU_COLS + (part * KS + ks) * 8, parts[part]);
            }
            umma::tmem_st_wait();
            umma::tc_fence_before();
            __syncwarp();
            if (lane == 0) umma::mbar_arrive(&values_full);
            // what the lane stores: piece `lane` % 8 of the half's rows lane / 8, 4 + lane / 8, ..
            const int stored = quarter * 32 + lane / 8, piece0 = half / 8 + lane % 8;
            T *to[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) to[j] = stored + 4 * j < count ? out + (t0 + list[stored + 4 * j]) * p.cols + piece0 * 8 : nullptr;
            for (int64_t cb = begin; cb < end; cb += EU_COLS, ++it) {
                const int slot = it % S::STAGES, acc = it & 1;
                uint8_t *tile = smem + slot * S::STAGE + 2 * S::W_BLOCK;
                alive = __all_sync(0xffffffffu, alive && umma::mbar_wait(&acc_full[acc], it >> 1 & 1, abort_flag, 11, &g_adapter_status) &&
                                                    umma::mbar_wait(&full[slot], it / S::STAGES & 1, abort_flag, 12, &g_adapter_status));
                const bool work = alive && quarter * 32 < count;
                if (work) {
                    umma::tc_fence_after();
                    uint8_t *own = tile + row * (EU_COLS * 2);
#pragma unroll
                    for (int c = 0; c < EU_COLS / 2; c += 32) {
                        uint4 old[4] = {};
                        if (base) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) old[k] = *reinterpret_cast<const uint4 *>(own + (((half + c) / 8 + k) ^ (row & 7)) * 16);
                        }
                        uint32_t r[32];
                        umma::tmem_ld_32x32b_x32(tmem + ((uint32_t)(quarter * 32) << 16) + acc * EU_COLS + half + c, r);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t *y = reinterpret_cast<uint32_t *>(&old[k]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 v = Pair<T>::unpack(y[e]);
                                y[e] = Pair<T>::pack(fmaf(__uint_as_float(r[8 * k + 2 * e]), f, v.x), fmaf(__uint_as_float(r[8 * k + 2 * e + 1]), f, v.y));
                            }
                            *reinterpret_cast<uint4 *>(own + (((half + c) / 8 + k) ^ (row & 7)) * 16) = old[k];
                        }
                    }
                    umma::tc_fence_before();
                }
                __syncwarp();
                if (lane == 0 && alive) umma::mbar_arrive(&acc_empty[acc]);
                if (work) {
                    const bool in = cb + piece0 * 8 < end;
                    uint4 v[8];                              // (all asked for before the first is stored)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int r = stored + 4 * j;
                        v[j] = *reinterpret_cast<const uint4 *>(tile + r * (EU_COLS * 2) + (piece0 ^ (r & 7)) * 16);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (to[j] && in) *reinterpret_cast<uint4 *>(to[j] + cb) = v[j];
                }
                __syncwarp();
                if (lane == 0 && alive) umma::mbar_arrive(&empty[slot]);
            }
        } else if (warp < EU_JOIN + EU_COPY) {
            // ---- copies ----
            const int me = tid - 32 * EU_JOIN;
            const int piece = me % 16;
            const T *rows[EU_TILE / 16];                     // this thread's piece of the rows of base
#pragma unroll
            for (int i = 0; i < EU_TILE / 16; ++i) rows[i] = base && me / 16 + 16 * i < count ? base + (t0 + list[me / 16 + 16 * i]) * p.cols + piece * 8 : nullptr;
            for (int64_t cb = begin; cb < end; cb += EU_COLS, ++it) {
                const int slot = it % S::STAGES;
                alive = alive && umma::mbar_wait(&empty[slot], (it / S::STAGES & 1) ^ 1, abort_flag, 13, &g_adapter_status);
                if (alive) {
                    const uint32_t to = ring + slot * S::STAGE;
                    const bool in = cb + piece * 8 < end;
                    // rows of w: blocks of 64 columns
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        const int rank = me / 16 + 16 * i;
                        const bool ok = in && rank < p.rank;
                        copy16(to + piece / 8 * S::W_BLOCK + rank * 128 + (piece % 8 ^ (rank & 7)) * 16, ok ? w + ((int64_t)a * p.rank + rank) * p.cols + cb + piece * 8 : w,
                               ok ? 16 : 0);
                    }
                    if (base) {
#pragma unroll
                        for (int i = 0; i < EU_TILE / 16; ++i) {
                            const int row = me / 16 + 16 * i;
                            if (rows[i]) copy16(to + 2 * S::W_BLOCK + row * (EU_COLS * 2) + (piece ^ (row & 7)) * 16, in ? rows[i] + cb : base, in ? 16 : 0);
                        }
                    }
                    copies_arrive(&full[slot]);
                }
                __syncwarp();
                if (lane == 0 && alive) umma::mbar_arrive(&full[slot]);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else {
            // ---- products ----
            const uint32_t idesc = umma::umma_idesc_f16(EU_COLS, !F16, false) | 1u << 16;      // (B MN-major)
            alive = __all_sync(0xffffffffu, alive && umma::mbar_wait(&values_full, turn & 1, abort_flag, 16, &g_adapter_status));
            umma::tc_fence_after();
            for (int64_t cb = begin; cb < end; cb += EU_COLS, ++it) {
                const int slot = it % S::STAGES, acc = it & 1;
                alive = __all_sync(0xffffffffu, alive && umma::mbar_wait(&acc_empty[acc], (it >> 1 & 1) ^ 1, abort_flag, 14, &g_adapter_status) &&
                                                    umma::mbar_wait(&full[slot], it / S::STAGES & 1, abort_flag, 15, &g_adapter_status));
                if (!alive) continue;
                umma::fence_proxy_async_smem();
                umma::tc_fence_after();
                const uint32_t at = ring + slot * S::STAGE;
#pragma unroll
                for (int part = PARTS<T> - 1; part >= 0; --part)          // (the smallest first: each MMA truncates what it adds to)
#pragma unroll
                    for (int k = 0; k < KS; ++k)
                        umma::umma_f16_ts(tmem + acc * EU_COLS, tmem + 2 * EU_COLS + (part * KS + k) * 8, umma::umma_smem_desc_mn(at + k * 2048, S::W_BLOCK), idesc,
                                          part != PARTS<T> - 1 || k != 0 ? 1u : 0u);
                umma::umma_commit(&acc_full[acc]);
            }
        }
        ++turn;
    }
    __syncthreads();
    umma::tc_fence_after();
    if (warp == EU_JOIN + EU_COPY) umma::tmem_dealloc(tmem, 512);
}

// ---- outer ---------------------------------------------------------------------------------------------------------------

constexpr int OUTER_LIST = 2048, OUTER_STEP = 32, OUTER_WINDOW = 1024;      // tokens of a list, of a stage; words of 32 tokens looked at together

// Which tokens of the window of 32 * WINDOW tokens from word w0 on are adapter a's (s_bits), and how many of them come before each word's (s_before);
// returns how many there are.  Made by WARPS warps, which meet at `barrier`.
template <int WARPS, int WINDOW, typename Barrier>
__device__ __forceinline__ int mark_tokens(const AdapterArgs &p, int a, int w0, uint32_t *s_bits, int *s_before, int *s_count, Barrier barrier) {
    constexpr int OWN = WINDOW / (32 * WARPS);                   // words of a thread
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, words = (int)((p.M + 31) / 32);
    barrier();
    for (int w = warp; w < WINDOW && w0 + w < words; w += 8 * WARPS) {
        int id[8];                                               // (all asked for before the first is looked at)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t t = (int64_t)(w0 + w + k * WARPS) * 32 + lane;
            id[k] = t < p.M ? __ldcg(p.index + t) : -1;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t bits = __ballot_sync(0xffffffffu, id[k] == a);
            if (lane == 0 && w + k * WARPS < WINDOW) s_bits[w + k * WARPS] = bits;
        }
    }
    barrier();
    int mine = 0;
#pragma unroll
    for (int k = 0; k < OWN; ++k) mine += w0 + (int)threadIdx.x * OWN + k < words ? __popc(s_bits[threadIdx.x * OWN + k]) : 0;
    int sum = mine;
    for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += o;
    }
    if (lane == 31) s_count[warp] = sum;
    barrier();
    int before = sum - mine, all = 0;
    for (int k = 0; k < WARPS; ++k) {
        before += k < warp ? s_count[k] : 0;
        all += s_count[k];
    }
#pragma unroll
    for (int k = 0; k < OWN; ++k) {
        const int w = threadIdx.x * OWN + k;
        s_before[w] = before;
        before += w0 + w < words ? __popc(s_bits[w]) : 0;
    }
    return all;
}
// Tokens `skip` to skip + n of the marked ones.  A lane a token.
template <int WARPS, int WINDOW>
__device__ __forceinline__ void list_tokens(const AdapterArgs &p, int w0, int skip, int n, const uint32_t *s_bits, const int *s_before, int *list) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, words = (int)((p.M + 31) / 32);
#pragma unroll 4
    for (int w = warp; w < WINDOW && w0 + w < words; w += WARPS) {
        const uint32_t bits = s_bits[w];
        const int place = s_before[w] + __popc(bits & ((1u << lane) - 1)) - skip;
        if ((bits >> lane & 1) && place >= 0 && place < n) list[place] = (w0 + w) * 32 + lane;
    }
}
// The end of outer: the CTAs of a cluster (along z) have sums [ranks][SUM_ROW] of 256 columns; each adds up its share of them and writes it.
constexpr int SUM_ROW = 260;             // (a row of sums, padded: eight rows meet in four banks otherwise)
template <typename T, int THREADS, int RANKS>
__device__ __forceinline__ void join_sums(float *sums, const AdapterArgs &p, int a, int rank0, int64_t col0, T *dw) {
    const cg::cluster_group cluster = cg::this_cluster();
    const int parts = gridDim.z, mine = blockIdx.z;
    for (int i = mine * THREADS + threadIdx.x; i < RANKS * 32; i += parts * THREADS) {        // eight columns of a rank
        const int rank = rank0 + i / 32;
        const int64_t at = col0 + i % 32 * 8;
        if (rank >= p.rank || at >= p.cols) continue;
        float4 u[8][2];                                          // (all asked for before the first is added)
#pragma unroll
        for (int o = 0; o < 8; ++o) {
            const float4 *from = reinterpret_cast<const float4 *>(cluster.map_shared_rank(sums, o < parts ? o : 0) + i / 32 * SUM_ROW + i % 32 * 8);
            if (o < parts) {
                u[o][0] = from[0];
                u[o][1] = from[1];
            }
        }
        float4 s0 = u[0][0], s1 = u[0][1];
#pragma unroll
        for (int o = 1; o < 8; ++o)
            if (o < parts) {
                s0.x += u[o][0].x; s0.y += u[o][0].y; s0.z += u[o][0].z; s0.w += u[o][0].w;
                s1.x += u[o][1].x; s1.y += u[o][1].y; s1.z += u[o][1].z; s1.w += u[o][1].w;
            }
        *reinterpret_cast<uint4 *>(dw + ((int64_t)a * p.rank + rank) * p.cols + at) =
            make_uint4(Pair<T>::pack(s0.x, s0.y), Pair<T>::pack(s0.z, s0.w), Pair<T>::pack(s1.x, s1.y), Pair<T>::pack(s1.z, s1.w));
    }
}
// RB blocks of 16 ranks a warp, RG groups of four warps with ranks of their own.
template <int RB, int RG, int PARTS> struct OuterShape {
    static constexpr int WARPS = 4 * RG, THREADS = 32 * WARPS;
    static constexpr int RANKS = 16 * RB * RG, ROW = RANKS * 2;               // bytes of a part of a token's rank values
    static constexpr int STAGE = OUTER_STEP * (512 + 2 * ROW), STAGES = RG == 1 ? 4 : 3;
    static constexpr int SPLIT = STAGE * STAGES, RING = SPLIT + (PARTS == 3 ? OUTER_STEP * 3 * ROW : 0);       // (bf16: the parts of the stage at work, behind the ring)
    static constexpr int SUMS = RANKS * SUM_ROW * 4, SMEM = RING > SUMS ? RING : SUMS;
    static __device__ __forceinline__ int swizzle(int token) { return ROW >= 128 ? token & 7 : ROW == 64 ? token >> 1 & 3 : token >> 2 & 1; }
};

// dw[a][rank0 .. + RANKS][256 columns] = f_a * sum over the adapter's tokens of h[t] x[t]^T.  The CTAs of a cluster (blockIdx.z) take equal shares of
// the tokens and add their sums through each other's shared memory.  Rows of x and of the rank values go through a ring, 32 tokens a stage.
// (For few tokens and ranks up to 16; 64 ranks in the registers of one warp would leave eight warps an SM.  The copies' issue, the barriers of a stage and the MMAs take turns: 8192 tokens,
// 14336 columns, rank 16, with shrink of 64 columns in front, 69 us of bf16, whose fp32 rank values are split a stage at a time, 70 of fp16.)
template <typename T, int RB, int RG>
__global__ void __launch_bounds__(128 * RG, RG == 2 ? 2 : 3) adapter_outer_kernel(void *hidden, const T *__restrict__ x, const AdapterArgs p, T *dw) {
    using S = OuterShape<RB, RG, PARTS<T>>;
    constexpr bool F16 = __is_same(T, __half);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32, r = lane / 4, c = lane % 4, wc = warp % 4, wr = warp / 4;
    const int rank_blocks = (p.rank + S::RANKS - 1) / S::RANKS, a = blockIdx.y / rank_blocks, rank0 = blockIdx.y % rank_blocks * S::RANKS;
    const int64_t col0 = (int64_t)blockIdx.x * 256;
    extern __shared__ __align__(128) uint8_t smem[];
    float *sums = reinterpret_cast<float *>(smem);               // [RANKS][SUM_ROW], at the end
    const uint32_t ring = smem_addr(smem);
    const Hidden<T> h(hidden, p.M, p.rank);
    __shared__ int list[OUTER_LIST + OUTER_STEP], s_count[S::WARPS];
    __shared__ uint32_t s_bits[OUTER_WINDOW];                    // which tokens of the window are the adapter's
    __shared__ int s_before[OUTER_WINDOW];                       // and how many of them come before each word's
    __shared__ float s_back[OUTER_LIST], s_big[S::WARPS];

    if (!p.behind) pdl_wait();
    pdl_launch_dependents();
    const int words = (int)((p.M + 31) / 32);
    auto mark = [&](int w0) { return mark_tokens<S::WARPS, OUTER_WINDOW>(p, a, w0, s_bits, s_before, s_count, [] { __syncthreads(); }); };
    int in_window = mark(0), all = in_window;
    for (int w0 = OUTER_WINDOW; w0 < words; w0 += OUTER_WINDOW) all += mark(w0);
    if (words > OUTER_WINDOW) in_window = mark(0);
    if (p.behind) pdl_wait();                                    // (the rank values are made by one of the launches before)
    const int share = (all + gridDim.z - 1) / gridDim.z, lo = blockIdx.z * share, hi = lo + share < all ? lo + share : all;

    // this thread's piece of a row of x (columns behind the last: zeros), and bytes of a row
    const int x_bytes = col0 + lane * 8 < p.cols ? 16 : 0;
    const uint8_t *xs0 = (const uint8_t *)(x + (x_bytes ? col0 + lane * 8 : 0));
    const uint32_t x_row = (uint32_t)p.cols * 2, h_row = (uint32_t)p.rank * (F16 ? 2 : 4), x_to = warp * 512 + (lane ^ (warp >> 1 & 3) << 1) * 16;
    // and its pieces of the rank values: 2 * ROW bytes a token, of both parts or of fp32
    constexpr int PIECES = S::ROW / 16, HJ = OUTER_STEP * PIECES * 2 / S::THREADS;
    const uint8_t *h_from[HJ];
    uint32_t h_to[HJ];
    int h_token[HJ], h_bytes[HJ];
#pragma unroll
    for (int j = 0; j < HJ; ++j) {
        const int i = threadIdx.x + S::THREADS * j;
        if constexpr (F16) {
            const int part = i / (OUTER_STEP * PIECES), token = i / PIECES % OUTER_STEP, piece = i % PIECES;
            h_token[j] = token;
            h_bytes[j] = rank0 + piece * 8 < p.rank ? 16 : 0;
            h_from[j] = (const uint8_t *)((part ? h.rest : h.top) + (h_bytes[j] ? rank0 + piece * 8 : 0));
            h_to[j] = OUTER_STEP * (512 + part * S::ROW) + token * S::ROW + (piece ^ S::swizzle(token)) * 16;
        } else {
            const int token = i / (2 * PIECES), piece = i % (2 * PIECES);
            h_token[j] = token;
            h_bytes[j] = rank0 + piece * 4 < p.rank ? 16 : 0;
            h_from[j] = (const uint8_t *)(h.sum + (h_bytes[j] ? rank0 + piece * 4 : 0));
            h_to[j] = OUTER_STEP * 512 + token * 2 * S::ROW + piece * 16;
        }
    }
    // a lane's places in the stage: token 2 c, piece r of its warp's columns; and rows of rank values for ldmatrix
    const uint32_t x_place = c * 1024 + wc * 128 + (r ^ c << 1) * 16;
    uint32_t h_place[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
        h_place[rb] = (lane % 8 + lane / 16 * 8) * S::ROW + (((wr * RB + rb) * 2 + lane / 8 % 2) ^ S::swizzle(lane % 8)) * 16;
    float acc[RB][8][4] = {};
    float big = 0.0f;                                            // fp16: the sums are of h / big, the largest power of two of a row so far: what is lost of a row is less
                                                                 // than 2^-38 of the largest one's values
    int window = 0, passed = 0;                                  // the marked window's first word, and the adapter's tokens in front of it
    for (int from = lo, n; from < hi; from += n) {
        while (passed + in_window <= from && window + OUTER_WINDOW < words) {
            passed += in_window;
            window += OUTER_WINDOW;
            in_window = mark(window);
        }
        if (passed + in_window <= from) break;                   // (an index that changes under the call)
        n = passed + in_window < hi ? passed + in_window - from : hi - from;      // (of one window)
        n = n < OUTER_LIST ? n : OUTER_LIST;
        __syncthreads();
        list_tokens<S::WARPS, OUTER_WINDOW>(p, window, from - passed, n, s_bits, s_before, list);
        __syncthreads();
        if (threadIdx.x < OUTER_STEP) list[n + threadIdx.x] = list[0];      // (the last stage's places behind the last token)
        __syncthreads();
        auto copy_stage = [&](int first, int stage) {
            if (first < n) {
                const uint32_t to = ring + stage * S::STAGE;
                // 32 rows of 32 pieces of x: a warp a row.  (Behind the last token a row is the first one's; its rank values are zeros.)
#pragma unroll
                for (int j = 0; j < OUTER_STEP / S::WARPS; ++j)
                    copy16(to + (x_to ^ (S::WARPS * j / 2 & 3) * 32) + S::WARPS * j * 512, xs0 + (uint64_t)(uint32_t)list[first + warp + S::WARPS * j] * x_row, x_bytes);
#pragma unroll
                for (int j = 0; j < HJ; ++j)
                    copy16(to + h_to[j], h_from[j] + (uint64_t)(uint32_t)list[first + h_token[j]] * h_row, first + h_token[j] < n ? h_bytes[j] : 0);
            }
            copies_commit();
        };
#pragma unroll
        for (int s = 0; s < S::STAGES - 1; ++s) copy_stage(s * OUTER_STEP, s);
        if constexpr (F16) {
            // powers of two of the rows, relative to the largest
            float most = 0.0f;
            for (int j = threadIdx.x; j < n; j += S::THREADS) {
                s_back[j] = __ldcg(h.back + list[j]);
                most = fmaxf(most, s_back[j]);
            }
            for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
            if (lane == 0) s_big[warp] = most;
            __syncthreads();
            most = big;
            for (int j = 0; j < S::WARPS; ++j) most = fmaxf(most, s_big[j]);
            if (big > 0.0f && most > big) {
                const float down = big / most;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int k = 0; k < 4; ++k) acc[rb][j][k] *= down;
            }
            big = most;
            for (int j = threadIdx.x; j < n; j += S::THREADS) s_back[j] /= big;
            // (the barrier of the first stage lies between this and its use)
        }
        int stage = 0;
        for (int first = 0; first < n; first += OUTER_STEP) {
            copies_wait<S::STAGES - 2>();
            __syncthreads();
            // (copies take about 1000 cycles of a stage to issue: of the two warps that share a quarter of the SM one makes its own before, one after its MMAs)
            const int refill = stage == 0 ? S::STAGES - 1 : stage - 1;
            if (wr == 0) copy_stage(first + (S::STAGES - 1) * OUTER_STEP, refill);
            const uint32_t place = ring + stage * S::STAGE, h_at = F16 ? place + OUTER_STEP * 512 : ring + S::SPLIT;
            if constexpr (!F16) {
                // the stage's rank values in parts (which all warps are done with since the barrier above)
                for (int i = threadIdx.x; i < OUTER_STEP * PIECES; i += S::THREADS) {
                    const int token = i / PIECES, piece = i % PIECES;
                    const float4 *from = reinterpret_cast<const float4 *>(smem + stage * S::STAGE + OUTER_STEP * 512 + token * 2 * S::ROW + piece * 32);
                    uint4 parts[3];
                    split8<T>(from[0], from[1], parts);
#pragma unroll
                    for (int part = 0; part < 3; ++part)
                        *reinterpret_cast<uint4 *>(smem + S::SPLIT + (part * OUTER_STEP + token) * S::ROW + (piece ^ S::swizzle(token)) * 16) = parts[part];
                }
                __syncthreads();
            }
            stage = stage + 1 == S::STAGES ? 0 : stage + 1;
#pragma unroll
            for (int step = 0; step < OUTER_STEP / 16; ++step) {
                if (first + step * 16 >= n || col0 + wc * 64 >= p.cols) break;
                uint4 raw[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) raw[k] = load_shared16(place + x_place + step * 8192 + k % 2 * 512 + k / 2 * 4096);
                uint32_t b[8][2];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    b[j][0] = column_pair(raw[0], raw[1], j);
                    b[j][1] = column_pair(raw[2], raw[3], j);
                }
                __half2 scale[2], more[2];                      // (as two factors: powers below 2^-24 as well)
                if constexpr (F16) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int i = first + step * 16 + 2 * c + 8 * k;
                        const float f0 = i < n ? s_back[i] : 0.0f, f1 = i + 1 < n ? s_back[i + 1] : 0.0f;
                        scale[k] = __floats2half2_rn(fmaxf(f0, 0x1p-24f), fmaxf(f1, 0x1p-24f));
                        more[k] = __floats2half2_rn(fminf(f0 * 0x1p24f, 1.0f), fminf(f1 * 0x1p24f, 1.0f));
                    }
                }
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    uint32_t ha[PARTS<T>][4];
#pragma unroll
                    for (int part = 0; part < PARTS<T>; ++part) {
                        load_matrices_transposed(h_at + h_place[rb] + (part * OUTER_STEP + step * 16) * S::ROW, ha[part]);
                        if constexpr (F16) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const __half2 y = __hmul2(__hmul2(*reinterpret_cast<const __half2 *>(&ha[part][k]), scale[k / 2]), more[k / 2]);
                                ha[part][k] = *reinterpret_cast<const uint32_t *>(&y);
                            }
                        }
                    }
                    // (the parts' products of 16 tokens, from the smallest on, then added in fp32: an MMA truncates what it adds to, a bias of 2^-24 of the sum each time)
#pragma unroll
                    for (int j0 = 0; j0 < 8; j0 += 4) {
                        float some[4][4];
#pragma unroll
                        for (int part = PARTS<T> - 1; part >= 0; --part)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (part == PARTS<T> - 1) Pair<T>::mma_new(some[j], ha[part], b[j0 + j][0], b[j0 + j][1]);
                                else Pair<T>::mma(some[j], ha[part], b[j0 + j][0], b[j0 + j][1]);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[rb][j0 + j][e] += some[j][e];
                    }
                }
            }
            if (wr != 0) copy_stage(first + (S::STAGES - 1) * OUTER_STEP, refill);
        }
        copies_wait<0>();
    }

    // sums of this CTA, in 16 neighbouring columns a lane; then those of the cluster
    const float f = (F16 ? big : 1.0f) * (p.scaling ? __ldcg(p.scaling + a) : 1.0f);
    __syncthreads();
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) sums[((wr * RB + rb) * 16 + r + k / 2 * 8) * SUM_ROW + wc * 64 + c * 16 + k % 2 * 8 + j] = acc[rb][j][k] * f;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    join_sums<T, S::THREADS, S::RANKS>(sums, p, a, rank0, col0, dw);
    cluster.sync();                                              // a CTA's sums stay until the others have read them
}

// The same on tcgen05, for adapters of many tokens: 64 ranks x 256 columns a CTA, reduced over tokens, 32 a stage.  Rows of x and of the rank values keep
// the order in which memory holds them, which is the MN-major form of both operands (blocks of 64 elements by 32 tokens, 128-byte swizzle).  Values and
// rests of 64 ranks are the two halves of the M dimension, so that one MMA multiplies both; their sums meet at the end.  Eight warps fill the ring with
// 16-byte cp.async of rows that a list names, one warp issues the MMAs; for fp16 two warps between them bring the rows' powers of two into the rank
// values.  The third part of bf16 takes MMAs of its own, with zeros as the other half.  (A warp with copies in flight does nothing else: a proxy fence, which the MMAs need between
// the copies and themselves, waits for all that its own thread has in flight: 86 us instead of 76.)  Bound by the rows of x and the rank values, which every 256 columns read
// again: 8192 tokens, 14336 columns, rank 64, on the 112 SMs that there are CTAs for: bf16 80 us (in two parts 73, mma.sync 129; fp32 rank values split on the way by one pair of warps
// 113, by three 93, into tensor memory 101; sixteen copying warps: the same, and 2 us more to begin).
// Stages go to two sets of sums in turn: an MMA truncates what it adds up, a bias toward zero that grows with the number of MMAs into one sum.  (4096 tokens an adapter, 14336 columns:
// bf16 gradients differ from the exact ones' roundings by 1.0e-4 of their 2-norm, with one set and the third part in the values' half by 2.2e-4, fp32 torch's by 0.7e-4.)
constexpr int OU_LIST = 1024, OU_WINDOW = 512;
template <typename T> struct OuterUmma {
    static constexpr int BLOCK = OUTER_STEP * 128, A = PARTS<T> * BLOCK, B = 4 * BLOCK, STAGE = A + B, STAGES = PARTS<T> == 2 ? 8 : 7, THREADS = 352;
    static constexpr int RING = PARTS<T> == 3 ? BLOCK : 0;                                                      // bf16: a block of zeros in front of the ring
    // All of an SM's tensor memory is taken, so no other kernel that wants some may fit beside: of two clusters that each hold one SM's and want another's both would wait for good.  (The smallest
    // such cluster kernel has 16 KB of shared memory; of 228 KB these and what is declared in the kernel leave less.)
    static constexpr int SMEM = 210 * 1024;
    static_assert(RING + STAGES * STAGE + 1024 <= SMEM, "zeros, the ring and its alignment");
    static_assert(64 * SUM_ROW * 4 <= STAGES * STAGE, "the sums take the ring's place");
};
template <typename T>
__global__ void __launch_bounds__(OuterUmma<T>::THREADS, 1) adapter_outer_umma_kernel(void *hidden, const T *__restrict__ x, const AdapterArgs p, T *dw) {
    using S = OuterUmma<T>;
    constexpr bool F16 = __is_same(T, __half);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const int rank_blocks = (p.rank + 63) / 64, a = blockIdx.y / rank_blocks, rank0 = blockIdx.y % rank_blocks * 64;
    const int64_t col0 = (int64_t)blockIdx.x * 256;
    extern __shared__ uint8_t raw_smem[];
    uint8_t *smem = raw_smem + ((1024u - (smem_addr(raw_smem) & 1023u)) & 1023u);      // bf16: zeros; [STAGES][parts of the rank values | 4 blocks of columns][tokens][128 B]
    float *sums = reinterpret_cast<float *>(smem);                                      // [64][SUM_ROW], at the end
    __shared__ int list[OU_LIST + OUTER_STEP], s_before[OU_WINDOW], s_count[8], s_end[S::STAGES], s_abort;
    __shared__ uint32_t s_bits[OU_WINDOW], s_tmem;
    __shared__ float s_back[F16 ? OU_LIST : 1], s_big[8], s_scale[F16 ? S::STAGES : 1][OUTER_STEP];
    __shared__ __align__(8) uint64_t full[S::STAGES], scaled[S::STAGES], empty[S::STAGES], done;
    volatile int *abort_flag = &s_abort;
    const Hidden<T> h(hidden, p.M, p.rank);

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::STAGES; ++i) {
            umma::mbar_init(&full[i], 256 + 8);                  // (copies of each thread, and each warp)
            umma::mbar_init(&scaled[i], 2);
            umma::mbar_init(&empty[i], 1);
            s_end[i] = 0;
        }
        umma::mbar_init(&done, 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        umma::fence_proxy_async_smem();
    }
    if constexpr (PARTS<T> == 3) {
        for (int i = threadIdx.x; i < S::BLOCK / 16; i += S::THREADS) reinterpret_cast<uint4 *>(smem)[i] = make_uint4(0, 0, 0, 0);
        umma::fence_proxy_async_smem();
    }
    if (warp == 8) umma::tmem_alloc(&s_tmem, 512);
    umma::tc_fence_before();
    __syncthreads();
    umma::tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    if (!p.behind) pdl_wait();
    pdl_launch_dependents();       // (not before the tensor memory is there: the launch behind may take as much of it, and waits for this one)

    int stages = 0;                // made in all
    float f = 0.0f;                // what the sums are multiplied by
    if (warp == 8) {
        // ---- products ----
        if (p.behind) pdl_wait();
        const uint32_t idesc = umma::umma_idesc_f16(256, !F16, true) | 1u << 16;      // (B MN-major as well)
        const uint32_t zeros = smem_addr(smem), ring = zeros + S::RING;
        for (;; ++stages) {
            const int slot = stages % S::STAGES;
            if (!__all_sync(0xffffffffu, umma::mbar_wait(F16 ? &scaled[slot] : &full[slot], stages / S::STAGES & 1, abort_flag, 1, &g_adapter_status))) break;
            if (*(volatile int *)&s_end[slot]) {
                umma::umma_commit(&done);
                break;
            }
            umma::fence_proxy_async_smem();
            umma::tc_fence_after();
            const uint32_t sum = tmem + (stages & 1) * 256;
            const uint32_t at = ring + slot * S::STAGE;
#pragma unroll
            for (int k = 0; k < OUTER_STEP / 16; ++k) {
                const uint64_t columns = umma::umma_smem_desc_mn(at + S::A + k * 2048, S::BLOCK);
                umma::umma_f16_ss(sum, umma::umma_smem_desc_mn(at + k * 2048, S::BLOCK), columns, idesc, (stages / 2 | k) != 0 ? 1u : 0u);
                // (the third part to the rests' half, below a block of zeros)
                if constexpr (!F16)
                    umma::umma_f16_ss(sum, umma::umma_smem_desc_mn(zeros + k * 2048, at + 2 * S::BLOCK - zeros), columns, idesc, 1u);
            }
            umma::umma_commit(&empty[slot]);
        }
    } else if (warp > 8) {
        // ---- fp16: rank values times their row's power of two ----
        if (p.behind) pdl_wait();
        if constexpr (F16)
            for (;; ++stages) {
                const int slot = stages % S::STAGES;
                if (!__all_sync(0xffffffffu, umma::mbar_wait(&full[slot], stages / S::STAGES & 1, abort_flag, 5, &g_adapter_status))) break;
                const bool end = *(volatile int *)&s_end[slot];
                if (!end) {
#pragma unroll
                    for (int i = 0; i < S::A / 16 / 64; ++i) {
                        const int at = (warp - 9) * 32 + lane + i * 64;      // of 16 bytes, eight a row
                        const float f = s_scale[slot][at / 8 % OUTER_STEP];
                        const __half2 scale = __float2half2_rn(fmaxf(f, 0x1p-24f)), more = __float2half2_rn(fminf(f * 0x1p24f, 1.0f));      // (powers below 2^-24 as well)
                        uint4 *own = reinterpret_cast<uint4 *>(smem + S::RING + slot * S::STAGE) + at, v = *own;
                        __half2 *y = reinterpret_cast<__half2 *>(&v);
#pragma unroll
                        for (int k = 0; k < 4; ++k) y[k] = __hmul2(__hmul2(y[k], scale), more);
                        *own = v;
                    }
                    umma::fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) umma::mbar_arrive(&scaled[slot]);
                if (end) break;
            }
    } else {
        // ---- copies ----
        const auto meet = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
        const int words = (int)((p.M + 31) / 32);
        auto mark = [&](int w0) { return mark_tokens<8, OU_WINDOW>(p, a, w0, s_bits, s_before, s_count, meet); };
        int in_window = mark(0), all = in_window;
        for (int w0 = OU_WINDOW; w0 < words; w0 += OU_WINDOW) all += mark(w0);
        if (words > OU_WINDOW) in_window = mark(0);
        if (p.behind) pdl_wait();                                // (the rank values are made by one of the launches before)
        const int share = (all + gridDim.z - 1) / gridDim.z, lo = blockIdx.z * share, hi = lo + share < all ? lo + share : all;
        float big = 1.0f;                                        // fp16: the sums are of h / big, the largest power of two of a row
        if constexpr (F16) {
            big = 0.0f;
#pragma unroll 4
            for (int w = warp; w < words; w += 8) {
                const int64_t t = (int64_t)w * 32 + lane;
                const int id = t < p.M ? __ldcg(p.index + t) : -1;
                const float back = t < p.M ? __ldcg(h.back + t) : 0.0f;      // (of a row without an adapter: anything)
                if (id == a) big = fmaxf(big, back);
            }
            for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
            if (lane == 0) s_big[warp] = big;
            meet();
            for (int i = 0; i < 8; ++i) big = fmaxf(big, s_big[i]);
        }
        f = big * (p.scaling ? __ldcg(p.scaling + a) : 1.0f);

        // this thread's pieces: of rows warp, warp + 8, .. of x piece `lane`; of row threadIdx / 8 of the rank values' parts piece threadIdx % 8
        const int x_bytes = col0 + lane * 8 < p.cols ? 16 : 0, token = threadIdx.x / 8, piece = threadIdx.x % 8, h_bytes = rank0 + piece * 8 < p.rank ? 16 : 0;
        const uint8_t *xs0 = (const uint8_t *)(x + (x_bytes ? col0 + lane * 8 : 0));
        const T *h0;
        if constexpr (F16) h0 = h.top;
        else h0 = h.parts;
        h0 += h_bytes ? rank0 + piece * 8 : 0;
        const int64_t part_size = p.M * p.rank;
        const uint32_t x_row = (uint32_t)p.cols * 2, h_row = (uint32_t)p.rank * 2, ring = smem_addr(smem) + S::RING;
        const uint32_t x_to = S::A + lane / 8 * S::BLOCK + warp * 128 + (lane % 8 ^ warp) * 16, h_to = token * 128 + (piece ^ (token & 7)) * 16;
        bool alive = true;                                       // (after a failed wait the loops go on without copies: the warps meet in them)
        int window = 0, passed = 0;
        for (int from = lo, n; from < hi; from += n) {
            while (passed + in_window <= from && window + OU_WINDOW < words) {
                passed += in_window;
                window += OU_WINDOW;
                in_window = mark(window);
            }
            if (passed + in_window <= from) break;               // (an index that changes under the call)
            n = passed + in_window < hi ? passed + in_window - from : hi - from;      // (of one window)
            n = n < OU_LIST ? n : OU_LIST;
            meet();
            list_tokens<8, OU_WINDOW>(p, window, from - passed, n, s_bits, s_before, list);
            meet();
            if constexpr (F16) {
                for (int j = threadIdx.x; j < n; j += 256) s_back[j] = __ldcg(h.back + list[j]) / big;
                meet();
            }
            const int count = (n + OUTER_STEP - 1) / OUTER_STEP;
            for (int i = 0; i < count; ++i, ++stages) {
                const int slot = stages % S::STAGES, first = i * OUTER_STEP;
                alive = alive && umma::mbar_wait(&empty[slot], (stages / S::STAGES & 1) ^ 1, abort_flag, 2, &g_adapter_status);
                if (alive) {
                    const uint32_t to = ring + slot * S::STAGE;
#pragma unroll
                    for (int j = 0; j < OUTER_STEP / 8; ++j) {
                        const int at = first + warp + 8 * j;
                        copy16(to + x_to + j * 1024, xs0 + (at < n ? (uint64_t)(uint32_t)list[at] * x_row : 0), at < n ? x_bytes : 0);
                    }
                    const int at = first + token;
                    const uint64_t row = at < n ? (uint64_t)(uint32_t)list[at] * h_row : 0;
#pragma unroll
                    for (int part = 0; part < PARTS<T>; ++part)
                        copy16(to + h_to + part * S::BLOCK, (const uint8_t *)(h0 + part * part_size) + row, at < n ? h_bytes : 0);
                    if constexpr (F16)
                        if (piece == 0) s_scale[slot][token] = at < n ? s_back[at] : 0.0f;
                    copies_arrive(&full[slot]);
                }
                __syncwarp();
                if (lane == 0 && alive) umma::mbar_arrive(&full[slot]);
            }
        }
        // one more stage, without tokens: the end
        const int slot = stages % S::STAGES;
        alive = alive && umma::mbar_wait(&empty[slot], (stages / S::STAGES & 1) ^ 1, abort_flag, 3, &g_adapter_status);
        if (threadIdx.x == 0) *(volatile int *)&s_end[slot] = 1;
        if (alive) copies_arrive(&full[slot]);
        __syncwarp();
        if (lane == 0 && alive) umma::mbar_arrive(&full[slot]);
        asm volatile("cp.async.wait_all;" ::: "memory");
        // ---- sums of this CTA: tensor memory's lanes 0 to 63 are the values' ranks, 64 to 127 the rests' ----
        if (warp < 4) alive = __all_sync(0xffffffffu, umma::mbar_wait(&done, 0, abort_flag, 4, &g_adapter_status));
        umma::tc_fence_after();
#pragma unroll
        for (int part = 1; part >= 0; --part) {
            if (warp < 4 && warp / 2 == part) {
                float *row = sums + (warp % 2 * 32 + lane) * SUM_ROW;
                for (int cb = 0; cb < 256; cb += 32) {
                    uint32_t r[32] = {};
                    if (alive && stages) umma::tmem_ld_32x32b_x32(tmem + ((uint32_t)(warp * 32) << 16) + cb, r);
                    if (alive && stages > 1) {
                        uint32_t odd[32];
                        umma::tmem_ld_32x32b_x32(tmem + ((uint32_t)(warp * 32) << 16) + 256 + cb, odd);
#pragma unroll
                        for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) + __uint_as_float(odd[k]));
                    }
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        float4 v = make_float4(__uint_as_float(r[k]), __uint_as_float(r[k + 1]), __uint_as_float(r[k + 2]), __uint_as_float(r[k + 3]));
                        float4 *to = reinterpret_cast<float4 *>(row + cb + k);
                        if (part == 0) {
                            const float4 rest = *to;
                            v = make_float4((v.x + rest.x) * f, (v.y + rest.y) * f, (v.z + rest.z) * f, (v.w + rest.w) * f);
                        }
                        *to = v;
                    }
                }
            }
            meet();
        }
        umma::tc_fence_before();
    }
    __syncwarp();
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (*abort_flag == 0) join_sums<T, S::THREADS, 64>(sums, p, a, rank0, col0, dw);
    cluster.sync();                                              // a CTA's sums stay until the others have read them
    umma::tc_fence_after();
    if (warp == 8) umma::tmem_dealloc(tmem, 512);
}

// ---- host side -------------------------------------------------------------------------------------------------------

constexpr int64_t FEW = TILE;       // tokens up to which each adapter has CTAs of its own

// What a kernel needs to know of a device once: its shared memory asked for, and how many of its CTAs an SM holds.
template <auto KERN>
int ctas_per_sm(int threads, int smem, int &n) {
    static std::atomic<int> known[64];
    int device = 0;
    BW_CUDA_TRY(cudaGetDevice(&device));
    n = device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
    if (n) return BW_OK;
    if (smem > 32 * 1024)      // (48 KB with what the kernel declares)
        BW_CUDA_TRY(cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    BW_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERN, threads, smem));
    if (n < 1) n = 1;
    if (device < 64) known[device].store(n, std::memory_order_relaxed);
    return BW_OK;
}
constexpr int SMS = 148;

// Clusters of `size` CTAs that the chip holds at once (the groups of SMs that a cluster has to fit into are of uneven sizes).
template <auto KERN>
int clusters_at_once(int size, int threads, int smem, int &n) {
    static std::atomic<int> known[64][8];
    int device = 0;
    BW_CUDA_TRY(cudaGetDevice(&device));
    n = device < 64 ? known[device][size - 1].load(std::memory_order_relaxed) : 0;
    if (n) return BW_OK;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    BW_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, KERN, &cfg));
    if (n < 1) n = 1;
    if (device < 64) known[device][size - 1].store(n, std::memory_order_relaxed);
    return BW_OK;
}
// Into how many parts, up to `most` (8 CTAs a cluster), each of `pieces` of work is cut: as few rounds of clusters as short as can be; a part costs
// `fixed` of an uncut piece on top.
template <auto KERN>
int cluster_parts(int64_t pieces, int64_t most, double fixed, int threads, int smem, int &best) {
    double least = 0.0;
    best = 1;
    for (int s = 1; s <= most && s <= 8; ++s) {
        int at_once = 0;
        const int rc = clusters_at_once<KERN>(s, threads, smem, at_once);
        if (rc != BW_OK) return rc;
        const double time = (double)((pieces + at_once - 1) / at_once) * (1.0 / s + fixed);
        if (s == 1 || time < least) {
            least = time;
            best = s;
        }
    }
    return BW_OK;
}
// The same for pieces that need not run together.
int parts_of(int64_t pieces, int64_t at_once, int64_t most, double fixed) {
    int best = 1;
    double least = 0.0;
    for (int s = 1; s <= most; ++s) {
        const double time = (double)((pieces * s + at_once - 1) / at_once) * (1.0 / s + fixed);
        if (s == 1 || time < least) {
            least = time;
            best = s;
        }
    }
    return best;
}
// CTAs among which a tile's adapters are dealt: with few tokens each may be another; prompts are runs of one.
int slots_of(const AdapterArgs &p) {
    const int most = p.M <= FEW ? 64 : p.M <= 512 ? 16 : 2, tokens = p.M < TILE ? (int)p.M : TILE;
    const int n = p.adapters + 1 < tokens ? p.adapters + 1 : tokens;
    return n < most ? n : most;
}

template <typename T, int NBR>
int shrink_fast(const T *x, const T *w, AdapterArgs p, void *h, cudaStream_t st) {
    constexpr int RANKS = 8 * NBR, FEW_SMEM = 7 * 16 * (RANKS + 1) * 4, RING = (TILE + RANKS) * 128 * SHRINK_STAGES, SUMS = TILE * (RANKS + 4) * 4,
                  SMEM = RING > SUMS ? RING : SUMS;
    p.slots = slots_of(p);
    const int64_t most = (p.cols + 255) / 256;                    // (a part has 256 columns at least; a cluster 8 CTAs at most)
    const unsigned tiles = (unsigned)((p.M + TILE - 1) / TILE);
    int per_sm = 0, rc;
    if (p.M <= FEW) {
        if ((rc = ctas_per_sm<adapter_shrink_few_kernel<T, NBR>>(256, FEW_SMEM, per_sm)) != BW_OK) return rc;
        const int parts = most < 8 ? (int)most : 8;
        const int64_t per_split = ((p.cols + parts - 1) / parts + 63) / 64 * 64;
        return launch_early("adapter_shrink_few_kernel", adapter_shrink_few_kernel<T, NBR>, dim3(parts, p.slots), 256, FEW_SMEM, st, dim3(parts), x, w, p, per_split, h);
    }
    if ((rc = ctas_per_sm<adapter_shrink_kernel<T, NBR>>(128, SMEM, per_sm)) != BW_OK) return rc;
    int parts = 1;
    if ((rc = cluster_parts<adapter_shrink_kernel<T, NBR>>(tiles, most, 0.02, 128, SMEM, parts)) != BW_OK) return rc;
    const int64_t per_split = ((p.cols + parts - 1) / parts + 63) / 64 * 64;
    return launch_early("adapter_shrink_kernel", adapter_shrink_kernel<T, NBR>, dim3(parts, tiles, p.slots), 128, SMEM, st, dim3(parts), x, w, p, per_split, h);
}
template <typename T>
int shrink(const void *x, const void *w, const AdapterArgs &p, void *h, cudaStream_t st) {
    if (p.rank <= 8) return shrink_fast<T, 1>((const T *)x, (const T *)w, p, h, st);
    if (p.rank <= 16) return shrink_fast<T, 2>((const T *)x, (const T *)w, p, h, st);
    if (p.rank <= 32) return shrink_fast<T, 4>((const T *)x, (const T *)w, p, h, st);
    if (p.rank <= 64) return shrink_fast<T, 8>((const T *)x, (const T *)w, p, h, st);
    return shrink_fast<T, 16>((const T *)x, (const T *)w, p, h, st);
}

template <typename T, int KS>
int expand_umma(void *h, const T *w, AdapterArgs p, const T *base, T *out, cudaStream_t st) {
    using S = ExpandShape<KS>;
    p.slots = p.adapters + 1 < 2 ? p.adapters + 1 : 2;
    int per_sm = 0;
    const int rc = ctas_per_sm<adapter_expand_umma_kernel<T, KS>>(EU_THREADS, S::SMEM, per_sm);
    if (rc != BW_OK) return rc;
    const int64_t tiles = (p.M + EU_TILE - 1) / EU_TILE, blocks = (p.cols + EU_COLS - 1) / EU_COLS, most = (blocks + 1) / 2;
    // (where an adapter's run of tokens ends, a tile has another one's as well)
    const int64_t passes = tiles + (p.adapters - 1 < tiles ? p.adapters - 1 : tiles);
    const int groups = parts_of(passes, SMS, most < 64 ? most : 64, 5.0 / blocks);      // (a start takes as long as five blocks)
    const int64_t per_group = (blocks + groups - 1) / groups * EU_COLS;
    return launch_early("adapter_expand_umma_kernel", adapter_expand_umma_kernel<T, KS>, dim3((unsigned)tiles, (unsigned)((p.cols + per_group - 1) / per_group), p.slots), EU_THREADS, S::SMEM,
                        st, dim3(1), h, w, p, per_group, base, out);
}
template <typename T, int KS>
int expand_fast(void *h, const T *w, AdapterArgs p, const T *base, T *out, cudaStream_t st) {
    // tcgen05 has one CTA an SM, whose start takes some microseconds.  Rank 64, bf16, shrink of 64 columns and expand, us, mma.sync / tcgen05: 8192 tokens of one
    // adapter to 14336 columns 146 / 91, of 8 167 / 109; 8192 tokens to 4096 columns of one 57 / 37, of 8 57 / 50; 4096 of two to 4096 33.6 / 33.0, to 1024 16.8 / 18.5; 1024 of one to 4096
    // 15.5 / 13.8, to 1024 10.1 / 12.3; 512 of one to 14336 20 / 15, of two 20 / 21.
    if constexpr (KS > 2)
        if (p.M >= 512 && p.M >= (int64_t)256 * p.adapters && p.M * p.cols >= (int64_t)(p.adapters == 1 ? 4 : 24) << 20) return expand_umma<T, KS>(h, w, p, base, out, st);
    constexpr int SMEM = (KS * 16 + TILE) * 128 * (KS <= 4 ? 4 : 3);
    p.slots = slots_of(p);
    if (p.M <= FEW)
        return launch_early("adapter_expand_few_kernel", adapter_expand_few_kernel<T, KS>, dim3((unsigned)((p.cols + 255) / 256), p.slots), 128, 0, st, dim3(1), h, w, p, base, out);
    int per_sm = 0;
    const int rc = ctas_per_sm<adapter_expand_kernel<T, KS>>(128, SMEM, per_sm);
    if (rc != BW_OK) return rc;
    const int64_t tiles = (p.M + TILE - 1) / TILE, blocks = (p.cols + 63) / 64, most = (blocks + 1) / 2;
    const int groups = parts_of(tiles, SMS * per_sm, most < 64 ? most : 64, 3.0 / blocks);
    const int64_t per_group = (blocks + groups - 1) / groups * 64;
    return launch_early("adapter_expand_kernel", adapter_expand_kernel<T, KS>, dim3((unsigned)tiles, (unsigned)((p.cols + per_group - 1) / per_group), p.slots), 128, SMEM, st, dim3(1),
                                                h, w, p, per_group, base, out);
}
template <typename T>
int expand(void *h, const void *w, const AdapterArgs &p, const void *base, void *out, cudaStream_t st) {
    if (p.rank <= 16) return expand_fast<T, 1>(h, (const T *)w, p, (const T *)base, (T *)out, st);
    if (p.rank <= 32) return expand_fast<T, 2>(h, (const T *)w, p, (const T *)base, (T *)out, st);
    if (p.rank <= 64) return expand_fast<T, 4>(h, (const T *)w, p, (const T *)base, (T *)out, st);
    return expand_fast<T, 8>(h, (const T *)w, p, (const T *)base, (T *)out, st);
}

template <typename T, int RB, int RG>
int outer_fast(void *h, const T *x, const AdapterArgs &p, T *dw, cudaStream_t st) {
    using S = OuterShape<RB, RG, PARTS<T>>;
    const int64_t blocks = (p.cols + 255) / 256, rows = (int64_t)p.adapters * ((p.rank + S::RANKS - 1) / S::RANKS), most = (p.M + 2 * OUTER_STEP - 1) / (2 * OUTER_STEP);
    int per_sm = 0, parts = 1, rc = ctas_per_sm<adapter_outer_kernel<T, RB, RG>>(S::THREADS, S::SMEM, per_sm);
    if (rc == BW_OK) rc = cluster_parts<adapter_outer_kernel<T, RB, RG>>(blocks * rows, most, 0.12, S::THREADS, S::SMEM, parts);
    if (rc != BW_OK) return rc;
    return launch_early("adapter_outer_kernel", adapter_outer_kernel<T, RB, RG>, dim3((unsigned)blocks, (unsigned)rows, parts), S::THREADS, S::SMEM, st, dim3(1, 1, parts), h, x, p, dw);
}
template <typename T>
int outer_umma(void *h, const T *x, const AdapterArgs &p, T *dw, cudaStream_t st) {
    const int64_t blocks = (p.cols + 255) / 256, rows = (int64_t)p.adapters * ((p.rank + 63) / 64), most = (p.M + 4 * OUTER_STEP - 1) / (4 * OUTER_STEP);
    int per_sm = 0, parts = 1, rc = ctas_per_sm<adapter_outer_umma_kernel<T>>(OuterUmma<T>::THREADS, OuterUmma<T>::SMEM, per_sm);
    // (a part's start and end take as long as about 384 of its tokens)
    if (rc == BW_OK) rc = cluster_parts<adapter_outer_umma_kernel<T>>(blocks * rows, most, 384.0 * p.adapters / p.M, OuterUmma<T>::THREADS, OuterUmma<T>::SMEM, parts);
    if (rc != BW_OK) return rc;
    return launch_early("adapter_outer_umma_kernel", adapter_outer_umma_kernel<T>, dim3((unsigned)blocks, (unsigned)rows, parts), OuterUmma<T>::THREADS, OuterUmma<T>::SMEM, st, dim3(1, 1, parts), h, x, p, dw);
}
template <typename T>
int outer(void *h, const void *x, const AdapterArgs &p, void *dw, cudaStream_t st) {
    // tcgen05 has 64 ranks' work for any rank and one CTA an SM, mma.sync two or three of less.  With shrink of 64 columns in front, us, mma.sync / tcgen05: bf16, rank 64, 14336 columns, 8192
    // tokens of one adapter 174 / 74 (fp16 143 / 96), of 16 220 / 124; 512 tokens of 4096 columns of one 21 / 12, of 16 (256 CTAs) 11 / 17; 1024 of 16 14 / 18; rank 32, 1024 columns, 2048 tokens
    // 17 / 14, 1024 tokens 11.7 / 11.8, 512 tokens 9.2 / 10.5; 1024 tokens of 4096 columns 16 / 13; 14336 columns, 8192 tokens of four 116 / 84, 512 tokens of four 13 / 19; rank 16, 14336
    // columns, 8192 tokens 69 / 75 (fp16 70 / 94).
    const int64_t rows = (int64_t)p.adapters * ((p.rank + 63) / 64);
    const bool at_once = (p.cols + 255) / 256 * rows <= SMS;
    static_assert(MANY <= 512, "of fewer tokens the rank values have no parts");
    if (p.M >= 512 && (p.rank > 32 ? at_once || p.M > 64 * rows : p.rank > 16 && (at_once || p.M >= 512 * rows) && (p.M >= 2048 || p.M * p.cols >= (int64_t)4 << 20)))
        return outer_umma<T>(h, (const T *)x, p, (T *)dw, st);
    if (p.rank <= 16) return outer_fast<T, 1, 1>(h, (const T *)x, p, (T *)dw, st);
    if (p.rank <= 32) return outer_fast<T, 2, 1>(h, (const T *)x, p, (T *)dw, st);
    return outer_fast<T, 2, 2>(h, (const T *)x, p, (T *)dw, st);
}

// The same three by the general kernels, whose rank values are fp32.
template <typename T>
int shrink_general(const void *x, const void *w, const AdapterArgs &p, void *h, cudaStream_t st) {
    adapter_shrink_general_kernel<T><<<(unsigned)((p.M * p.rank + 3) / 4), 128, 0, st>>>((const T *)x, p.M, p.cols, (const T *)w, p.adapters, p.rank, p.index, (float *)h);
    return check_launch("adapter_shrink_general_kernel");
}
template <typename T>
int expand_general(void *h, const void *w, const AdapterArgs &p, const void *base, void *out, cudaStream_t st) {
    adapter_expand_general_kernel<T><<<dim3((unsigned)((p.cols + 255) / 256), (unsigned)(p.M < 16384 ? p.M : 16384)), 256, 0, st>>>(
        (const float *)h, p.M, p.cols, (const T *)w, p.adapters, p.rank, p.index, p.scaling, (const T *)base, (T *)out);
    return check_launch("adapter_expand_general_kernel");
}
template <typename T>
int outer_general(void *h, const void *x, const AdapterArgs &p, void *dw, cudaStream_t st) {
    adapter_outer_general_kernel<T><<<dim3((unsigned)(p.adapters * p.rank), (unsigned)((p.cols + 255) / 256)), 256, 0, st>>>(
        (const float *)h, (const T *)x, p.M, p.cols, p.rank, p.index, p.scaling, (T *)dw);
    return check_launch("adapter_outer_general_kernel");
}

// One form for all passes of an adapter, forward and backward, by sizes alone: what holds the rank values depends on it.
bool fast_sizes(int64_t M, int64_t N, int64_t K, int n, int r) {
    return r % 8 == 0 && r <= 128 && K % 8 == 0 && N % 8 == 0 && M < (int64_t)65535 * TILE && (int64_t)n * 2 <= 65535;
}

template <typename T>
int forward(const void *x, int64_t M, int64_t N, int64_t K, const void *down, const void *up, int n, int r, const int32_t *index, const float *scaling,
            const void *base, void *out, void *h, cudaStream_t st) {
    const bool fast = fast_sizes(M, N, K, n, r);
    const AdapterArgs in = {M, K, index, nullptr, n, r, 1, false}, to = {M, N, index, scaling, n, r, 1, true};
    const int rc = fast ? shrink<T>(x, down, in, h, st) : shrink_general<T>(x, down, in, h, st);
    if (rc != BW_OK) return rc;
    return fast ? expand<T>(h, up, to, base, out, st) : expand_general<T>(h, up, to, base, out, st);
}
template <typename T>
int backward(const void *dy, const void *x, int64_t M, int64_t N, int64_t K, const void *down, const void *up, int n, int r, const int32_t *index,
             const float *scaling, void *h, void *dx, void *d_down, void *d_up, void *dh, cudaStream_t st) {
    const bool fast = fast_sizes(M, N, K, n, r);
    const bool behind = M > 0 && (dx || d_down);
    const AdapterArgs in = {M, N, index, nullptr, n, r, 1, false}, over_k = {M, K, index, scaling, n, r, 1, behind}, over_n = {M, N, index, scaling, n, r, 1, behind};
    int rc = BW_OK;
    if (behind) rc = fast ? shrink<T>(dy, up, in, dh, st) : shrink_general<T>(dy, up, in, dh, st);
    if (rc == BW_OK && M > 0 && dx) rc = fast ? expand<T>(dh, down, over_k, nullptr, dx, st) : expand_general<T>(dh, down, over_k, nullptr, dx, st);
    if (rc == BW_OK && d_down) rc = fast ? outer<T>(dh, x, over_k, d_down, st) : outer_general<T>(dh, x, over_k, d_down, st);
    if (rc == BW_OK && d_up) rc = fast ? outer<T>(h, dy, over_n, d_up, st) : outer_general<T>(h, dy, over_n, d_up, st);
    return rc;
}

}  // namespace

// (two 16-bit parts and a power of two a row; fp32 values, of bf16 and of the general kernels, are less; three 16-bit parts more of many tokens of bf16)
size_t adapter_hidden_bytes(int64_t M, int r) { return (size_t)M * r * (M >= MANY ? 10 : 4) + (size_t)M * 4; }

int adapter_device_status() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_adapter_status, sizeof(int)) != cudaSuccess) return -1;
    if (v) (void)cudaMemcpyToSymbol(g_adapter_status, &zero, sizeof(int));
    return v;
}

int adapter_forward(const void *x, int dtype, int64_t M, int64_t N, int64_t K, const void *down, const void *up, int n, int r, const int32_t *index,
                    const float *scaling, const void *base, void *out, void *h, cudaStream_t st) {
    if (dtype == BW_F16) return forward<__half>(x, M, N, K, down, up, n, r, index, scaling, base, out, h, st);
    return forward<__nv_bfloat16>(x, M, N, K, down, up, n, r, index, scaling, base, out, h, st);
}
int adapter_backward(const void *dy, int dtype, const void *x, int64_t M, int64_t N, int64_t K, const void *down, const void *up, int n, int r,
                     const int32_t *index, const float *scaling, void *h, void *dx, void *d_down, void *d_up, void *workspace, cudaStream_t st) {
    if (dtype == BW_F16) return backward<__half>(dy, x, M, N, K, down, up, n, r, index, scaling, h, dx, d_down, d_up, workspace, st);
    return backward<__nv_bfloat16>(dy, x, M, N, K, down, up, n, r, index, scaling, h, dx, d_down, d_up, workspace, st);
}

}  // namespace bw
