// Log probabilities of given tokens with the entropy and the largest alternatives (bw_token_log_probs), and their gradient.
//
// Of a row x with largest value m:  s = sum 2^u, w = sum 2^u u  with u = (x - m) / ln 2;
//     log p[j] = (x[j] - m) - ln s,   H = ln s - ln2 * w / s
// The gradient of g log p[t] + e H + sum g_i log p[t_i] in x[j] is  p[j] (-(g + sum g_i) - e (log p[j] + H)) + (j == t) g + sum (j == t_i) g_i.
//
// One pass over the row with the running maximum; x - m is formed before the product, so that masks of the type's lowest value stay finite or become
// exact zeros.  Sums are fp32: 32 terms (16 of fp32 logits) by themselves, then those sums, then a tree: a chain of 500 equal terms rounds the same way each time and was
// off by 7e-6.  Bound by the bytes of the logits where there are many rows, by latency where there are few (bf16, with entropy): 8192 x 131072 333 us, 6.4 TB/s (the measured copy
// rate is 6.5), their gradient 640 us, 6.7 TB/s (1120 of rows that start elsewhere than their gradient); 61 x 131071 7.0 to 8.0 us; one row of 50272 2.9 to 3.6 us.  Twenty alternatives add 20 us to
// 2000 x 131071 (92 to 98), 10 to 2000 x 32000 (28), 4 to 61 x 131071, five add 3 to one row: six barriers' worth of latency behind each row, of which an SM's other CTAs hide a part.  Rows whose masks leave
// fewer values than alternatives are searched digit by digit (search_share): 61 x 131071 with all but three masked and five alternatives 120 us, 2000 x 32000 313, one row of 50272 35.
//
// A row is taken by a cluster of one to eight CTAs, which join through distributed shared memory.
#include <cooperative_groups.h>

#include <type_traits>

#include "early_launch.cuh"

namespace bw {
namespace {

namespace cg = cooperative_groups;

constexpr int THREADS = 256, UNROLL = 4, BLOCKS = 16;     // of a CTA (of short rows fewer, N below); 16-byte loads of a step; blocks of steps of a thread
constexpr int STEP = THREADS * UNROLL;                     // 16-byte pieces of a CTA's step
constexpr int CANDIDATES = 512;
constexpr int SMS = 148;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// The order of the alternatives: falling value, rising index; NaN before all.  Larger is better; nothing is 0.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0xfffffffeu;                       // (below the mark of no value yet, whatever the index)
    const uint32_t b = __float_as_uint(x + 0.0f);         // (-0 counts as 0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
    return order == 0xfffffffeu ? NAN : __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float ld_l2(const float *p) { return __ldcg(p); }
__device__ __forceinline__ float ld_l2(const __half *p) { return __half2float(__ldcg(p)); }
__device__ __forceinline__ float ld_l2(const __nv_bfloat16 *p) { return __bfloat162float(__ldcg(p)); }

// 16 bytes of a row.
template <typename T> struct Piece {
    static constexpr int V = 16 / sizeof(T);
    uint4 raw;
    __device__ __forceinline__ void load(const T *p) { raw = __ldcg(reinterpret_cast<const uint4 *>(p)); }
    // (in the place of pieces that are not there: -infinity)
    __device__ __forceinline__ void nothing() {
        const uint32_t w = __is_same(T, float) ? 0xff800000u : __is_same(T, __half) ? 0xfc00fc00u : 0xff80ff80u;
        raw = make_uint4(w, w, w, w);
    }
    __device__ __forceinline__ float2 pair(int i) const {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(&raw);
        if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else if constexpr (__is_same(T, __half)) return __half22float2(*reinterpret_cast<const __half2 *>(w + i));
        else return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
    __device__ __forceinline__ void put(int i, float2 v) {
        uint32_t *w = reinterpret_cast<uint32_t *>(&raw);
        if constexpr (sizeof(T) == 4) {
            w[2 * i] = __float_as_uint(v.x);
            w[2 * i + 1] = __float_as_uint(v.y);
        } else if constexpr (__is_same(T, __half)) *reinterpret_cast<__half2 *>(w + i) = __float22half2_rn(v);
        else *reinterpret_cast<__nv_bfloat162 *>(w + i) = __float22bfloat162_rn(v);
    }
};
// The largest value of pieces; NaN where there is one.
template <typename T>
__device__ __forceinline__ float largest(const Piece<T> (&x)[UNROLL]) {
    if constexpr (sizeof(T) == 4) {
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) m = max_nan(m, max_nan(x[u].pair(i).x, x[u].pair(i).y));
        return m;
    } else {
        using T2 = typename std::conditional<__is_same(T, __half), __half2, __nv_bfloat162>::type;
        T2 m = *reinterpret_cast<const T2 *>(&x[0].raw.x);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) m = __hmax2_nan(m, reinterpret_cast<const T2 *>(&x[u].raw)[i]);
        return max_nan(to_f32(m.x), to_f32(m.y));
    }
}

// The running maximum and sums of some values of a row.
struct Sums {
    float m, s, w;
    // To a larger maximum.  (Without a value above -infinity there is nothing to keep, but for a NaN.)
    __device__ __forceinline__ void raise(float to) {
        if (m == -INFINITY) {
            s *= 0.0f;
            w = 0.0f;
        } else {
            // (products rounded by themselves: the same log probability with the entropy and without; with alternatives too, where they do not change how many threads
            // take the row, which threads_of says: the last bits are those of the order of the sums)
            const float d = __fmul_rn(m - to, LOG2E), f = ex2(d);
            // (what fell by so much that nothing of it is left: infinite d)
            w = f == 0.0f ? 0.0f : f * fmaf(s, d, w);
            s = __fmul_rn(s, f);
        }
        m = to;
    }
};

struct LogProbs {
    const void *logits;
    const int64_t *tokens;
    float *log_probs, *entropy, *top_log_probs;
    int64_t *top_tokens;
    float4 *stats;                       // m, log2 s, H
    int64_t stride, rows;
    int vocab, top, cluster;
};

// A row as 16-byte pieces on their boundaries and the values before and behind them (`extra` of them), which rank 0 takes; and a rank's share of the pieces.
template <typename T> struct Row {
    const T *x;
    int head, behind, extra, v0, v1;
    __device__ __forceinline__ Row(const T *row, int vocab, int rank, int ranks) : x(row) {
        constexpr int V = Piece<T>::V;
        head = (int)((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(T));
        if (head > vocab) head = vocab;
        const int pieces = (vocab - head) / V, each = (pieces + ranks - 1) / ranks;
        behind = head + pieces * V;
        extra = rank == 0 ? head + vocab - behind : 0;
        v0 = rank * each < pieces ? rank * each : pieces;
        v1 = v0 + each < pieces ? v0 + each : pieces;
    }
    __device__ __forceinline__ const T *piece(int v) const { return x + head + (int64_t)v * Piece<T>::V; }
    __device__ __forceinline__ int extra_at(int i) const { return i < head ? i : behind + i - head; }
};

// The values of a call's rows that are looked at for alternatives.
//
// The threads of a row's CTAs form 64 groups.  The top-th largest of the groups' largest values is a bound from below: `top` groups hold a value that
// reaches it.  Only blocks that reach it are read again, some more than `top` of them in all CTAs together, and the values that reach it are ranked.  Where too many do (many equal
// values, as masks leave them; many large ones in few threads' places) a CTA finds the `top` best of its share digit by digit instead.
constexpr int GROUPS = 64;
template <int N> struct __align__(16) TopScratch {
    float largest[BLOCKS][N];                    // of a thread's blocks
    __align__(16) uint32_t group[GROUPS];              // the groups' largest values, of all CTAs
    __align__(16) uint64_t list[CANDIDATES + 2];       // this CTA's candidates: (order << 32) | ~index
    __align__(16) uint64_t all[N == THREADS ? CANDIDATES : 2];      // all CTAs' (rank 0)
    uint64_t best[32];
    uint32_t histogram[256], entry[N];
    int count, entries, need, counts[8];
    uint32_t least[N / 32], prefix;
    int scan[N / 32];
};

__device__ __forceinline__ uint64_t candidate(float x, int at) { return (uint64_t)order_of(x) << 32 | (uint32_t)~at; }

// The best `top` of n candidates, in order, into `best`; 0 where there are fewer.  All candidates differ.
template <int N>
__device__ __forceinline__ void rank_candidates(uint64_t *list, int n, int top, uint64_t *best) {
    const int tid = threadIdx.x;
    if (tid < top) best[tid] = 0;
    if (tid < 2) list[n + tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += N) {
        const uint64_t mine = list[i];
        int before = 0;
#pragma unroll 4
        for (int k = 0; k < n; k += 2) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(list + k);
            before += (two.x > mine) + (two.y > mine);
        }
        if (before < top) best[before] = mine;
    }
    __syncthreads();
}

// The best `top` values of a rank's share, as candidates into s.list: the top-th largest value is found eight bits at a time.
template <typename T, int N>
__device__ __noinline__ void search_share(TopScratch<N> &s, const Row<T> &row, int top) {
    constexpr int V = Piece<T>::V;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    __syncthreads();
    if (tid == 0) {
        s.prefix = 0;
        s.need = top;
        s.count = 0;
    }
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += N) s.histogram[i] = 0;
        __syncthreads();
        const uint32_t prefix = s.prefix;
        auto count = [&](float x) {
            const uint32_t o = order_of(x);
            if (shift == 24 || o >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&s.histogram[o >> shift & 255], 1u);
        };
        for (int v = row.v0 + tid; v < row.v1; v += N) {
            Piece<T> x;
            x.load(row.piece(v));
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                count(x.pair(i).x);
                count(x.pair(i).y);
            }
        }
        if (tid < row.extra) count(ld_l2(row.x + row.extra_at(tid)));
        __syncthreads();
        if (tid == 0) {
            int need = s.need, digit = 255;
            while (digit > 0 && (int)s.histogram[digit] < need) need -= (int)s.histogram[digit--];
            s.need = need;
            s.prefix = prefix | (uint32_t)digit << shift;
        }
        __syncthreads();
    }
    const uint32_t bound = s.prefix;
    const int need = s.need;
    // (fewer than `top` values are larger; of the equal ones the first `need` in rising order: before the pieces, in them, behind them)
    int taken = 0;
    auto round = [&](const float (&x)[V], int n, int at) {      // n values of this thread from index `at` on; threads' indexes rise
        int equal = 0;
        for (int i = 0; i < V; ++i)
            if (i < n) {
                const uint32_t o = order_of(x[i]);
                if (o > bound) {
                    const int k = atomicAdd(&s.count, 1);
                    if (k < CANDIDATES) s.list[k] = candidate(x[i], at + i);
                }
                equal += o == bound;
            }
        if (!__syncthreads_or(equal)) return;
        int sum = equal;
        for (int d = 1; d < 32; d *= 2) {
            const int o = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += o;
        }
        if (lane == 31) s.scan[warp] = sum;
        __syncthreads();
        int before = taken + sum - equal, all = 0;
        for (int i = 0; i < N / 32; ++i) {
            before += i < warp ? s.scan[i] : 0;
            all += s.scan[i];
        }
        for (int i = 0; i < V; ++i)
            if (i < n && order_of(x[i]) == bound && before++ < need) {
                const int k = atomicAdd(&s.count, 1);
                if (k < CANDIDATES) s.list[k] = candidate(x[i], at + i);
            }
        taken += all;
        __syncthreads();
    };
    float x[V];
    const int head = row.extra ? row.head : 0;
    x[0] = tid < head ? ld_l2(row.x + tid) : 0.0f;
    round(x, tid < head, tid);
    for (int v0 = row.v0; v0 < row.v1; v0 += N) {
        Piece<T> piece;
        if (v0 + tid < row.v1) piece.load(row.piece(v0 + tid));
        else piece.nothing();
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            x[2 * i] = piece.pair(i).x;
            x[2 * i + 1] = piece.pair(i).y;
        }
        round(x, v0 + tid < row.v1 ? V : 0, row.head + (v0 + tid) * V);
    }
    const int rest = row.extra - head;
    x[0] = tid < rest ? ld_l2(row.x + row.behind + tid) : 0.0f;
    round(x, tid < rest, row.behind + tid);
    __syncthreads();
}

// This CTA's candidates into s.list, s.count of them (at most `room`, which is `top` or more).  s.group holds the groups' largest values; `key` is this thread's largest
// value; those of its blocks of `per` steps lie in s.largest; `extra` is its value before or behind the pieces.
template <typename T, int N>
__device__ __forceinline__ void find_candidates(TopScratch<N> &s, const Row<T> &row, int top, int room, int blocks, int per, uint32_t key, float extra) {
    constexpr int V = Piece<T>::V, BLOCK = UNROLL * V;      // values of a thread's step: 16 or 32
    static_assert(BLOCK <= 32, "a lane a value");
    const int tid = threadIdx.x, lane = tid % 32;
    constexpr int EACH = N / GROUPS;         // threads that compare one group's value with the others'
    static_assert(EACH == 1 || EACH == 2 || EACH == 4, "one, two or four threads a group");
    const uint32_t mine = s.group[tid / EACH];
    int larger = 0;
#pragma unroll
    for (int i = 0; i < GROUPS / EACH; i += 4) {
        const uint4 k = *reinterpret_cast<const uint4 *>(s.group + tid % EACH * (GROUPS / EACH) + i);
        larger += (k.x > mine) + (k.y > mine) + (k.z > mine) + (k.w > mine);
    }
#pragma unroll
    for (int d = 1; d < EACH; d *= 2) larger += __shfl_xor_sync(0xffffffffu, larger, d);
    const uint32_t low = __reduce_min_sync(0xffffffffu, larger < top ? mine : 0xffffffffu);
    if (lane == 0) s.least[tid / 32] = low;
    if (tid == 0) s.count = s.entries = 0;
    __syncthreads();
    uint32_t least = s.least[0];
#pragma unroll
    for (int i = 1; i < N / 32; ++i) least = min(least, s.least[i]);
    auto offer = [&](float x, int at) {
        if (order_of(x) < least) return;
        const int i = atomicAdd(&s.count, 1);
        if (i < room) s.list[i] = candidate(x, at);
    };
    if (key >= least) {
        if (tid < row.extra) offer(extra, row.extra_at(tid));
        uint32_t hits = 0;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
            if (b < blocks) hits |= (uint32_t)(order_of(s.largest[b][tid]) >= least) << b;
        if (hits) {
            int at = atomicAdd(&s.entries, __popc(hits));
            for (; hits; hits &= hits - 1, ++at)
                if (at < N) s.entry[at] = (__ffs(hits) - 1) * N + tid;
        }
    }
    __syncthreads();
    const int entries = s.entries;
    if (entries <= N) {
        // a warp a block, four of them in flight
        for (int step = 0; step < per; ++step)
            for (int i0 = tid / 32; i0 < entries; i0 += 4 * (N / 32)) {
                float x[4];
                int at[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i = i0 + k * (N / 32), entry = i < entries ? (int)s.entry[i] : 0;
                    const int v = row.v0 + (entry / N * per + step) * (N * UNROLL) + lane / V * N + entry % N;
                    at[k] = i < entries && lane < BLOCK && v < row.v1 ? row.head + v * V + lane % V : -1;
                    if (at[k] >= 0) x[k] = ld_l2(row.x + at[k]);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (at[k] >= 0) offer(x[k], at[k]);
            }
        __syncthreads();
        if (s.count <= room) return;
    }
    search_share(s, row, top);
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// The sums of `lanes` neighbouring lanes (a power of two, and other lanes' the same again) as one.
__device__ __forceinline__ Sums joined(Sums a, int lanes) {
    const float m = value_of(__reduce_max_sync(0xffffffffu, order_of(a.m)));
    if (m > a.m) a.raise(m);
    for (int d = lanes / 2; d; d >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, d);
        a.w += __shfl_xor_sync(0xffffffffu, a.w, d);
    }
    return a;
}

// A row a cluster, of CTAs of N threads.
template <typename T, int N, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(N, (TOP ? 4 : 5) * THREADS / N) log_probs_kernel(const LogProbs p) {
    constexpr int V = Piece<T>::V, WARPS = N / 32, STEP = N * UNROLL;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const int rank = (int)(blockIdx.x % p.cluster);
    const int64_t r = blockIdx.x / p.cluster;
    __shared__ Sums s_warp[WARPS], s_all[8];
    __shared__ typename std::conditional<TOP, TopScratch<N>, int>::type s_top;
    const cg::cluster_group cluster = cg::this_cluster();
    if (p.cluster > 1) cluster_arrive();                   // (all CTAs have begun before one writes into another's memory)
    pdl_wait();
    pdl_launch_dependents();

    const Row<T> row((const T *)p.logits + r * p.stride, p.vocab, rank, p.cluster);
    const int64_t t = p.tokens ? __ldcg(p.tokens + r) : -1;
    Piece<T> next[UNROLL];
    auto load = [&](int step) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int v = row.v0 + step * STEP + u * N + tid;
            if (v < row.v1) next[u].load(row.piece(v));
            else next[u].nothing();
        }
    };
    load(0);
    const float extra = tid < row.extra ? ld_l2(row.x + row.extra_at(tid)) : -INFINITY;
    const float xt = t >= 0 && t < p.vocab ? ld_l2(row.x + t) : NAN;
    // padding: nothing of the row is asked for.  (Its first step, at most 16 KB a CTA, is read all the same: loads that waited for the token would come later in every row.)
    const bool skipped = !ENTROPY && !TOP && t < 0;
    const int steps = skipped ? 0 : (row.v1 - row.v0 + STEP - 1) / STEP, per = (steps + BLOCKS - 1) / BLOCKS;
    Sums a = {-INFINITY, 0.0f, 0.0f};
    uint32_t key = 0;
    float block = -INFINITY;
    int in_block = 0, blocks = 0;
    bool any = false;                                    // whether the block has a piece: a thread's last one may have none
    for (int step = 0; step < steps; ++step) {
        Piece<T> x[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) x[u] = next[u];
        if (step + 1 < steps) load(step + 1);
        const float m = largest(x);
        if (m > a.m) a.raise(m);
        if constexpr (TOP) {
            block = max_nan(block, m);
            any |= row.v0 + step * STEP + tid < row.v1;
            if (++in_block == per || step + 1 == steps) {
                if (any) {
                    s_top.largest[blocks++][tid] = block;
                    key = max(key, order_of(block));
                }
                block = -INFINITY;
                in_block = 0;
                any = false;
            }
        }
        const float by = a.m == -INFINITY ? 0.0f : -a.m;
        float2 s = {0.0f, 0.0f}, w = {0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float2 d = fmul2(fadd2(x[u].pair(i), make_float2(by, by)), make_float2(LOG2E, LOG2E)), e = make_float2(ex2(d.x), ex2(d.y));
                s = fadd2(s, e);
                // (0 * -infinity is not wanted: below 2^-1000 a weight is 0.  NaN stands in s.)
                if constexpr (ENTROPY) w = ffma2(e, make_float2(fmaxf(d.x, -1000.0f), fmaxf(d.y, -1000.0f)), w);
            }
        a.s += s.x + s.y;
        if constexpr (ENTROPY) a.w += w.x + w.y;
    }
    if (tid < row.extra && !skipped) {
        if constexpr (TOP) key = max(key, order_of(extra));
        // (NaN is larger than no maximum: its difference goes into the sum)
        if (extra > a.m) a.raise(extra);
        const float d = __fmul_rn(extra - (a.m == -INFINITY ? 0.0f : a.m), LOG2E), e = ex2(d);
        a.s += e;
        if constexpr (ENTROPY) a.w += e * fmaxf(d, -1000.0f);
    }
    const int room = CANDIDATES / p.cluster;
    if constexpr (TOP) {
        const int size = N * p.cluster / GROUPS;             // threads of a group, 1 to 32
        uint32_t k = key;
        for (int d = 1; d < size; d *= 2) k = max(k, __shfl_xor_sync(0xffffffffu, k, d));
        if (p.cluster > 1) cluster_wait();
        if (tid % size == 0)
            for (int i = 0; i < p.cluster; ++i) {
                uint32_t *to = s_top.group + rank * (GROUPS / p.cluster) + tid / size;
                *(p.cluster > 1 ? cluster.map_shared_rank(to, i) : to) = k;
            }
        if (p.cluster > 1) cluster_arrive();                 // (on their way while the sums are joined)
    }
    a = joined(a, 32);
    if (lane == 0) s_warp[warp] = a;
    __syncthreads();
    a = joined(s_warp[lane % WARPS], WARPS);                 // (in every warp)
    if (p.cluster > 1) {
        cluster_wait();
        if (tid == 0) *cluster.map_shared_rank(s_all + rank, 0) = a;
    }
    if constexpr (TOP) {
        find_candidates(s_top, row, p.top, room, blocks, per, key, extra);
        const int n = s_top.count;
        if (p.cluster > 1) {
            uint64_t *to = cluster.map_shared_rank(s_top.all, 0) + rank * room;
            for (int i = tid; i < n; i += N) to[i] = s_top.list[i];
            if (tid == 0) *cluster.map_shared_rank(s_top.counts + rank, 0) = n;
        } else rank_candidates<N>(s_top.list, n, p.top, s_top.best);
    }
    if (p.cluster > 1) {
        cluster_arrive();
        if (rank != 0) return;
        cluster_wait();
        if constexpr (TOP) {
            // (s_top.list, whose candidates are rank 0's part of `all`, takes them all, a warp those of one rank)
            // (clusters are of CTAs of eight warps)
            const int mine = lane < p.cluster ? s_top.counts[lane] : 0;
            int sum = mine;
            for (int d = 1; d < 8; d *= 2) {
                const int o = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += o;
            }
            const int n = __shfl_sync(0xffffffffu, sum, 7), from = __shfl_sync(0xffffffffu, sum - mine, warp), here = __shfl_sync(0xffffffffu, mine, warp);
            for (int k = lane; k < here; k += 32) s_top.list[from + k] = s_top.all[warp * room + k];
            __syncthreads();
            rank_candidates<N>(s_top.list, n, p.top, s_top.best);
        }
        a = joined(s_all[lane % p.cluster], p.cluster);
    }
    // (infinities of either sign as the largest value, and NaN: nothing is known of the row)
    const float log2s = fabsf(a.m) == INFINITY ? NAN : log2f(a.s), ln_s = __fmul_rn(LN2, log2s), h = ENTROPY ? ln_s - LN2 * (a.w / a.s) : 0.0f;
    if (tid == 0) {
        if (p.tokens) p.log_probs[r] = t < 0 ? 0.0f : (xt - a.m) - ln_s;
        if (ENTROPY) p.entropy[r] = h;
        if (p.stats) p.stats[r] = skipped ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : make_float4(a.m, log2s, h, 0.0f);
    }
    if constexpr (TOP)
        if (tid < p.top) {
            const uint64_t best = s_top.best[tid];
            p.top_tokens[r * p.top + tid] = (uint32_t)~best;
            p.top_log_probs[r * p.top + tid] = (value_of((uint32_t)(best >> 32)) - a.m) - ln_s;
        }
}

struct LogProbsGrad {
    const void *logits;
    void *grad;
    const int64_t *tokens, *top_tokens;
    const float4 *stats;
    const float *g, *e, *g_top;
    int64_t stride;
    int vocab, top, parts;               // parts: CTAs of a row
};

// Bound by the bytes of the logits and of their gradient.  ALIGNED: pieces of a row start where those of its gradient do.  The entries of the tokens are written again
// behind a barrier, by themselves: no comparison in the loop.
template <typename T, int N, bool ENTROPY, bool ALIGNED>
__global__ void __launch_bounds__(N, 4 * THREADS / N) log_probs_grad_kernel(const LogProbsGrad p) {
    constexpr int V = Piece<T>::V, STEP = N * UNROLL;
    const int tid = threadIdx.x, part = (int)(blockIdx.x % p.parts);
    const int64_t r = blockIdx.x / p.parts;
    pdl_wait();
    pdl_launch_dependents();
    const T *x = (const T *)p.logits + r * p.stride;
    T *out = (T *)p.grad + r * p.vocab;
    const float4 st = __ldcg(p.stats + r);
    const int64_t t = p.g ? __ldcg(p.tokens + r) : -1;
    const float given = t < 0 ? 0.0f : __ldcg(p.g + r), g = t >= p.vocab && given != 0.0f ? NAN : given, e = ENTROPY ? __ldcg(p.e + r) : 0.0f;
    const int top = p.g_top ? p.top : 0;
    float all = g;
    bool any = g != 0.0f || e != 0.0f;
    for (int i = 0; i < top; ++i) {
        const float gi = __ldcg(p.g_top + r * top + i);
        all += gi;
        any |= gi != 0.0f;
    }
    const float c = -fmaf(e, st.z, all), slope = -e * LN2;
    auto value = [&](float v) {
        const float u = fmaf(v - st.x, LOG2E, -st.y);
        // (0 * -infinity is not wanted: where a probability is 0, so is its gradient)
        return ex2(u) * (ENTROPY ? fmaf(slope, fmaxf(u, -1000.0f), c) : c);
    };
    const Row<T> row(ALIGNED ? x : (const T *)out, p.vocab, part, p.parts);      // (of the gradient's boundaries where they differ)
    if (!any) {                          // a row that nothing is asked of (padding): zeros, whatever stands in it
        for (int v = row.v0 + tid; v < row.v1; v += N) *reinterpret_cast<uint4 *>(out + row.head + (int64_t)v * V) = make_uint4(0, 0, 0, 0);
        if (tid < row.extra) out[row.extra_at(tid)] = from_f32<T>(0.0f);
        return;
    }
    const int steps = (row.v1 - row.v0 + STEP - 1) / STEP;
    Piece<T> next[UNROLL];
    auto load = [&](int step) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int v = row.v0 + step * STEP + u * N + tid;
            if (v >= row.v1) continue;
            if constexpr (ALIGNED) next[u].load(row.piece(v));
            else
#pragma unroll
                for (int i = 0; i < V / 2; ++i) next[u].put(i, make_float2(ld_l2(x + row.head + v * V + 2 * i), ld_l2(x + row.head + v * V + 2 * i + 1)));
        }
    };
    if (steps) load(0);
    for (int step = 0; step < steps; ++step) {
        Piece<T> y[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) y[u] = next[u];
        if (step + 1 < steps) load(step + 1);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int v = row.v0 + step * STEP + u * N + tid;
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float2 d = ffma2(fadd2(y[u].pair(i), make_float2(-st.x, -st.x)), make_float2(LOG2E, LOG2E), make_float2(-st.y, -st.y));
                const float2 prob = make_float2(ex2(d.x), ex2(d.y));
                float2 f = make_float2(c, c);
                if constexpr (ENTROPY) f = ffma2(make_float2(slope, slope), make_float2(fmaxf(d.x, -1000.0f), fmaxf(d.y, -1000.0f)), f);
                y[u].put(i, fmul2(prob, f));
            }
            if (v < row.v1) __stcs(reinterpret_cast<uint4 *>(out + row.head + (int64_t)v * V), y[u].raw);
        }
    }
    if (tid < row.extra) out[row.extra_at(tid)] = from_f32<T>(value(ld_l2(x + row.extra_at(tid))));
    __syncthreads();
    if (tid <= top) {
        const int64_t at = tid < top ? __ldcg(p.top_tokens + r * top + tid) : t;
        const int64_t from = row.head + (int64_t)row.v0 * V, to = row.head + (int64_t)row.v1 * V;
        const bool mine = (at >= from && at < to) || (part == 0 && ((at >= 0 && at < row.head) || (at >= row.behind && at < p.vocab)));
        if (mine) {
            float v = value(ld_l2(x + at)), more = at == t ? g : 0.0f;
            for (int i = 0; i < top; ++i)
                if (__ldcg(p.top_tokens + r * top + i) == at) more += __ldcg(p.g_top + r * top + i);
            out[at] = from_f32<T>(v + more);
        }
    }
}

// CTAs of a row, of at least a step (16 KB) each, rows of more than two steps: so many that all rows together have one an SM; the first division where two an SM have more than 64 KB each; rows of more
// than 384 KB until there are four.  us a call among others / alone (with the wait for the GPU), entropy and twenty alternatives, 1, 2, 4, 8 CTAs: 16 x 50272 bf16 8.5/20.1, 8.2/19.7, 7.0/18.6, 6.9/18.5;
// 61 x 50272 8.5/20.2, 8.2/19.8, 9.3/19.6, 9.1/20.7; 61 x 131071 13.3/24.7, 10.5/22.1, 12.0/21.4, 11.2/23.0; 128 x 131072 17.3/28.8, 14.5/26.0, 15.4/26.7, 21.3/32.4; 128 x 32000 6.9/18.8, 9.5/19.7, 9.4/21.2,
// 16.9/28.3; 61 x 131071 fp32 28.0/39.6, 17.6/29.3, 12.8/24.2, 12.4/24.3.
int ctas_of(int64_t rows, int64_t vocab, size_t size) {
    const int64_t bytes = vocab * (int64_t)size;
    int n = 1;
    while (n < 8 && rows * n * 2 <= (bytes > 384 << 10 ? 4 * SMS : n == 1 && bytes > 128 << 10 ? 2 * SMS : SMS) && bytes > (int64_t)n * STEP * 16 && bytes > 2 * STEP * 16) n *= 2;
    return n;
}

// Threads of a CTA.  A row's end (its sums, its alternatives) costs a CTA as much whatever its threads are: short rows, and long ones with alternatives where there are many, take fewer.  bf16 with entropy,
// 64 / 128 / 256 threads, without alternatives: 8000 x 1000 10.7 / 18.9 / 35.8 us, 8000 x 8000 26.5 / 29.6 / 39.8, 8000 x 16000 46.4 / 48.4 / 56.9, 2000 x 32000 33.2 / 28.8 / 27.2; with five: 20 x 4000 5.1 / 4.6 / 4.8, 8000 x 1000
// 27.6 / 46.1 / 75.8, 300 x 8000 6.4 / 5.7 / 7.6, 2000 x 8000 14.1 / 16.3 / 22.5, 600 x 32000 15.9 / 17.6 / 15.5, 2000 x 32000 36.9 / 34.7 / 39.5, 2000 x 131071 126 / 103 / 105.
int threads_of(int64_t rows, int64_t vocab, size_t size, int cluster, bool top) {
    const int64_t bytes = vocab * (int64_t)size;
    if (cluster > 1) return THREADS;
    // (of 1 KB: fewer pieces than groups of two threads)
    if (bytes < 1 << 10 || (bytes <= 8 << 10 && rows >= SMS) || (bytes <= 16 << 10 && rows >= 2000)) return 64;
    return bytes <= 32 << 10 || (top && bytes <= 256 << 10 && rows >= 8 * SMS) ? 128 : THREADS;
}

template <typename T, bool ENTROPY, bool TOP>
int log_probs_launch(const LogProbs &p, cudaStream_t st) {
    const int n = threads_of(p.rows, p.vocab, sizeof(T), p.cluster, TOP);
    if (n == 64) return launch_early("log_probs_kernel", log_probs_kernel<T, 64, ENTROPY, TOP>, dim3((unsigned)p.rows), 64, 0, st, dim3(1), p);
    if (n == 128) return launch_early("log_probs_kernel", log_probs_kernel<T, 128, ENTROPY, TOP>, dim3((unsigned)p.rows), 128, 0, st, dim3(1), p);
    return launch_early("log_probs_kernel", log_probs_kernel<T, THREADS, ENTROPY, TOP>, dim3((unsigned)(p.rows * p.cluster)), THREADS, 0, st, dim3(p.cluster), p);
}
template <typename T>
int log_probs_typed(LogProbs &p, cudaStream_t st) {
    p.cluster = ctas_of(p.rows, p.vocab, sizeof(T));
    if (p.top) return p.entropy ? log_probs_launch<T, true, true>(p, st) : log_probs_launch<T, false, true>(p, st);
    return p.entropy ? log_probs_launch<T, true, false>(p, st) : log_probs_launch<T, false, false>(p, st);
}

// CTAs of a row of the gradient, which do not join: so many that all rows together fill the SMs twice over, of at least a step (16 KB) each; and of at most 64 KB.
// (8192 x 131072 bf16: 657 us with one, 650 two, 640 four, 669 eight; 2048 x 32000 46, 48, 58, 91; 61 x 131071 15.6, 10.5, 8.5, 8.9.)
int parts_of(int64_t rows, int64_t vocab, size_t size) {
    int n = 1;
    while (n < 8 && ((rows * n < 8 * SMS && vocab * (int64_t)size > (int64_t)n * STEP * 16) || vocab * (int64_t)size > (int64_t)n << 16)) n *= 2;
    return n;
}

// Threads of a CTA of the gradient: fewer for many short rows.  (bf16 with an entropy's gradient, 64 / 128 / 256: 8000 x 1000 11.4 / 18.2 / 34.4 us, 8000 x 8000 45.0 / 46.7 / 60.4, 8000 x 16000 84.8 / 82.7 / 90.8, 2000 x 32000
// 50.1 / 46.5 / 45.5.)
int grad_threads_of(int64_t rows, int64_t vocab, size_t size) {
    const int64_t bytes = vocab * (int64_t)size;
    return rows < SMS || bytes > 32 << 10 ? THREADS : bytes <= 16 << 10 ? 64 : 128;
}

template <typename T, bool ENTROPY, bool ALIGNED>
int log_probs_grad_launch(const LogProbsGrad &p, int64_t rows, cudaStream_t st) {
    const int n = grad_threads_of(rows, p.vocab, sizeof(T));
    if (n == 64) return launch_early("log_probs_grad_kernel", log_probs_grad_kernel<T, 64, ENTROPY, ALIGNED>, dim3((unsigned)(rows * p.parts)), 64, 0, st, dim3(1), p);
    if (n == 128) return launch_early("log_probs_grad_kernel", log_probs_grad_kernel<T, 128, ENTROPY, ALIGNED>, dim3((unsigned)(rows * p.parts)), 128, 0, st, dim3(1), p);
    return launch_early("log_probs_grad_kernel", log_probs_grad_kernel<T, THREADS, ENTROPY, ALIGNED>, dim3((unsigned)(rows * p.parts)), THREADS, 0, st, dim3(1), p);
}
template <typename T>
int log_probs_grad_typed(LogProbsGrad &p, int64_t rows, cudaStream_t st) {
    p.parts = parts_of(rows, p.vocab, sizeof(T));
    const uintptr_t apart = (reinterpret_cast<uintptr_t>(p.logits) - reinterpret_cast<uintptr_t>(p.grad)) % 16;
    const bool aligned = apart == 0 && (rows == 1 || (p.stride - p.vocab) * (int64_t)sizeof(T) % 16 == 0);
    if (p.e) return aligned ? log_probs_grad_launch<T, true, true>(p, rows, st) : log_probs_grad_launch<T, true, false>(p, rows, st);
    return aligned ? log_probs_grad_launch<T, false, true>(p, rows, st) : log_probs_grad_launch<T, false, false>(p, rows, st);
}

}  // namespace

int token_log_probs(const void *logits, int dtype, int64_t rows, int64_t vocab, int64_t stride, const int64_t *tokens, float *log_probs, float *entropy,
                    int top, float *top_log_probs, int64_t *top_tokens, float *stats, cudaStream_t st) {
    LogProbs p = {logits, tokens, log_probs, entropy, top_log_probs, top_tokens, (float4 *)stats, stride, rows, (int)vocab, top, 1};
    if (dtype == BW_F32) return log_probs_typed<float>(p, st);
    if (dtype == BW_F16) return log_probs_typed<__half>(p, st);
    return log_probs_typed<__nv_bfloat16>(p, st);
}

int token_log_probs_grad(const void *logits, int dtype, int64_t rows, int64_t vocab, int64_t stride, const int64_t *tokens, const float *stats,
                         const float *g, const float *e, int top, const int64_t *top_tokens, const float *g_top, void *grad, cudaStream_t st) {
    LogProbsGrad p = {logits, grad, tokens, top_tokens, (const float4 *)stats, g, e, g_top, stride, (int)vocab, top, 1};
    if (dtype == BW_F32) return log_probs_grad_typed<float>(p, rows, st);
    if (dtype == BW_F16) return log_probs_grad_typed<__half>(p, rows, st);
    return log_probs_grad_typed<__nv_bfloat16>(p, rows, st);
}

}  // namespace bw
