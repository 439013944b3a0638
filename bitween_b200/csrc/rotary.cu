// Rotary positions (bw_rotate) and appends to the quantised cache with the rotation on the way (bw_kv_append_rotated).
//
// Pair j of a row's first R values, at (j, j + R/2) or (2j, 2j+1), is turned by the angle of its axis's position:
//     (a, b) -> (a c - b s, b c + a s),   (c, s) = table[position][j]
// The transposed rotation, which the gradient needs, has -s.
//
// Bound by the bytes of the rows.  A thread has 16 values of a head, both of each pair among them, and takes the same place of up to eight heads of its token, so
// that cosines and sines (64 bytes, from L2) are read once for them.  16384 tokens of 32 and 8 heads of 128, bf16: 58.2 us, 5.9 TB/s, 0.90 of the measured copy rate (four heads a thread
// 66.1 us, 16 59.6; CTAs of 256 threads 65.0; loads of two heads in flight instead of four 60.7).  The same rows rotated, 8 heads of keys and values quantised to 4 bits: 71.8 us, 6.0 TB/s
// (with the means of kv_cache.cu; one value a load and a division each: 790).  Pairs whose axes change from one to the next look their positions up one by one: 62.6 and 77.6 us.
#include "early_launch.cuh"
#include "kv_rows.cuh"
#include "rotary.cuh"

namespace bw {
namespace {

constexpr int THREADS = 128, BATCH = 4;      // of a CTA; heads whose loads are in flight together

struct RotateRows {
    const void *x[2];
    void *out[2];
    int64_t stride[2], head_stride[2], tokens;
    int heads[2], dim;
    int slots;                           // threads of a piece of a token: each takes every slots-th head
    Divisor by_pieces, by_slots;
};

// The rows of thread `i` of a call.
template <typename T>
__device__ __forceinline__ void rotate_rows(const RotateRows &p, const Rotary &r, uint32_t i) {
    const uint32_t rest = p.by_pieces(i), token = p.by_slots(rest);
    const int piece = (int)(i - rest * (uint32_t)(p.dim / 16)), slot = (int)(rest - token * (uint32_t)p.slots), heads = p.heads[0] + p.heads[1];
    if (token >= p.tokens) return;
    const Turn turn(r, token, piece, true);
    for (int h0 = slot; h0 < heads; h0 += BATCH * p.slots) {
        Eight<T> a[BATCH], b[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int h = h0 + k * p.slots;
            if (h >= heads) break;
            const T *x = h < p.heads[0] ? (const T *)p.x[0] + (int64_t)token * p.stride[0] + h * p.head_stride[0]
                                        : (const T *)p.x[1] + (int64_t)token * p.stride[1] + (h - p.heads[0]) * p.head_stride[1];
            a[k].load(x + turn.at0);
            b[k].load(x + turn.at1);
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int h = h0 + k * p.slots;
            if (h >= heads) break;
            if (turn.turns) {
                float x[16];
                a[k].get(x);
                b[k].get(x + 8);
                turn(r, x);
                a[k].put(x);
                b[k].put(x + 8);
            }
            T *out = h < p.heads[0] ? (T *)p.out[0] + ((int64_t)token * p.heads[0] + h) * p.dim : (T *)p.out[1] + ((int64_t)token * p.heads[1] + h - p.heads[0]) * p.dim;
            a[k].store(out + turn.at0);
            b[k].store(out + turn.at1);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) rotate_kernel(const RotateRows p, const Rotary r) {
    pdl_wait();
    pdl_launch_dependents();
    rotate_rows<T>(p, r, blockIdx.x * THREADS + threadIdx.x);
}

// Any size and stride: a warp the heads of a token slots apart from `slot`, a lane every 32nd pair, whose cosine and sine it keeps for all of them.  (The 16384 tokens from
// above off a 16-byte boundary 114 us, with 20 pairs of a head 156; a row a warp and each value by itself 750.)
template <typename T>
__device__ __forceinline__ void rotate_any(const RotateRows &p, const Rotary &r, int64_t token, int slot) {
    const int lane = threadIdx.x % 32, heads = p.heads[0] + p.heads[1];
    auto rows = [&](int h, const T *&x, T *&out) {
        if (h < p.heads[0]) {
            x = (const T *)p.x[0] + token * p.stride[0] + h * p.head_stride[0];
            out = (T *)p.out[0] + (token * p.heads[0] + h) * p.dim;
        } else {
            x = (const T *)p.x[1] + token * p.stride[1] + (h - p.heads[0]) * p.head_stride[1];
            out = (T *)p.out[1] + (token * p.heads[1] + h - p.heads[0]) * p.dim;
        }
    };
    for (int pair = lane; pair < r.pairs; pair += 32) {
        const int first = r.interleaved ? 2 * pair : pair, second = r.interleaved ? first + 1 : pair + r.pairs;
        const float2 t = turn_of(r, token, pair);
        for (int h = slot; h < heads; h += p.slots) {
            const T *x;
            T *out;
            rows(h, x, out);
            const float u = to_f32(x[first]), v = to_f32(x[second]);
            out[first] = from_f32<T>(turned_first(u, v, t));
            out[second] = from_f32<T>(turned_second(u, v, t));
        }
    }
    for (int d = 2 * r.pairs + lane; d < p.dim; d += 32)
        for (int h = slot; h < heads; h += p.slots) {
            const T *x;
            T *out;
            rows(h, x, out);
            out[d] = x[d];
        }
}

template <typename T>
__global__ void __launch_bounds__(256) rotate_general_kernel(const RotateRows p, const Rotary r) {
    const int64_t i = (int64_t)blockIdx.x * 8 + threadIdx.x / 32, token = i / p.slots;
    if (token < p.tokens) rotate_any<T>(p, r, token, (int)(i - token * p.slots));
}

struct AppendRotated {
    RotateRows q;                        // one tensor, or none (no heads)
    const void *k, *v;
    const int64_t *slots;
    int32_t *codes[2];
    __half2 *params;
    KvRows rows;
    int kv_slots;                        // threads of a piece of a token, of keys and values
    unsigned kv_ctas;                    // the first CTAs take those, the others queries
    Divisor by_kv_slots;
};

// The 16 values of a thread, eight at `at0` and eight at `at1`, as codes of a row whose ends are known.
template <int BITS>
__device__ __forceinline__ void store_codes(const float (&x)[16], float lo, float hi, int32_t *row, int at0, int at1, __half2 *constants, bool first) {
    constexpr float Q = (1 << BITS) - 1, RQ = 1.0f / Q;
    constexpr int WORDS = BITS == 8 ? 2 : 1, EACH = 8 / WORDS;
    const float span = div_by_recip(__fsub_rn(hi, lo), Q, RQ);
    const bool ok = span <= 65504.0f;        // (not with a NaN or an infinity in the row, nor beyond fp16's range)
    const __half scale = scale_up(span);
    const float s = __half2float(scale), rs = __frcp_rn(s), z = rintf(div_by_recip(-lo, s, rs));
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint32_t words[WORDS] = {};
        if (ok) {
            float c[8];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float2 t = fadd2(div_by_recip2(make_float2(x[8 * half + i], x[8 * half + i + 1]), s, rs), make_float2(z, z));
                const float2 y = fadd2(make_float2(fminf(t.x, Q), fminf(t.y, Q)), make_float2(MAGIC, MAGIC));
                c[i] = y.x;
                c[i + 1] = y.y;
            }
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                uint32_t word = 0, extra = 0;
#pragma unroll
                for (int i = EACH - 1; i >= 0; --i) {
                    word = (word << BITS) + __float_as_uint(c[w * EACH + i]);
                    extra = (extra << BITS) + MAGIC_BITS;
                }
                words[w] = word - extra;
            }
        }
        uint8_t *to = reinterpret_cast<uint8_t *>(row) + (half ? at1 : at0) * BITS / 8;
        if constexpr (BITS == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(words[0], words[1]);
        else if constexpr (BITS == 4) *reinterpret_cast<uint32_t *>(to) = words[0];
        else *reinterpret_cast<uint16_t *>(to) = (uint16_t)words[0];
    }
    if (first) *constants = ok ? __halves2half2(scale, __float2half_rn(z)) : __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0));
}

// A group of lanes (a power of two) a row of k and the row of v beside it, of every kv_slots-th head of a token.
template <typename T, int BITS>
__global__ void __launch_bounds__(THREADS) kv_append_rotated_kernel(const AppendRotated p, const Rotary r) {
    pdl_wait();
    pdl_launch_dependents();
    if (blockIdx.x >= p.kv_ctas) {
        rotate_rows<T>(p.q, r, (blockIdx.x - p.kv_ctas) * THREADS + threadIdx.x);
        return;
    }
    const int lanes = p.rows.lanes, piece = threadIdx.x % lanes;
    const uint32_t rest = blockIdx.x * (THREADS / lanes) + threadIdx.x / lanes, token = p.by_kv_slots(rest);
    const int slot0 = (int)(rest - token * (uint32_t)p.kv_slots);
    const int64_t slot = token < p.rows.tokens ? __ldcg(p.slots + token) : -1;
    const bool live = slot >= 0 && slot < p.rows.slots && 16 * piece < p.rows.dim;
    const Turn turn(r, token, piece, live);
    for (int h0 = 0; h0 < p.rows.heads; h0 += p.kv_slots) {      // (alike for all lanes: they meet in the ends of the rows)
        const int h = h0 + slot0;
        const bool mine = live && h < p.rows.heads;
        float x[2][16] = {}, lo[2] = {}, hi[2] = {};
        if (mine) {
            Eight<T> a[2], b[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const T *from = (const T *)(j ? p.v : p.k) + (int64_t)token * p.rows.stride[j] + h * p.rows.head_stride[j];
                a[j].load(from + (j ? 16 * piece : turn.at0));
                b[j].load(from + (j ? 16 * piece + 8 : turn.at1));
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                a[j].get(x[j]);
                b[j].get(x[j] + 8);
            }
            turn(r, x[0]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    lo[j] = min_nan(lo[j], x[j][i]);
                    hi[j] = max_nan(hi[j], x[j][i]);
                }
        }
        for (int d = lanes / 2; d; d >>= 1)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                lo[j] = min_nan(lo[j], __shfl_xor_sync(0xffffffffu, lo[j], d));
                hi[j] = max_nan(hi[j], __shfl_xor_sync(0xffffffffu, hi[j], d));
            }
        if (!mine) continue;
        const int64_t to = cache_row(p.rows, slot, h);
#pragma unroll
        for (int j = 0; j < 2; ++j)
            store_codes<BITS>(x[j], lo[j], hi[j], p.codes[j] + to * p.rows.words, j ? 16 * piece : turn.at0, j ? 16 * piece + 8 : turn.at1, p.params + 2 * to + j, piece == 0);
    }
}

// Any size and stride: a warp a row of k or v, or the heads of q that are slots apart (316 to 330 us).
template <typename T, int BITS>
__global__ void __launch_bounds__(256) kv_append_rotated_general_kernel(const AppendRotated p, const Rotary r) {
    constexpr float Q = (1 << BITS) - 1, RQ = 1.0f / Q;
    __shared__ uint8_t s_codes[8][256];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, kv = p.rows.heads, all = p.q.slots + 2 * kv;
    const int64_t row = (int64_t)blockIdx.x * 8 + warp, token = row / all;
    if (token >= p.rows.tokens) return;
    int h = (int)(row - token * all);
    if (h >= 2 * kv) {
        rotate_any<T>(p.q, r, token, h - 2 * kv);
        return;
    }
    const int j = h >= kv;
    if (j) h -= kv;
    const int64_t slot = p.slots[token];
    if (slot < 0 || slot >= p.rows.slots) return;
    const T *x = (const T *)(j ? p.v : p.k) + token * p.rows.stride[j] + h * p.rows.head_stride[j];
    float v[8], lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        v[i] = d >= p.rows.dim ? 0.0f : j ? to_f32(x[d]) : turned_value(r, x, token, d);
        lo = min_nan(lo, v[i]);
        hi = max_nan(hi, v[i]);
    }
    for (int d = 16; d; d >>= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, d));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, d));
    }
    const float span = div_by_recip(__fsub_rn(hi, lo), Q, RQ);
    const bool ok = span <= 65504.0f;
    const __half scale = scale_up(span);
    const float s = __half2float(scale), rs = __frcp_rn(s), z = rintf(div_by_recip(-lo, s, rs));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        if (d < p.rows.dim) s_codes[warp][d] = ok ? (uint8_t)fminf(rintf(__fadd_rn(div_by_recip(v[i], s, rs), z)), Q) : 0;
    }
    __syncwarp();
    const int64_t to = cache_row(p.rows, slot, h);
    for (int w = lane; w < p.rows.words; w += 32) {
        uint32_t word = 0;
        for (int i = 0; i < 32 / BITS; ++i) word |= (uint32_t)s_codes[warp][w * (32 / BITS) + i] << (i * BITS);
        p.codes[j][to * p.rows.words + w] = (int32_t)word;
    }
    if (lane == 0) p.params[2 * to + j] = ok ? __halves2half2(scale, __float2half_rn(z)) : __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0));
}

Rotary rotary_of(const bw_rotary &r, bool inverse) {
    Rotary p = {};
    p.table = (const float2 *)r.table;
    p.positions = r.positions;
    p.max_positions = r.max_positions;
    p.axis_stride = r.axis_stride;
    p.pairs = r.rotary_dim / 2;
    p.interleaved = r.interleaved != 0;
    p.sign = inverse ? -1.0f : 1.0f;
    for (int i = 0; i < p.pairs; ++i) p.axis[i] = r.axes ? r.axes[i] : 0;
    for (int piece = 0; 8 * piece + 7 < p.pairs; ++piece) {
        bool one = true;
        for (int i = 1; i < 8; ++i) one = one && p.axis[8 * piece + i] == p.axis[8 * piece];
        p.whole |= (uint32_t)one << piece;
    }
    return p;
}

// Whether rows can be taken in pieces of 16 values, 16 bytes a load.
bool pieces_ok(const Rotary &r, int dim) { return dim <= 256 && dim % 16 == 0 && r.pairs % 8 == 0; }
bool rows_ok(const void *x, int64_t stride, int64_t head_stride, size_t size) {
    return aligned_to(x, 16) && stride * (int64_t)size % 16 == 0 && head_stride * (int64_t)size % 16 == 0;
}
// Threads of a piece of a token: eight heads a thread where that leaves 1024 threads an SM, else four, two or one (figures at the top).
int slots_of(int64_t tokens, int dim, int heads) {
    int each = 8;
    while (each > 1 && tokens * (dim / 16) * ((heads + each - 1) / each) < 148 * 1024) each /= 2;
    return (heads + each - 1) / each;
}
// Warps of a token on the general kernel: eight heads a warp where that leaves 32 warps an SM, else four, two or one.
int warps_of(int64_t tokens, int heads) {
    int each = 8;
    while (each > 1 && tokens * ((heads + each - 1) / each) < 148 * 32) each /= 2;
    return (heads + each - 1) / each;
}
// The threads of a call's rows; 0 where the general kernel takes them.
int64_t fast_rows(RotateRows &p, const Rotary &r, size_t size) {
    const int heads = p.heads[0] + p.heads[1];
    if (!pieces_ok(r, p.dim)) return 0;
    for (int i = 0; i < 2; ++i)
        if (p.heads[i] && (!rows_ok(p.x[i], p.stride[i], p.head_stride[i], size) || !aligned_to(p.out[i], 16))) return 0;
    p.slots = slots_of(p.tokens, p.dim, heads);
    p.by_pieces = divisor((uint32_t)(p.dim / 16));
    p.by_slots = divisor((uint32_t)p.slots);
    const int64_t threads = p.tokens * (p.dim / 16) * p.slots;
    return threads + THREADS < (int64_t)1 << 32 ? threads : 0;
}

template <typename T>
int rotate_typed(RotateRows &p, const Rotary &r, cudaStream_t st) {
    if (const int64_t threads = fast_rows(p, r, sizeof(T)))
        return launch_early("rotate_kernel", rotate_kernel<T>, dim3((unsigned)((threads + THREADS - 1) / THREADS)), THREADS, 0, st, dim3(1), p, r);
    p.slots = warps_of(p.tokens, p.heads[0] + p.heads[1]);
    rotate_general_kernel<T><<<(unsigned)((p.tokens * p.slots + 7) / 8), 256, 0, st>>>(p, r);
    return check_launch("rotate_general_kernel");
}

template <typename T, int BITS>
int append_rotated_typed(AppendRotated &p, const Rotary &r, cudaStream_t st) {
    const KvRows &k = p.rows;
    bool fast = pieces_ok(r, k.dim) && rows_ok(p.k, k.stride[0], k.head_stride[0], sizeof(T)) && rows_ok(p.v, k.stride[1], k.head_stride[1], sizeof(T));
    int64_t q_threads = 0;
    if (fast && p.q.heads[0]) fast = (q_threads = fast_rows(p.q, r, sizeof(T))) > 0;
    p.kv_slots = slots_of(k.tokens, k.dim, k.heads);
    const int64_t kv_ctas = (k.tokens * p.kv_slots * k.lanes + THREADS - 1) / THREADS, ctas = kv_ctas + (q_threads + THREADS - 1) / THREADS;
    if (fast && ctas < (int64_t)1 << 31 && kv_ctas * THREADS < (int64_t)1 << 32) {
        p.kv_ctas = (unsigned)kv_ctas;
        p.by_kv_slots = divisor((uint32_t)p.kv_slots);
        return launch_early("kv_append_rotated_kernel", kv_append_rotated_kernel<T, BITS>, dim3((unsigned)ctas), THREADS, 0, st, dim3(1), p, r);
    }
    p.q.slots = p.q.heads[0] ? warps_of(k.tokens, p.q.heads[0]) : 0;
    const int64_t rows = k.tokens * (p.q.slots + 2 * k.heads);
    kv_append_rotated_general_kernel<T, BITS><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(p, r);
    return check_launch("kv_append_rotated_general_kernel");
}
template <typename T>
int append_rotated_bits(AppendRotated &p, const Rotary &r, int bits, cudaStream_t st) {
    return bits == 2 ? append_rotated_typed<T, 2>(p, r, st) : bits == 4 ? append_rotated_typed<T, 4>(p, r, st) : append_rotated_typed<T, 8>(p, r, st);
}

}  // namespace

int rotate(const bw_rotary &rotary, int64_t tokens, int dim, int dtype, bool inverse, const void *const *x, const int *heads, const int64_t *strides,
           void *const *out, cudaStream_t st) {
    RotateRows p = {};
    p.tokens = tokens;
    p.dim = dim;
    for (int i = 0; i < 2; ++i) {
        p.x[i] = x[i];
        p.out[i] = out[i];
        p.heads[i] = heads[i];
        p.stride[i] = strides[2 * i];
        p.head_stride[i] = strides[2 * i + 1];
    }
    const Rotary r = rotary_of(rotary, inverse);
    if (dtype == BW_F32) return rotate_typed<float>(p, r, st);
    if (dtype == BW_F16) return rotate_typed<__half>(p, r, st);
    return rotate_typed<__nv_bfloat16>(p, r, st);
}

int kv_append_rotated(const bw_rotary &rotary, const void *q, int q_heads, int64_t q_stride, int64_t q_head_stride, void *q_out, const void *k, const void *v,
                      int dtype, int64_t tokens, const int64_t *strides, const int64_t *slots, int heads, int dim, int bits, int64_t pages, int page_size,
                      int32_t *kc, int32_t *vc, void *params, cudaStream_t st) {
    AppendRotated p = {};
    p.q.x[0] = q;
    p.q.out[0] = q_out;
    p.q.heads[0] = q_heads;
    p.q.stride[0] = q_stride;
    p.q.head_stride[0] = q_head_stride;
    p.q.tokens = tokens;
    p.q.dim = dim;
    p.k = k;
    p.v = v;
    p.slots = slots;
    p.codes[0] = kc;
    p.codes[1] = vc;
    p.params = (__half2 *)params;
    p.rows = kv_rows(tokens, heads, dim, bits, pages, page_size);
    for (int i = 0; i < 2; ++i) {
        p.rows.stride[i] = strides[2 * i];
        p.rows.head_stride[i] = strides[2 * i + 1];
    }
    const Rotary r = rotary_of(rotary, false);
    if (dtype == BW_F32) return append_rotated_bits<float>(p, r, bits, st);
    if (dtype == BW_F16) return append_rotated_bits<__half>(p, r, bits, st);
    return append_rotated_bits<__nv_bfloat16>(p, r, bits, st);
}

}  // namespace bw
