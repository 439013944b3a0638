// The tiled kernels of attention over the quantised cache, compiled for a window and sinks: only the tiles of 16 tokens that hold a visible
// one are in the line of work, and tokens of those tiles that are not visible are masked like those behind the sequence.
//
// 64 sequences of up to 131071 tokens, window 4096 and 64 sinks, 32 and 8 heads of 128, 8 bits, bf16: 99.5 us with the join, 5.7 TB/s of the visible rows, 0.87 of the measured
// copy rate (on the general kernel 5.5 ms); 16 of up to 8192, window 1000, 4 bits: 11.2 to 12.0 us. Those are 128 units of 33 steps, which take two CTAs a unit: five steps of a warp and the
// join of a cluster. One CTA (nine steps) takes 11.3, two 12.0, four (three steps) 12.1: a cluster's start and join cost what its fewer steps save.
#include "kv_attend_tiles.cuh"

namespace bw {

int attend_window_tiles(const AttendArgs &a, int64_t batch, int dtype, int bits, void *workspace, cudaStream_t st) {
    FastArgs f = {};
    if (!fast_args(f, batch, a.heads, a.kv_heads, a.dim, bits, a.pages, a.page_size, a.max_pages, a.window, a.sinks)) return BW_ERR_UNSUPPORTED;
    f.a = a;
    f.slots = (float *)workspace;
    return dtype == BW_F16 ? launch_bits<true, __half>(f, bits, st) : launch_bits<true, __nv_bfloat16>(f, bits, st);
}

}  // namespace bw
