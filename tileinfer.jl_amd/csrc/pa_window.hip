// Split-KV decode with a sliding window, and over 8-bit block caches: the forms FP8 and WIN of the paged decode kernel
// (pa_decode.hpp), their launches and the paths of ti_window_attention.
//
// Bound as without a window: HBM for batches (32 tokens on 4096 keys of an 8-bit block cache, 32 / 8 heads of 128: 46.2 us,
// 5.8 TB/s; 32 tokens on 100 to 32768 keys with a window of 4096, bf16, 71 us, 7.0 TB/s of the keys seen, some of which the
// Infinity Cache holds), the chain of loads and the combine's launch for one sequence (a window of 1024: 7.9 us, 5.1 of them
// here). Windows that are full hold the same keys, so a batch is not shared out by length
// (8 INT8 sequences on 8000 to 32768 keys with a window of 8192: 39.1 -> 31.7 us).
#include "pa_decode.hpp"

using namespace ti;
using namespace ti_decode;

namespace {

template <int D, bool INT8, bool PG16, bool FP8, bool WIN>
void launch_decode_w(const DecodeParams &p, int rowb, dim3 grid, hipStream_t s) {
    // INT8 launches of at most one work-group per CU work on their steps' tiles together, as without a window
    if constexpr (INT8 && D == 128) {
        if (rowb == 1 && (unsigned long long)grid.x * grid.y * grid.z <= 256) {
            decode_kernel<D, 1, INT8, PG16, 4, 1, true, false, false, FP8, WIN><<<grid, 256, 0, s>>>(p);
            return;
        }
    }
    switch (rowb) {
        case 1: decode_kernel<D, 1, INT8, PG16, 4, 1, false, false, false, FP8, WIN><<<grid, 256, 0, s>>>(p); break;
        case 2: decode_kernel<D, 2, INT8, PG16, 4, 1, false, false, false, FP8, WIN><<<grid, 256, 0, s>>>(p); break;
        default: decode_kernel<D, 2, INT8, PG16, 4, 2, false, false, false, FP8, WIN><<<grid, 256, 0, s>>>(p); break;
    }
}

template <int D>
void launch_decode(const DecodeParams &p, int kind, bool window, int rowb, dim3 grid, hipStream_t s) {
    const bool whole = p.P % 16 == 0 && p.pshift >= 0;   // a tile lies in one page
    if (kind == TI_KV_FP8) {
        if (window) launch_decode_w<D, false, true, true, true>(p, rowb, grid, s);
        else launch_decode_w<D, false, true, true, false>(p, rowb, grid, s);
    } else if (kind == TI_KV_INT8) {
        if (whole) launch_decode_w<D, true, true, false, true>(p, rowb, grid, s);
        else launch_decode_w<D, true, false, false, true>(p, rowb, grid, s);
    } else {
        if (whole) launch_decode_w<D, false, true, false, true>(p, rowb, grid, s);
        else launch_decode_w<D, false, false, false, true>(p, rowb, grid, s);
    }
}

}  // namespace

// Steps of a window that the decode kernel takes, and the others (as without one: api.hip).
bool ti_window_decodes(const ti_attention_args *a, const ti_kv_cache *c) {
    const int rows = a->q_heads / c->kv_heads * a->max_query_len;
    return a->max_query_len <= 16 && (rows <= 32 || (a->max_query_len == 1 && rows <= 64));
}

int ti_launch_decode_window(const ti_attention_args *a, const ti_kv_cache *c, const ti_decode_plan &pl, ti_window win, hipStream_t s) {
    DecodeParams p = decode_params(a, c, pl);
    p.window = win.size;
    p.sinks = win.sinks;
    const int rowb = (pl.rows + 15) / 16;
    const dim3 grid = pl.flat ? dim3(pl.flat, c->kv_heads, 1) : dim3(pl.splits, c->kv_heads, a->num_seqs);
    if (c->head_dim == 128) launch_decode<128>(p, c->kind, win.size > 0, rowb, grid, s);
    else launch_decode<64>(p, c->kind, win.size > 0, rowb, grid, s);
    if (hipGetLastError() != hipSuccess) return TI_ERR_LAUNCH;
    if (pl.splits == 1) return TI_OK;
    return ti_launch_combine(a, c, pl.rows, pl.flat ? pl.flat / a->num_seqs : pl.splits, s, pl.flat, p.meta);
}
