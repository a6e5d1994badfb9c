// The pages that a query keeps by the bounds of their keys (page_bounds.hip).
//
// A query row q (one token, one query head) as whole numbers w_d = rint(q_d 2^-e), e the least exponent
// with |q| <= 127 2^e, has with any key inside a page's bounds at most the product
//   2^e 2^e_page sum_d (w_d hi_d where w_d > 0, else w_d lo_d) = 2^e 2^e_page (relu(w) . hi + min(w, 0) . lo):
// one int8 matrix product of depth 2 D, whose sums stay below 2^22 and are exact. The score of a page
// for a token and KV head is the largest over the G query heads, two multiplications by powers of
// two: exact, so equal scores are equal bounds and not roundings, and the kept pages do not depend
// on how the work is split.
//
// Scores become 32-bit keys in the scores' order, 0 for pages that are not up for choice (those kept
// anyway, and those past the last visible one). The key of the last page kept by score is found by
// bisection between the smallest and the largest key, counting the keys above the middle: it ends
// when the count is right, after about log2 of the pages and a few steps, and at the latest after 32
// (equal keys). Then one pass over the pages in order writes the kept ones.
//
// Two forms. select_kernel holds a token tile's keys in LDS and does both steps in one launch.
// scores_kernel and keep_kernel share a tile's pages out over several work-groups, the keys going
// through the workspace, for few tokens over wide tables and for tables that LDS does not hold.
#include "page_bounds.hpp"

using namespace ti;
using namespace ti_pages;

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int WAVES = 16, THREADS = WAVES * 64;
constexpr int ROUND = 256;   // keys read by a wave at once: rows of keys are padded to it with zeros

struct SelectParams {
    const void *q;
    const int8_t *bounds;
    const float *scale;
    const int32_t *positions, *qsl, *bt;
    int32_t *tables, *lengths;
    uint32_t *keys;   // two launches: [total][Hk][pitch]
    int bt_stride, num_pages, P, Hk, Hq, G, nmax, total, keep, sinks, window, causal, f32;
    int pitch, split;   // keys per (token, KV head); work-groups that share a token tile's pages
};

// What one token sees: pages [0, seen), of which [c0, c1) are up for choice and `need` kept by score.
struct Seen {
    int last, seen, c0, c1, kept, need;
    __device__ Seen(const SelectParams &p, const Step &st, int t) {
        last = st.start + (p.causal ? t : st.n - 1);
        seen = min(last / p.P + 1, p.bt_stride);
        c0 = min(p.sinks, seen);
        c1 = max(c0, seen - p.window);
        kept = min(seen, p.keep);
        need = kept - (seen - (c1 - c0));
    }
};

// Larger score, larger key, never 0; NaN (an infinite page scale times 0) counts as the largest.
__device__ __forceinline__ uint32_t order_key(float x) {
    x += 0.0f;   // -0 and 0 are one score
    const uint32_t u = __float_as_uint(x);
    return x != x ? 0xffffffffu : ((int32_t)u < 0 ? ~u : u | 0x80000000u);
}

// The largest of GP neighbouring lanes, in all of them (GP a power of two up to 16).
template <int CTRL> __device__ __forceinline__ float dpp_max(float x) {
    return fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, false)));
}
template <int GP> __device__ __forceinline__ float group_max(float x) {
    if (GP >= 2) x = dpp_max<0xb1>(x);    // quad_perm 1 0 3 2
    if (GP >= 4) x = dpp_max<0x4e>(x);    // quad_perm 2 3 0 1
    if (GP >= 8) x = dpp_max<0x141>(x);   // row_half_mirror: the other quad of eight lanes
    if (GP >= 16) x = dpp_max<0x140>(x);  // row_mirror: the other half of sixteen
    return x;
}

// A tile of RT x 16 query rows: rows of a token are its G heads, padded to GP (a power of two up to 16);
// WIDE (G > 16): one token's heads over all RT blocks. TT tokens a tile.
template <int GP, int RT, bool WIDE> struct Tile {
    static constexpr int ROWS = RT * 16, TT = WIDE ? 1 : ROWS / GP;
};

// The whole-number operands of a tile's rows in LDS: relu(w) then min(w, 0), and 2^e (a row that is not
// finite: zeros). 16 lanes per row.
template <int D, int GP, int RT, bool WIDE>
__device__ __forceinline__ void quantize_rows(const SelectParams &p, const Step &st, int h, int t0, int tid, int8_t (*w)[2 * D],
                                              float *forth) {
    constexpr int E = D / 16;
    for (int r = tid / 16; r < RT * 16; r += THREADS / 16) {
        const int t = WIDE ? t0 : t0 + r / GP, g = WIDE ? r : r % GP, c = (tid & 15) * E;
        const bool ok = t < st.n && g < p.G;
        const size_t src = ((size_t)(st.tok0 + (ok ? t : t0)) * p.Hq + h * p.G + (ok ? g : 0)) * D + c;
        float x[E], a = 0.0f;
        if (p.f32) {
#pragma unroll
            for (int i = 0; i < E; i++) x[i] = Elt<float>::ld((const float *)p.q, src + i);
        } else {
#pragma unroll
            for (int i = 0; i < E; i++) x[i] = Elt<uint16_t>::ld((const uint16_t *)p.q, src + i);
        }
#pragma unroll
        for (int i = 0; i < E; i++) {
            a = fabsf(x[i]) < INFINITY ? fmaxf(a, fabsf(x[i])) : INFINITY;
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) a = fmaxf(a, __shfl_xor(a, o));
        const bool fine = a < INFINITY;
        const int e = bound_exponent(fine ? a : 0.0f);
        const float back = fine ? power(-e) : 0.0f;
        uint32_t up[E / 4], dn[E / 4];
#pragma unroll
        for (int i = 0; i < E / 4; i++) {
            up[i] = dn[i] = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int v = fine ? (int)rintf(x[4 * i + k] * back) : 0;
                up[i] |= (uint32_t)max(v, 0) << (8 * k);
                dn[i] |= ((uint32_t)min(v, 0) & 255u) << (8 * k);
            }
        }
#pragma unroll
        for (int i = 0; i < E / 4; i++) {
            *reinterpret_cast<uint32_t *>(&w[r][c + 4 * i]) = up[i];
            *reinterpret_cast<uint32_t *>(&w[r][D + c + 4 * i]) = dn[i];
        }
        if ((tid & 15) == 0) forth[r] = power(e);
    }
}

// The keys of a tile's tokens for the 16-page tiles j = first, first + step, ... < ntiles, by one wave:
// S = bounds W on v_mfma_i32_16x16x64_i8 (A: lane l holds page l % 16's bytes 16 (l / 16) .. + 16 of each
// 64; B: a query row's, the same way), so lane l gets row l % 16's products with pages 4 (l / 16) .. + 3,
// and the heads of a token are neighbouring lanes. dst(t, page) is where four keys of token t0 + t go.
template <int D, int GP, int RT, bool WIDE, typename Dst>
__device__ __forceinline__ void score_pages(const SelectParams &p, const Step &st, int b, int h, int t0, int lane, int first, int step,
                                            int ntiles, int most, const int8_t (*w)[2 * D], const float *forth, Dst dst) {
    constexpr int NK = 2 * D / 64;
    constexpr int TPB = WIDE ? 1 : 16 / GP;   // tokens per 16-row block
    const int r16 = lane & 15, kg = lane >> 4;
    const int32_t *bt = p.bt + (size_t)b * p.bt_stride;
    i32x4 q[RT][NK];
    float f[RT];
    int c0[RT], c1[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
#pragma unroll
        for (int i = 0; i < NK; i++) q[rt][i] = *reinterpret_cast<const i32x4 *>(&w[rt * 16 + r16][i * 64 + kg * 16]);
        f[rt] = forth[rt * 16 + r16];
        const int t = WIDE ? t0 : t0 + rt * TPB + r16 / GP;
        const Seen s(p, st, min(t, st.n - 1));
        c0[rt] = s.c0;
        c1[rt] = t < st.n ? s.c1 : 0;
    }
    struct Page {
        i32x4 b[NK];
        float scale;
    };
    auto load = [&](int j, Page &pg) {
        const int id = page_of(bt, min(j * 16 + r16, most - 1), p.bt_stride, p.num_pages);
        const size_t at = (size_t)id * p.Hk + h;
        const int8_t *src = p.bounds + at * 2 * D + kg * 16;
#pragma unroll
        for (int i = 0; i < NK; i++) pg.b[i] = *reinterpret_cast<const i32x4 *>(src + i * 64);
        pg.scale = p.scale[at];
    };
    auto use = [&](int j, const Page &pg) {
        float ps[4], s[4];
#pragma unroll
        for (int k = 0; k < 4; k++) ps[k] = __shfl(pg.scale, 4 * kg + k);
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            i32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < NK; i++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(pg.b[i], q[rt][i], acc, 0, 0, 0);
            const bool head = (WIDE ? rt * 16 + r16 : r16 % GP) < p.G;   // a padding row counts for nothing
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float x = head ? (float)acc[k] * f[rt] : -INFINITY;
                s[k] = WIDE && rt > 0 ? fmaxf(s[k], x) : x;
            }
            if (WIDE && rt < RT - 1) continue;
            u32x4 key;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int page = j * 16 + 4 * kg + k;
                const uint32_t o = order_key(group_max<GP>(s[k]) * ps[k]);
                key[k] = page >= c0[rt] && page < c1[rt] ? o : 0u;
            }
            const int t = WIDE ? 0 : rt * TPB + r16 / GP;
            if (r16 % GP == 0 && t0 + t < st.n) *reinterpret_cast<u32x4 *>(dst(t, j * 16 + 4 * kg)) = key;
        }
    };
    int j = first;
    if constexpr (RT > 1) {   // its operands leave no registers for a second set
        Page pg;
        for (; j < ntiles; j += step) {
            load(j, pg);
            use(j, pg);
        }
        return;
    }
    // two sets in turn: the next tile's loads are issued before this one is worked on
    Page pa, pb;
    if (j < ntiles) {
        load(j, pa);
        while (true) {
            load(min(j + step, ntiles - 1), pb);
            use(j, pa);
            j += step;
            if (j >= ntiles) break;
            load(min(j + step, ntiles - 1), pa);
            use(j, pb);
            j += step;
            if (j >= ntiles) break;
        }
    }
}

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    return v;
}

// Writes one token's kept pages and its number of keys. keys: `span` of them (a multiple of ROUND).
// NW waves share the work (1: no barrier is passed; else all of the work-group call it together,
// red holding 3 NW + 3 words of LDS).
template <int NW, typename Keys>
__device__ __forceinline__ void keep_pages(const SelectParams &p, const Seen &s, Keys keys, int span, size_t pair, const int32_t *bt,
                                           int lane, int w, int *red) {
    // limit: keys above it are kept, and `ties` of those equal to it
    uint32_t limit = 1;
    int ties = 0x7fffffff, parity = 0;
    auto total = [&](int v) {   // the sum over the waves, alternating between two cells
        if constexpr (NW == 1) return v;
        parity ^= 1;
        if (lane == 0) red[parity * NW + w] = v;
        __syncthreads();
        int sum = 0;
#pragma unroll
        for (int i = 0; i < NW; i++) sum += red[parity * NW + i];
        return sum;
    };
    const int stride = NW * ROUND;
    if (s.need < s.c1 - s.c0 && s.need > 0) {
        uint32_t top = 0, low = 0xffffffffu;
        for (int i = w * ROUND + 4 * lane; i < span; i += stride) {
            const u32x4 k = *reinterpret_cast<const u32x4 *>(keys + i);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                top = max(top, k[e]);
                low = min(low, k[e] - 1);   // 0 wraps to the largest: not up for choice
            }
        }
        top = wave_umax(top);
        low = ~wave_umax(~low);
        if constexpr (NW > 1) {
            uint32_t *r = reinterpret_cast<uint32_t *>(red);
            if (lane == 0) r[w] = top, r[2 * NW + w] = low;   // cells that total() writes after a barrier
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NW; i++) top = max(top, r[i]), low = min(low, r[2 * NW + i]);
        }
        low++;
        int above = 0;   // keys > top: fewer than need; keys >= low: at least need
        bool exact = false;
        while (low < top && !exact) {
            const uint32_t d = top - low, mid = low + d / 2 + (d & 1);
            int c = 0;
            for (int i = w * ROUND + 4 * lane; i < span; i += stride) {
                const u32x4 k = *reinterpret_cast<const u32x4 *>(keys + i);
#pragma unroll
                for (int e = 0; e < 4; e++) c += __popcll(__ballot(k[e] >= mid));
            }
            c = total(c);
            if (c >= s.need) {
                low = mid;
                exact = c == s.need;
            } else {
                top = mid - 1;
                above = c;
            }
        }
        limit = low;
        ties = exact ? 0x7fffffff : s.need - above;
    } else if (s.need <= 0) {
        limit = 0xffffffffu;   // none by score
        ties = 0;
    }
    // pages in order: wave w takes [i0, i1)
    const int seen64 = (s.seen + 63) & ~63, part = NW == 1 ? seen64 : ((seen64 / 64 + NW - 1) / NW) * 64;
    const int i0 = min(w * part, seen64), i1 = min(i0 + part, seen64);
    int base = 0, eq = 0;
    auto page = [&](int i, bool &sure, bool &even) {
        const uint32_t k = keys[i];
        const bool cand = i >= s.c0 && i < s.c1;
        sure = i < s.seen && (!cand || k > limit);
        even = cand && k == limit;
    };
    if constexpr (NW > 1) {
        int ns = 0, ne = 0;
        for (int i = i0; i < i1; i += 64) {
            bool sure, even;
            page(i + lane, sure, even);
            ns += __popcll(__ballot(sure));
            ne += __popcll(__ballot(even));
        }
        __syncthreads();
        if (lane == 0) red[w] = ns, red[NW + w] = ne;
        __syncthreads();
        for (int i = 0; i < w; i++) base += red[i], eq += red[NW + i];
    }
    int32_t *out = p.tables + pair * p.keep;
    const unsigned long long below = (1ull << lane) - 1;
    for (int i = i0; i < i1; i += 64) {
        bool sure, even;
        page(i + lane, sure, even);
        const unsigned long long ms = __ballot(sure), me = __ballot(even);
        // pages written before this one: the sure ones, and the equal ones while there was room
        const int q = eq + __popcll(me & below), at = base + __popcll(ms & below) + min(q, ties);
        if ((sure || (even && q < ties)) && at < s.kept) out[at] = bt[i + lane];
        base += __popcll(ms);
        eq += __popcll(me);
    }
    for (int i = s.kept + w * 64 + lane; i < p.keep; i += NW * 64) out[i] = 0;
    if (w == 0 && lane == 0) {
        const long long l = (long long)(s.kept - 1) * p.P + min(s.last + 1 - (s.seen - 1) * p.P, p.P);
        p.lengths[pair] = (int)l;
    }
}

// Grid (Hk, token tiles, B), the keys of the tile's tokens in LDS.
template <int D, int GP, int RT, bool WIDE>
__global__ void __launch_bounds__(THREADS) select_kernel(SelectParams p) {
    using TL = Tile<GP, RT, WIDE>;
    __shared__ __attribute__((aligned(16))) int8_t w[TL::ROWS][2 * D];
    __shared__ float forth[TL::ROWS];
    __shared__ int red[3 * WAVES + 3];
    extern __shared__ __attribute__((aligned(16))) uint32_t keys[];   // [TT][pitch]
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x, b = blockIdx.z;
    const Step st = step_of(p.qsl, p.positions, b, p.nmax, p.total);
    for (int t0 = blockIdx.y * TL::TT; t0 < st.n; t0 += gridDim.y * TL::TT) {
        __syncthreads();   // the tile before this one is done with LDS
        const int tokens = min(TL::TT, st.n - t0);
        const int most = Seen(p, st, t0 + tokens - 1).seen, ntiles = (most + 15) >> 4;
        const int span = (most + ROUND - 1) / ROUND * ROUND;
        quantize_rows<D, GP, RT, WIDE>(p, st, h, t0, tid, w, forth);
        for (int i = ntiles * 16 + tid; i < span; i += THREADS)
            for (int t = 0; t < tokens; t++) keys[t * p.pitch + i] = 0;
        __syncthreads();
        score_pages<D, GP, RT, WIDE>(p, st, b, h, t0, lane, wv, WAVES, ntiles, most, w, forth,
                                     [&](int t, int page) { return keys + t * p.pitch + page; });
        __syncthreads();
        const int32_t *bt = p.bt + (size_t)b * p.bt_stride;
        if constexpr (TL::TT == 1) {
            keep_pages<WAVES>(p, Seen(p, st, t0), (const uint32_t *)keys, span, (size_t)(st.tok0 + t0) * p.Hk + h, bt, lane, wv, red);
        } else {
            for (int t = wv; t < tokens; t += WAVES)
                keep_pages<1>(p, Seen(p, st, t0 + t), (const uint32_t *)keys + t * p.pitch, span,
                              (size_t)(st.tok0 + t0 + t) * p.Hk + h, bt, lane, 0, red);
        }
    }
}

// The keys of a token tile to the workspace: grid (Hk x split, token tiles, B).
template <int D, int GP, int RT, bool WIDE>
__global__ void __launch_bounds__(THREADS) scores_kernel(SelectParams p) {
    using TL = Tile<GP, RT, WIDE>;
    __shared__ __attribute__((aligned(16))) int8_t w[TL::ROWS][2 * D];
    __shared__ float forth[TL::ROWS];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x % p.Hk, part = blockIdx.x / p.Hk, b = blockIdx.z;
    const Step st = step_of(p.qsl, p.positions, b, p.nmax, p.total);
    for (int t0 = blockIdx.y * TL::TT; t0 < st.n; t0 += gridDim.y * TL::TT) {
        __syncthreads();
        const int tokens = min(TL::TT, st.n - t0);
        const int most = Seen(p, st, t0 + tokens - 1).seen, ntiles = (most + 15) >> 4;
        const int span = (most + ROUND - 1) / ROUND * ROUND;
        quantize_rows<D, GP, RT, WIDE>(p, st, h, t0, tid, w, forth);
        auto at = [&](int t, int page) { return p.keys + ((size_t)(st.tok0 + t0 + t) * p.Hk + h) * p.pitch + page; };
        if (part == 0)
            for (int i = ntiles * 16 + tid; i < span; i += THREADS)
                for (int t = 0; t < tokens; t++) *at(t, i) = 0;
        __syncthreads();
        score_pages<D, GP, RT, WIDE>(p, st, b, h, t0, lane, part * WAVES + wv, p.split * WAVES, ntiles, most, w, forth, at);
    }
}

// Kept pages of one token and KV head from the workspace: grid (Hk, tokens, B). `tt` is the scores'
// token tile: rows of keys are padded to the last visible page of their tile.
__global__ void __launch_bounds__(THREADS) keep_kernel(SelectParams p, int tt) {
    __shared__ int red[3 * WAVES + 3];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x, b = blockIdx.z;
    const Step st = step_of(p.qsl, p.positions, b, p.nmax, p.total);
    for (int t = blockIdx.y; t < st.n; t += gridDim.y) {
        const int most = Seen(p, st, min(t / tt * tt + tt, st.n) - 1).seen, span = (most + ROUND - 1) / ROUND * ROUND;
        const size_t pair = (size_t)(st.tok0 + t) * p.Hk + h;
        __syncthreads();   // the token before this one is done with red
        keep_pages<WAVES>(p, Seen(p, st, t), (const uint32_t *)p.keys + pair * p.pitch, span, pair, p.bt + (size_t)b * p.bt_stride,
                          lane, wv, red);
    }
}

// LDS that select_kernel's keys may take: one work-group of 16 waves and its operands on a CU.
constexpr int LDS_KEYS = 136 << 10;

template <int D, int GP, int RT, bool WIDE>
int launch(SelectParams p, int num_seqs, hipStream_t s) {
    constexpr int TT = Tile<GP, RT, WIDE>::TT;
    const long long tiles = (p.nmax + (long long)TT - 1) / TT, groups = tiles * num_seqs * p.Hk;
    const unsigned y = (unsigned)min(tiles, 32768LL);   // longer steps loop
    const size_t bytes = (size_t)TT * p.pitch * sizeof(uint32_t);
    // One launch while the keys fit LDS and either the launch's work-groups fill half of the chip or a
    // table is short; a wide table's pages are shared out over work-groups otherwise.
    if (bytes <= (size_t)LDS_KEYS && (groups >= 128 || p.bt_stride <= 2048)) {
        auto kernel = select_kernel<D, GP, RT, WIDE>;
        if (bytes > (48u << 10) &&
            hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != hipSuccess)
            return TI_ERR_LAUNCH;
        kernel<<<dim3(p.Hk, y, num_seqs), THREADS, bytes, s>>>(p);
        return hipGetLastError() == hipSuccess ? TI_OK : TI_ERR_LAUNCH;
    }
    p.split = 1;
    while (groups * p.split < 256 && p.split * WAVES * 32 < p.bt_stride) p.split <<= 1;
    scores_kernel<D, GP, RT, WIDE><<<dim3(p.Hk * p.split, y, num_seqs), THREADS, 0, s>>>(p);
    if (hipGetLastError() != hipSuccess) return TI_ERR_LAUNCH;
    keep_kernel<<<dim3(p.Hk, min(p.nmax, 32768), num_seqs), THREADS, 0, s>>>(p, TT);
    return hipGetLastError() == hipSuccess ? TI_OK : TI_ERR_LAUNCH;
}

// Query rows per tile: 64 where the steps' tokens fill them and the launch still has work-groups for
// every CU (bounds are then read once for four blocks of rows), else 16.
template <int D, int GP>
int launch_rows(const SelectParams &p, int num_seqs, hipStream_t s) {
    constexpr int TT = Tile<GP, 4, false>::TT;
    const long long groups = ((long long)p.nmax + TT - 1) / TT * num_seqs * p.Hk;
    if (groups >= 256 && p.nmax >= TT && (size_t)TT * p.pitch * 4 <= (size_t)LDS_KEYS) return launch<D, GP, 4, false>(p, num_seqs, s);
    return launch<D, GP, 1, false>(p, num_seqs, s);
}

template <int D>
int launch_heads(const SelectParams &p, int num_seqs, hipStream_t s) {
    if (p.G > 16) return launch<D, 16, 4, true>(p, num_seqs, s);
    if (p.G > 8) return launch_rows<D, 16>(p, num_seqs, s);
    if (p.G > 4) return launch_rows<D, 8>(p, num_seqs, s);
    if (p.G > 2) return launch_rows<D, 4>(p, num_seqs, s);
    if (p.G > 1) return launch_rows<D, 2>(p, num_seqs, s);
    return launch_rows<D, 1>(p, num_seqs, s);
}

int key_pitch(const ti_select_args *a) { return (int)(((long long)a->block_table_stride + ROUND - 1) / ROUND * ROUND); }

}  // namespace

size_t ti_select_bytes(const ti_select_args *a) {
    return (size_t)a->total_tokens * a->kv_heads * key_pitch(a) * sizeof(uint32_t);
}

int ti_launch_select_pages(const ti_select_args *a, hipStream_t s) {
    SelectParams p{};
    p.q = a->q;
    p.bounds = a->bounds.bounds;
    p.scale = a->bounds.scale;
    p.positions = a->positions;
    p.qsl = a->query_start_loc;
    p.bt = a->block_tables;
    p.tables = a->tables;
    p.lengths = a->lengths;
    p.keys = (uint32_t *)a->workspace;
    p.bt_stride = a->block_table_stride;
    p.num_pages = a->num_pages;
    p.P = a->page_size;
    p.Hk = a->kv_heads;
    p.Hq = a->q_heads;
    p.G = a->q_heads / a->kv_heads;
    p.nmax = a->max_query_len;
    p.total = a->total_tokens;
    p.keep = a->keep;
    p.sinks = a->sinks;
    p.window = a->window;
    p.causal = a->causal;
    p.pitch = key_pitch(a);
    p.split = 1;
    p.f32 = a->dtype == TI_F32;
    return a->head_dim == 128 ? launch_heads<128>(p, a->num_seqs, s) : launch_heads<64>(p, a->num_seqs, s);
}
