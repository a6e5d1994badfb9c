// The pages that a query keeps by the bounds of their keys (page_bounds.hip).
//
// A query row q (one token, one query head; times its dimensions' channels) becomes whole numbers
// w_d = rint(q_d 2^-e), e the least exponent with |q| <= 127 2^e; the row 2^e w so rounded has with any key
// inside a page's bounds at most the product
//   2^e 2^e_page sum_d (w_d hi_d where w_d > 0, else w_d lo_d) = 2^e 2^e_page (relu(w) . hi + min(w, 0) . lo):
// one int8 matrix product of depth 2 D, whose sums stay below 2^22 and are exact. The score of a page
// for a token and KV head is the largest over the G query heads, two multiplications by powers of
// two: exact, so equal scores are equal bounds and not roundings, and the kept pages do not depend
// on how the work is split.
//
// Scores become 32-bit keys in the scores' order, 0 for pages that are not up for choice (those kept
// anyway, and those past the last visible one). The key of the last page kept by score is found by counting keys
// in parts of their range: in two by one wave where a work-group has a token for each, in as many parts as
// it has threads where it has one token. Then one pass over the pages in order writes the kept ones.
//
// Two forms. select_kernel holds a token tile's keys in LDS and does both steps in one launch.
// scores_kernel and keep_kernel share a tile's pages out over several work-groups, the keys going
// through the workspace, for few tokens over wide tables and for tables that LDS does not hold.
#include <algorithm>

#include "page_bounds.hpp"

using namespace ti;
using namespace ti_pages;

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int ROUND = 256;   // keys read by a wave at once: rows of keys are padded to it with zeros
constexpr int ONE = 8 * ROUND;   // the most keys that one wave searches (they stay in registers)

struct SelectParams {
    const void *q;
    const int8_t *bounds;
    const float *scale, *channel;
    const int32_t *positions, *qsl, *bt;
    int32_t *tables, *lengths;
    uint32_t *keys;   // two launches: [rows][Hk][pitch] (Part)
    int bt_stride, num_pages, P, Hk, Hq, G, nmax, total, keep, sinks, window, causal, f32, pshift;
    int pitch, split;   // keys per (token, KV head); work-groups that share a token tile's pages
    int first, end;     // two launches: the packed tokens that they work on; end 0: all, a sequence's from row b nmax on
};

// Two launches: the tokens begin .. end - 1 of a sequence that they work on, and the workspace's row of its token 0.
struct Part {
    int begin, end, row;
    __device__ Part(const SelectParams &p, const Step &st, int b) {
        begin = p.end ? max(p.first - st.tok0, 0) : 0;
        end = p.end ? min(st.n, p.end - st.tok0) : st.n;
        row = p.end ? st.tok0 - p.first : b * p.nmax;
    }
};

// What one token sees: pages [0, seen), of which [c0, c1) are up for choice and `need` kept by score.
struct Seen {
    int last, seen, c0, c1, kept, need;
    __device__ Seen(const SelectParams &p, const Step &st, int t) {
        last = st.start + (p.causal ? t : st.n - 1);
        seen = min((p.pshift >= 0 ? last >> p.pshift : last / p.P) + 1, p.bt_stride);
        c0 = min(p.sinks, seen);
        c1 = max(c0, seen - p.window);
        kept = min(seen, p.keep);
        need = kept - (seen - (c1 - c0));
    }
};

// Larger score, larger key, never 0; NaN (an infinite page scale times 0) counts as infinite.
__device__ __forceinline__ uint32_t order_key(float x) {
    x = x != x ? INFINITY : x + 0.0f;   // -0 and 0 are one score
    const int32_t u = (int32_t)__float_as_uint(x);
    return (uint32_t)(u ^ (u >> 31 | (int32_t)0x80000000));
}

template <int CTRL> __device__ __forceinline__ int dpp(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, false); }
// Sum of a wave's values, wave-uniform: within rows of 16 lanes by mirrored halves, across them by lane reads.
__device__ __forceinline__ int wave_total(int x) {
    x += dpp<0xb1>(x);    // quad_perm 1 0 3 2
    x += dpp<0x4e>(x);    // quad_perm 2 3 0 1
    x += dpp<0x141>(x);   // row_half_mirror
    x += dpp<0x140>(x);   // row_mirror
    return (__builtin_amdgcn_readlane(x, 0) + __builtin_amdgcn_readlane(x, 16)) +
           (__builtin_amdgcn_readlane(x, 32) + __builtin_amdgcn_readlane(x, 48));
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t x) {
    x = max(x, (uint32_t)dpp<0xb1>((int)x));
    x = max(x, (uint32_t)dpp<0x4e>((int)x));
    x = max(x, (uint32_t)dpp<0x141>((int)x));
    x = max(x, (uint32_t)dpp<0x140>((int)x));
    return max(max((uint32_t)__builtin_amdgcn_readlane((int)x, 0), (uint32_t)__builtin_amdgcn_readlane((int)x, 16)),
               max((uint32_t)__builtin_amdgcn_readlane((int)x, 32), (uint32_t)__builtin_amdgcn_readlane((int)x, 48)));
}

// A tile of RT x 16 query rows: rows of a token are its G heads, padded to GP (a power of two up to 16);
// WIDE (G > 16): one token's heads over all RT blocks. TT tokens a tile.
template <int GP, int RT, bool WIDE> struct Tile {
    static constexpr int ROWS = RT * 16, TT = WIDE ? 1 : ROWS / GP;
};

// The whole-number operands of a tile's rows in LDS: relu(w) then min(w, 0), and 2^e (a row that is not
// finite: zeros; a row that pads the heads: NaN, which no maximum takes). 16 lanes per row.
template <int D, int GP, int RT, bool WIDE, int W>
__device__ __forceinline__ void quantize_rows(const SelectParams &p, const Step &st, int h, int t0, int tid, int8_t (*w)[2 * D],
                                              float *forth) {
    constexpr int E = D / 16;
    for (int r = tid / 16; r < RT * 16; r += W * 4) {
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
        if (p.channel) {
#pragma unroll
            for (int i = 0; i < E; i++) x[i] *= p.channel[h * D + c + i];
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
        if ((tid & 15) == 0) forth[r] = g < p.G ? power(e) : NAN;
    }
}

// The keys of a tile's tokens for the 16-page tiles j = first, first + step, ... < ntiles, by one wave:
// S = W bounds on v_mfma_i32_16x16x64_i8 (A: lane l holds row l % 16's bytes 16 (l / 16) .. + 16 of each
// 64; B: a page's, the same way), so lane l gets the products of page l % 16 with rows 4 (l / 16) .. + 3:
// the heads of a token are a lane's registers (and those of other 16-lane groups for GP > 4), its page's
// scale is at hand, and few vector instructions are left beside the loads: with the operands the other
// way round (heads in lanes) they bound the kernel (512 tokens on 64k: 17 us of scores, 2048 pages
// 11.6). dst(t, page) is where the key of token t0 + t goes, from <= t < tokens.
template <int D, int GP, int RT, bool WIDE, typename Dst>
__device__ __forceinline__ void score_pages(const SelectParams &p, int b, int h, int from, int tokens, int lane, int first, int step, int ntiles,
                                            int most, const int8_t (*w)[2 * D], const float *forth, Dst dst) {
    constexpr int NK = 2 * D / 64;
    constexpr int HL = GP < 4 ? GP : 4, TL = 4 / HL;   // heads and tokens of a lane's four rows
    const int r16 = lane & 15, kg = lane >> 4;
    const int32_t *bt = p.bt + (size_t)b * p.bt_stride;
    i32x4 q[RT][NK];
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int i = 0; i < NK; i++) q[rt][i] = *reinterpret_cast<const i32x4 *>(&w[rt * 16 + r16][i * 64 + kg * 16]);
    struct Page {
        i32x4 b[NK];
        float scale;
    };
    // a tile's page ids are loaded a tile ahead of its bounds, so that one wait does not follow another
    auto ids = [&](int j) { return bt[min(j * 16 + r16, most - 1)]; };
    auto load = [&](int raw, Page &pg) {
        const int id = clamp_page(raw, p.num_pages);
        const size_t at = (size_t)id * p.Hk + h;
        const int8_t *src = p.bounds + at * 2 * D + kg * 16;
#pragma unroll
        for (int i = 0; i < NK; i++) pg.b[i] = *reinterpret_cast<const i32x4 *>(src + i * 64);
        pg.scale = p.scale[at];
    };
    auto use = [&](int j, const Page &pg) {
        float s[TL];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            i32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < NK; i++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(q[rt][i], pg.b[i], acc, 0, 0, 0);
            const f32x4 f = *reinterpret_cast<const f32x4 *>(&forth[rt * 16 + 4 * kg]);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float x = (float)acc[k] * f[k];
                s[k / HL] = k % HL || (WIDE && rt) ? fmaxf(s[k / HL], x) : x;
            }
            if (WIDE && rt < RT - 1) continue;
            if (GP >= 8) s[0] = fmaxf(s[0], __shfl_xor(s[0], 16));
            if (GP >= 16) s[0] = fmaxf(s[0], __shfl_xor(s[0], 32));
#pragma unroll
            for (int n = 0; n < TL; n++) {
                const int t = WIDE ? 0 : (rt * 16 + 4 * kg + n * HL) / GP;
                if (4 * kg % GP == 0 && t >= from && t < tokens) *dst(t, j * 16 + r16) = order_key(s[n] * pg.scale);
            }
        }
    };
    int j = first;
    if (j >= ntiles) return;
    int ia = ids(j), ib = ids(j + step);
    if constexpr (RT > 1) {   // its operands leave no registers for a second set of bounds
        Page pg;
        for (; j < ntiles; j += step) {
            load(ia, pg);
            ia = ib;
            ib = ids(j + 2 * step);
            use(j, pg);
        }
    } else {
        // two sets in turn: the next tile's loads are issued before this one is worked on
        Page pa, pb;
        load(ia, pa);
        ia = ids(j + 2 * step);
        while (true) {
            if (j + step < ntiles) load(ib, pb);
            ib = ids(j + 3 * step);
            use(j, pa);
            j += step;
            if (j >= ntiles) break;
            if (j + step < ntiles) load(ia, pa);
            ia = ids(j + 3 * step);
            use(j, pb);
            j += step;
            if (j >= ntiles) break;
        }
    }
}

// The last page kept by score: keys above `limit` are kept, and `ties` of those equal to it.
struct Limit {
    uint32_t limit;
    int ties;
};
// The search by one wave that holds all keys, between the smallest and the largest: a step takes 0.2 us for 512
// keys and 0.4 for 2048, so the next one is where the count would be right if the keys lay evenly (512 tokens on
// 64k keys 31.0 us by halves only, 29.3 so). Where few keys are left between the ends, these close in on them:
// equal keys end the search then and not after all 24 halvings of their digits.
template <int NG> __device__ __forceinline__ Limit narrow(const Seen &s, const uint32_t *keys, int span, int lane) {
    u32x4 k[NG];
    uint32_t top = 0, low = 0xffffffffu;
#pragma unroll
    for (int n = 0; n < NG; n++) {
        k[n] = n * ROUND < span ? *reinterpret_cast<const u32x4 *>(keys + n * ROUND + 4 * lane) : (u32x4){0u, 0u, 0u, 0u};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            top = max(top, k[n][e]);
            low = min(low, k[n][e] - 1);   // 0 wraps to the largest
        }
    }
    top = wave_umax(top);
    low = ~wave_umax(~low) + 1;
    int from = s.c1 - s.c0, above = 0;   // keys >= low: at least need; keys > top: fewer
    bool closed = false;
    int step = 1;
    while (low < top) {
        if (!closed && from - above <= 4) {
            closed = true;
            uint32_t most = 0, least = 0xffffffffu;
#pragma unroll
            for (int n = 0; n < NG; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    most = max(most, k[n][e] <= top ? k[n][e] : 0u);
                    least = min(least, k[n][e] >= low ? k[n][e] : 0xffffffffu);
                }
            top = wave_umax(most);
            low = ~wave_umax(~least);
            continue;
        }
        // where the count would be right if the keys lay evenly; every fourth step halves
        const uint32_t d = top - low;
        const float part = step++ & 3 ? (float)(from - s.need) * __builtin_amdgcn_rcpf((float)(from - above)) : 0.5f;
        const uint32_t mid = low + min(max((uint32_t)((float)d * part), 1u), d);
        int c = 0;
#pragma unroll
        for (int n = 0; n < NG; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) c += k[n][e] >= mid;
        c = wave_total(c);
        if (c == s.need) return {mid - 1, 0};
        if (c > s.need) {
            low = mid;
            from = c;
        } else {
            top = mid - 1;
            above = c;
        }
    }
    return {low, s.need - above};
}

// Keys that are not up for choice become 0; *found: there is nothing to search.
__device__ __forceinline__ Limit begin_search(const Seen &s, uint32_t *keys, int span, int tid, int threads, bool *found) {
    for (int i = tid; i < s.c0; i += threads) keys[i] = 0;
    for (int i = s.c1 + tid; i < span; i += threads) keys[i] = 0;
    *found = s.need >= s.c1 - s.c0 || s.need <= 0;
    return Limit{s.need <= 0 ? 0xffffffffu : 0u, 0};   // none, or every candidate
}

// By one wave, up to ONE keys.
__device__ __forceinline__ Limit find_limit(const Seen &s, uint32_t *keys, int span, int lane) {
    bool found;
    const Limit l = begin_search(s, keys, span, lane, 64, &found);
    if (found) return l;
    if (span <= 2 * ROUND) return narrow<2>(s, keys, span, lane);
    if (span <= 5 * ROUND) return narrow<5>(s, keys, span, lane);
    return narrow<8>(s, keys, span, lane);
}

// The words of LDS that the waves of a work-group search with.
template <int W> struct SearchLds {
    int hist[W * 64];   // keys in each part of the range; then the keys of one part
    int sum[2 * W];
    int part, above, held, listed;
};

// By the W waves of a work-group, any number of keys: they are counted in as many equal parts of their range as
// there are threads, and the part that holds the last one kept is searched on: with up to 64 keys (the usual
// case, after one round) each lane ranks one of them, else as the range was. The waves' barriers and not the
// keys are the cost: 8192 keys take what 512 do.
template <int W>
__device__ __forceinline__ Limit find_limit_together(const Seen &s, uint32_t *keys, int span, int lane, int w, SearchLds<W> &m) {
    constexpr int BINS = W * 64, BITS = __builtin_ctz(BINS);
    const int tid = w * 64 + lane;
    bool found;
    const Limit l = begin_search(s, keys, span, tid, BINS, &found);
    m.hist[tid] = 0;
    if (tid == 0) m.listed = 0;
    __syncthreads();   // (keys may be in global memory)
    if (found) return l;
    uint32_t top = 0, low = 0xffffffffu;
    for (int i = 4 * tid; i < span; i += 4 * BINS) {
        const u32x4 k = *reinterpret_cast<const u32x4 *>(keys + i);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            top = max(top, k[e]);
            low = min(low, k[e] - 1);   // 0 wraps to the largest
        }
    }
    top = wave_umax(top);
    low = wave_umax(~low);
    if (lane == 0) m.sum[w] = (int)top, m.sum[W + w] = (int)low;
    __syncthreads();
    top = wave_umax(lane < W ? (uint32_t)m.sum[lane] : 0u);
    low = ~wave_umax(lane < W ? (uint32_t)m.sum[W + lane] : 0u) + 1;
    int need = s.need;   // of the keys in [low, top]; larger ones are all kept
    while (low < top) {
        const int shift = max(32 - __builtin_clz(top - low) - BITS, 0);
        for (int i = 4 * tid; i < span; i += 4 * BINS) {
            const u32x4 k = *reinterpret_cast<const u32x4 *>(keys + i);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (k[e] >= low && k[e] <= top) atomicAdd(&m.hist[(k[e] - low) >> shift], 1);
        }
        __syncthreads();
        const int part = BINS - 1 - tid, c = m.hist[part];
        m.hist[part] = 0;
        int upto = c;   // keys of this part and the ones above it
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 63) m.sum[w] = upto;
        __syncthreads();
        upto += wave_total(lane < w ? m.sum[lane] : 0);
        if (upto >= need && upto - c < need) {
            m.part = part;
            m.above = upto - c;
            m.held = c;
        }
        __syncthreads();
        need -= m.above;
        low += (uint32_t)m.part << shift;
        top = low + min(top - low, (1u << shift) - 1);
        if (need == m.held) return {low - 1, 0};
        if (m.held > 64) continue;
        const int held = m.held;
        for (int i = 4 * tid; i < span; i += 4 * BINS) {
            const u32x4 k = *reinterpret_cast<const u32x4 *>(keys + i);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (k[e] >= low && k[e] <= top) m.hist[atomicAdd(&m.listed, 1)] = (int)k[e];
        }
        __syncthreads();
        const uint32_t mine = lane < held ? (uint32_t)m.hist[lane] : 0u;
        int more = 0, same = 0;
        for (int j = 0; j < held; j++) {
            const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)mine, j);
            more += other > mine;
            same += other == mine;
        }
        const unsigned long long last = __ballot(lane < held && more < need && more + same >= need);
        const int at = __builtin_ctzll(last);
        return {(uint32_t)__builtin_amdgcn_readlane((int)mine, at), need - __builtin_amdgcn_readlane(more, at)};
    }
    return {low, need};
}

// Writes a token's number of keys.
__device__ __forceinline__ void write_length(const SelectParams &p, const Seen &s, size_t pair) {
    const long long n = (long long)(s.kept - 1) * p.P + min(s.last + 1 - (s.seen - 1) * p.P, p.P);
    p.lengths[pair] = (int)n;
}

// Writes one token's kept pages in order, zeros behind them, and its number of keys, by one wave. The kept
// pages' places take the place of keys that have been read, so that one load of up to 64 ids is waited for and not
// one for each 64 pages.
__device__ __forceinline__ void write_pages(const SelectParams &p, const Seen &s, const Limit &l, uint32_t *keys, size_t pair,
                                            const int32_t *bt, int lane) {
    const unsigned long long below = (1ull << lane) - 1;
    int base = 0, eq = 0;
    uint32_t next = keys[lane];
    for (int i0 = 0; i0 < s.seen; i0 += 64) {
        const uint32_t k = next;
        const int i = i0 + lane;
        next = keys[min(i + 64, s.seen - 1)];
        const bool cand = i >= s.c0 && i < s.c1;
        const bool sure = i < s.seen && (!cand || k > l.limit), even = cand && k == l.limit;
        const unsigned long long ms = __ballot(sure), me = __ballot(even);
        // pages kept before this one: the sure ones, and the equal ones while there was room
        const int q = eq + __popcll(me & below), at = base + __popcll(ms & below) + min(q, l.ties);
        if ((sure || (even && q < l.ties)) && at < s.kept) keys[at] = i;
        base += __popcll(ms);
        eq += __popcll(me);
    }
    int32_t *out = p.tables + pair * p.keep;
    for (int i = lane; i < p.keep; i += 64) out[i] = i < s.kept ? bt[keys[i]] : 0;
    if (lane == 0) write_length(p, s, pair);
}

// The same by the NW waves of a work-group, which share the pages; red: 2 NW words of LDS.
template <int NW>
__device__ __forceinline__ void write_pages_together(const SelectParams &p, const Seen &s, const Limit &l, const uint32_t *keys, size_t pair,
                                                     const int32_t *bt, int lane, int w, int *red) {
    const int steps = (s.seen + 63) >> 6, part = (steps + NW - 1) / NW;
    const int i0 = min(w * part, steps) * 64, i1 = min((w + 1) * part, steps) * 64;
    auto page = [&](int i, bool &sure, bool &even) {
        const uint32_t k = keys[i];
        const bool cand = i >= s.c0 && i < s.c1;
        sure = i < s.seen && (!cand || k > l.limit);
        even = cand && k == l.limit;
    };
    int ns = 0, ne = 0;
    for (int i = i0; i < i1; i += 64) {
        bool sure, even;
        page(i + lane, sure, even);
        ns += __popcll(__ballot(sure));
        ne += __popcll(__ballot(even));
    }
    if (lane == 0) red[w] = ns, red[NW + w] = ne;
    __syncthreads();
    int base = wave_total(lane < w ? red[lane] : 0), eq = wave_total(lane < w ? red[NW + lane] : 0);
    int32_t *out = p.tables + pair * p.keep;
    const unsigned long long below = (1ull << lane) - 1;
    int next = bt[min(i0 + lane, s.seen - 1)];
    for (int i = i0; i < i1; i += 64) {
        const int id = next;
        next = bt[min(i + 64 + lane, s.seen - 1)];
        bool sure, even;
        page(i + lane, sure, even);
        const unsigned long long ms = __ballot(sure), me = __ballot(even);
        // pages written before this one: the sure ones, and the equal ones while there was room
        const int q = eq + __popcll(me & below), at = base + __popcll(ms & below) + min(q, l.ties);
        if ((sure || (even && q < l.ties)) && at < s.kept) out[at] = id;
        base += __popcll(ms);
        eq += __popcll(me);
    }
    for (int i = s.kept + w * 64 + lane; i < p.keep; i += NW * 64) out[i] = 0;
    if (w == 0 && lane == 0) write_length(p, s, pair);
}

// The search as a call, for tiles of several blocks of rows, where it is the exception: in line it would take
// registers from the scores' loop, which spills then (512 tokens on 64k keys 31.3 us, in line 32.9).
template <int W>
__device__ __attribute__((noinline)) Limit find_limit_apart(const Seen &s, uint32_t *keys, int span, int lane, int w, SearchLds<W> &m) {
    return find_limit_together<W>(s, keys, span, lane, w, m);
}

// One token's pages by the whole work-group of W waves.
template <int W, bool APART>
__device__ __forceinline__ void keep_together(const SelectParams &p, const Seen &s, uint32_t *keys, int span, size_t pair,
                                              const int32_t *bt, int lane, int w, SearchLds<W> &m) {
    Limit l;
    if constexpr (APART) l = find_limit_apart<W>(s, keys, span, lane, w, m);
    else l = find_limit_together<W>(s, keys, span, lane, w, m);
    __syncthreads();   // m is read
    write_pages_together<W>(p, s, l, keys, pair, bt, lane, w, m.sum);
}

// Grid (Hk, token tiles, B), the keys of the tile's tokens in LDS.
template <int D, int GP, int RT, bool WIDE, int W>
__global__ void __launch_bounds__(W * 64) select_kernel(SelectParams p) {
    using TL = Tile<GP, RT, WIDE>;
    __shared__ __attribute__((aligned(16))) int8_t w[TL::ROWS][2 * D];
    __shared__ float forth[TL::ROWS];
    __shared__ SearchLds<W> search;
    extern __shared__ __attribute__((aligned(16))) uint32_t keys[];   // [TT][pitch]
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x, b = blockIdx.z;
    const Step st = step_of(p.qsl, p.positions, b, p.nmax, p.total);
    for (int t0 = blockIdx.y * TL::TT; t0 < st.n; t0 += gridDim.y * TL::TT) {
        __syncthreads();   // the tile before this one is done with LDS
        const int tokens = min(TL::TT, st.n - t0);
        const int most = Seen(p, st, t0 + tokens - 1).seen, ntiles = (most + 15) >> 4;
        const int span = (most + ROUND - 1) / ROUND * ROUND;
        quantize_rows<D, GP, RT, WIDE, W>(p, st, h, t0, tid, w, forth);
        __syncthreads();
        score_pages<D, GP, RT, WIDE>(p, b, h, 0, tokens, lane, wv, W, ntiles, most, w, forth,
                                     [&](int t, int page) { return keys + t * p.pitch + page; });
        __syncthreads();
        const int32_t *bt = p.bt + (size_t)b * p.bt_stride;
        if (tokens == 1 || span > ONE) {
            for (int t = 0; t < tokens; t++) {
                keep_together<W, (RT > 1 && !WIDE)>(p, Seen(p, st, t0 + t), keys + t * p.pitch, span, (size_t)(st.tok0 + t0 + t) * p.Hk + h, bt, lane,
                                               wv, search);
                __syncthreads();   // its LDS is read
            }
        } else {
            for (int t = wv; t < tokens; t += W) {
                const Seen s(p, st, t0 + t);
                const Limit l = find_limit(s, keys + t * p.pitch, span, lane);
                write_pages(p, s, l, keys + t * p.pitch, (size_t)(st.tok0 + t0 + t) * p.Hk + h, bt, lane);
            }
        }
    }
}

// The keys of a token tile to the workspace: grid (Hk x split, token tiles, B).
template <int D, int GP, int RT, bool WIDE, int W>
__global__ void __launch_bounds__(W * 64) scores_kernel(SelectParams p) {
    using TL = Tile<GP, RT, WIDE>;
    __shared__ __attribute__((aligned(16))) int8_t w[TL::ROWS][2 * D];
    __shared__ float forth[TL::ROWS];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x % p.Hk, part = blockIdx.x / p.Hk, b = blockIdx.z;
    const Step st = step_of(p.qsl, p.positions, b, p.nmax, p.total);
    const Part own(p, st, b);
    for (int t0 = own.begin / TL::TT * TL::TT + blockIdx.y * TL::TT; t0 < own.end; t0 += gridDim.y * TL::TT) {
        __syncthreads();
        const int tokens = min(TL::TT, own.end - t0);
        const int most = Seen(p, st, t0 + tokens - 1).seen, ntiles = (most + 15) >> 4;
        quantize_rows<D, GP, RT, WIDE, W>(p, st, h, t0, tid, w, forth);
        __syncthreads();
        score_pages<D, GP, RT, WIDE>(p, b, h, max(own.begin - t0, 0), tokens, lane, part * W + wv, p.split * W, ntiles, most, w, forth,
                                     [&](int t, int page) { return p.keys + ((size_t)(own.row + t0 + t) * p.Hk + h) * p.pitch + page; });
    }
}

// Kept pages of one token and KV head from the workspace: grid (Hk, tokens, B). The keys are read into LDS
// where it holds them (`lds` of them).
template <int W> __global__ void __launch_bounds__(W * 64) keep_kernel(SelectParams p, int lds) {
    __shared__ SearchLds<W> search;
    extern __shared__ __attribute__((aligned(16))) uint32_t held[];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x, b = blockIdx.z;
    const Step st = step_of(p.qsl, p.positions, b, p.nmax, p.total);
    const Part own(p, st, b);
    for (int t = own.begin + blockIdx.y; t < own.end; t += gridDim.y) {
        const Seen s(p, st, t);
        const int span = (s.seen + ROUND - 1) / ROUND * ROUND;
        const size_t pair = (size_t)(st.tok0 + t) * p.Hk + h;
        uint32_t *keys = p.keys + ((size_t)(own.row + t) * p.Hk + h) * p.pitch;
        __syncthreads();   // the token before this one is done with LDS
        const int32_t *bt = p.bt + (size_t)b * p.bt_stride;
        if (span <= lds) {
            for (int i = 4 * tid; i < span; i += W * 256)
                *reinterpret_cast<u32x4 *>(held + i) = *reinterpret_cast<const u32x4 *>(keys + i);
            __syncthreads();
            keep_together<W, false>(p, s, held, span, pair, bt, lane, wv, search);
        } else {
            keep_together<W, false>(p, s, keys, span, pair, bt, lane, wv, search);
        }
    }
}

// LDS that select_kernel's keys may take: one work-group of 16 waves and its operands on a CU.
constexpr int LDS_KEYS = 128 << 10;
bool allow_lds(const void *kernel, size_t bytes) {
    return bytes <= (32u << 10) || hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == hipSuccess;
}

// Keys of a tile, in LDS.
size_t key_bytes(const SelectParams &p, int tile) { return (size_t)min(tile, p.nmax) * p.pitch * sizeof(uint32_t); }

// One launch while the keys fit LDS and either there is a work-group for every CU or a table is short: one token
// over 512 pages takes 11.0 us so and 13.0 in two launches, over 1024 15.4 and 13.2, over 2048 23.7 and 13.8;
// 256 work-groups over 2048 pages each 39.7 and 45.4, 128 26.2 and 24.0.
template <int TT> bool fits_one_launch(const SelectParams &p, long long groups) {
    return key_bytes(p, TT) <= (size_t)LDS_KEYS && (groups >= 256 || p.bt_stride <= 768);
}

// Bytes of a token's keys in the workspace, and of the workspace. Where LDS holds the keys of a tile of TT tokens, two
// launches are taken for fewer than 256 work-groups only, for at most 255 / Hk tiles. Where it does not, longer steps
// are worked on in parts of PART_BYTES (with 4 tokens a tile at least 255 work-groups each up to 32768 table entries;
// beyond, a tile's pages are shared out over several).
constexpr size_t PART_BYTES = 128u << 20;
size_t row_bytes(int Hk, int pitch) { return (size_t)Hk * pitch * sizeof(uint32_t); }
size_t scratch_bytes(int total, int Hk, int pitch, int TT) {
    const size_t row = row_bytes(Hk, pitch);
    const size_t most = (size_t)TT * pitch * sizeof(uint32_t) <= LDS_KEYS ? 255u / Hk * TT * row : PART_BYTES;
    return std::min(total * row, std::max(row, most));
}

template <int D, int GP, int RT, bool WIDE, int W>
int launch_one(const SelectParams &p, unsigned y, int num_seqs, hipStream_t s) {
    const size_t bytes = key_bytes(p, Tile<GP, RT, WIDE>::TT);
    auto kernel = select_kernel<D, GP, RT, WIDE, W>;
    if (!allow_lds((const void *)kernel, bytes)) return TI_ERR_LAUNCH;
    kernel<<<dim3(p.Hk, y, num_seqs), W * 64, bytes, s>>>(p);
    return hipGetLastError() == hipSuccess ? TI_OK : TI_ERR_LAUNCH;
}

template <int D, int GP, int RT, bool WIDE>
int launch(SelectParams p, int num_seqs, hipStream_t s) {
    constexpr int TT = Tile<GP, RT, WIDE>::TT, W = 16;
    const long long tiles = (p.nmax + (long long)TT - 1) / TT, groups = tiles * num_seqs * p.Hk;
    const unsigned y = (unsigned)min(tiles, 32768LL);   // longer steps loop
    if (fits_one_launch<TT>(p, groups)) {
        // 4 waves for short tables, whose pages give 16 waves little to do, and for several work-groups per CU,
        // which wait for each other less (while LDS holds four): 128 pages and 64 work-groups 7.1 us and 7.8 with
        // 16, 512 and 512 19.2 and 25.2, 2048 and 512 68 and 76; 2048 and 128 27.7 and 25.9. Single tokens of 1 to 32
        // sequences (8 to 256 work-groups): 64 pages 5.5 and 6.2, 256 9.3-11.0 and 12.9-13.3, 512 11.7-13.4 and
        // 15.3-16.6; 768 14.2-17.0 and 17.4-20.0, where tiles of several tokens were not measured.
        if constexpr (RT == 1)
            if (key_bytes(p, TT) <= (32u << 10) && (p.bt_stride <= 512 || groups >= 512)) return launch_one<D, GP, RT, WIDE, 4>(p, y, num_seqs, s);
        return launch_one<D, GP, RT, WIDE, W>(p, y, num_seqs, s);
    }
    if constexpr (RT == 1 || WIDE) {   // launch_rows takes tiles of several tokens' blocks for one launch only
        const size_t held = std::min((size_t)p.pitch * sizeof(uint32_t), (size_t)LDS_KEYS);
        if (!allow_lds((const void *)keep_kernel<W>, held)) return TI_ERR_LAUNCH;
        // All tokens at once where the workspace has a row for each that the sequences can have (always, where LDS holds
        // a tile's keys), or for each row of the packed tokens, else as many rows at a time as it has. A part of a
        // sequence may begin inside a tile.
        const int rows = (int)(scratch_bytes(p.total, p.Hk, p.pitch, TT) / row_bytes(p.Hk, p.pitch));
        const bool whole = (long long)num_seqs * p.nmax <= rows;
        const long long most = std::min(tiles, ((long long)rows + TT - 1) / TT + 1);
        p.split = 1;
        while (std::min(groups, most * num_seqs * p.Hk) * p.split < 256 && p.split * W * 32 < p.bt_stride) p.split <<= 1;
        for (p.first = 0;; p.first = p.end) {
            p.end = whole ? 0 : p.total - p.first > rows ? p.first + rows : p.total;
            scores_kernel<D, GP, RT, WIDE, W><<<dim3(p.Hk * p.split, min(y, (unsigned)most), num_seqs), W * 64, 0, s>>>(p);
            if (hipGetLastError() != hipSuccess) return TI_ERR_LAUNCH;
            keep_kernel<W><<<dim3(p.Hk, min(min(p.nmax, rows), 32768), num_seqs), W * 64, held, s>>>(p, (int)(held / sizeof(uint32_t)));
            if (hipGetLastError() != hipSuccess) return TI_ERR_LAUNCH;
            if (whole || p.end == p.total) return TI_OK;
        }
    }
    return TI_ERR_LAUNCH;
}

// Query rows per tile: 64 (32 where a token's heads do not fill a lane's four rows or go past them: 64 spill
// there) where the steps' tokens fill them and the launch still has work-groups for every CU (bounds are then
// read once for several blocks of rows: 512 tokens on 64k keys 31 us, 91 with 16 rows), else 16 (128 tokens 25 and 30).
template <int D, int GP>
int launch_rows(const SelectParams &p, int num_seqs, hipStream_t s) {
    constexpr int RT = GP == 4 || GP == 16 ? 4 : 2, TT = Tile<GP, RT, false>::TT;
    const long long groups = ((long long)p.nmax + TT - 1) / TT * num_seqs * p.Hk;
    if (groups >= 256 && p.nmax >= TT && key_bytes(p, TT) <= (size_t)LDS_KEYS) return launch<D, GP, RT, false>(p, num_seqs, s);
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
    const int G = a->q_heads / a->kv_heads;
    const int TT = G > 8 ? 1 : G > 4 ? 2 : G > 2 ? 4 : G > 1 ? 8 : 16;   // a tile's tokens in two launches (launch_heads)
    return scratch_bytes(a->total_tokens, a->kv_heads, key_pitch(a), TT);
}

int ti_launch_select_pages(const ti_select_args *a, hipStream_t s) {
    SelectParams p{};
    p.q = a->q;
    p.bounds = a->bounds.bounds;
    p.scale = a->bounds.scale;
    p.channel = a->bounds.channel;
    p.positions = a->positions;
    p.qsl = a->query_start_loc;
    p.bt = a->block_tables;
    p.tables = a->tables;
    p.lengths = a->lengths;
    p.keys = (uint32_t *)a->workspace;
    p.bt_stride = a->block_table_stride;
    p.num_pages = a->num_pages;
    p.P = a->page_size;
    p.pshift = (p.P & (p.P - 1)) == 0 ? __builtin_ctz(p.P) : -1;
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
