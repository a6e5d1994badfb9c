// Neighbouring tokens of a step over the joined list of their chosen pages: for the sparse forms of the paged
// kernels (pa_decode.hpp, pa_generic.hip).
#pragma once

#include <type_traits>

#include "common.hpp"

namespace ti_group {
using namespace ti;

// Keys of a table that holds `most`: lengths below 0 are none. (Clamped before anything is taken off, which
// would wrap for lengths near -2^31.)
__device__ __forceinline__ int table_keys(int length, int most) { return min(max(length, 0), most); }

// The same over the pages of a group's tokens (GROUP, see group_pages): page u holds `most` keys that
// one of the tokens sees. Tiles past them read the page's last tile that has some.
struct GroupMap {
    const int2 *pages;   // LDS: {page, most}
    int P, pshift, Hk, h, len;
    __device__ __forceinline__ int2 page(int pos) const {
        const int2 e = pages[pos >> pshift];
        return make_int2(__builtin_amdgcn_readfirstlane(e.x), __builtin_amdgcn_readfirstlane(e.y));
    }
    __device__ __forceinline__ int first(int pos, int most) const { return min(pos & (P - 1), (most - 1) & ~15); }
    __device__ __forceinline__ long long row_s(int pos) const {
        const int2 e = page(pos);
        return ((long long)e.x * Hk + h) * P + first(pos, e.y);
    }
    __device__ __forceinline__ int last(int pos) const {
        const int most = page(pos).y;
        return most - 1 - first(pos, most);
    }
    __device__ __forceinline__ long long row(int) const { return 0; }   // whole tiles only
};

// Groups of tokens over chosen pages. The tables of up to GROUP_PAGES entries in all are joined into one
// list of pages in LDS, each with the number of its keys that each token sees (0: not in its table), so
// that a page that several tokens keep is read and multiplied once for all their rows. An entry's place is
// that of its first mention (position in the table first, then token): found with a hash table in LDS whose
// slots keep the smallest mention, so the list does not depend on the order of the threads. Where a token
// names a page twice, every entry is a page of its own. red: 2 + NT / 64 words of LDS; the last one then holds the
// tokens that have keys, a bit each.
constexpr int GROUP_PAGES = 1024, GROUP_SLOTS = 2 * GROUP_PAGES;
struct GroupLds {
    int2 pages[GROUP_PAGES];             // {page, keys that some token sees}
    union {
        struct {                         // while the list is made
            int id[GROUP_SLOTS], first[GROUP_SLOTS];
            uint32_t seen[GROUP_SLOTS];
        } slot;
        char rest[1];                    // then the value tiles
    };
};

template <int NT, typename Params>
__device__ __forceinline__ int group_pages(const Params &p, GroupLds &g, uint16_t *lim, int *red, int tok0, int h, int q0, int q1) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, K = p.bt_stride, TG = p.tg, entries = TG * K;
    constexpr int EACH = GROUP_PAGES / NT;
    int id[EACH], slot[EACH], keys[EACH];
    // both loads of an entry at once, in front of the LDS's clearing
#pragma unroll
    for (int n = 0; n < EACH; n++) {
        const int x = n * NT + tid, a = x / TG, tok = tok0 + x - a * TG;
        keys[n] = id[n] = 0;
        if (x < entries && tok < p.total) {
            keys[n] = p.lengths[tok * p.Hk + h];
            id[n] = p.bt[((size_t)tok * p.Hk + h) * K + a];
        }
    }
    for (int i = tid; i < GROUP_SLOTS; i += NT) g.slot.id[i] = -1, g.slot.first[i] = 0x7fffffff, g.slot.seen[i] = 0;
    for (int i = tid; i < entries * TG; i += NT) lim[i] = 0;
    if (tid == 0) red[0] = 0;
    __syncthreads();
#pragma unroll
    for (int n = 0; n < EACH; n++) {
        const int x = n * NT + tid, a = x / TG, tok = tok0 + x - a * TG;
        const int len = table_keys(keys[n], K * p.P);
        keys[n] = x < entries && tok >= q0 && tok < q1 ? min(len - a * p.P, p.P) : 0;
        id[n] = clamp_page(id[n], p.num_pages);
    }
    const unsigned long long keyed = __ballot(tid < TG && keys[0] > 0);   // wave 0: the tokens' first entries
    if (tid == 0) red[1 + NT / 64] = (int)keyed;
#pragma unroll
    for (int n = 0; n < EACH; n++) {
        if (keys[n] <= 0) continue;
        const int x = n * NT + tid;
        int s = (int)(((uint32_t)id[n] * 2654435761u) >> 21) & (GROUP_SLOTS - 1);
        while (true) {   // fewer entries than slots: a free one or the page's own is found
            const int was = atomicCAS(&g.slot.id[s], -1, id[n]);
            if (was == -1 || was == id[n]) break;
            s = (s + 1) & (GROUP_SLOTS - 1);
        }
        slot[n] = s;
        atomicMin(&g.slot.first[s], x);
        const uint32_t bit = 1u << (x % TG);
        if (atomicOr(&g.slot.seen[s], bit) & bit) red[0] = 1;   // named twice by one token
    }
    __syncthreads();
    const bool apart = red[0] != 0;
    // places in order of mention
    int base = 0;
#pragma unroll
    for (int n = 0; n < EACH; n++) {
        const int x = n * NT + tid;
        const bool first = keys[n] > 0 && (apart || g.slot.first[slot[n]] == x);
        const unsigned long long m = __ballot(first);
        __syncthreads();
        if (lane == 0) red[1 + w] = __popcll(m);
        __syncthreads();
        int at = base + __popcll(m & ((1ull << lane) - 1));
#pragma unroll
        for (int i = 0; i < NT / 64; i++) {
            if (i < w) at += red[1 + i];
            base += red[1 + i];
        }
        if (first) {
            g.pages[at] = make_int2(id[n], 0);
            if (!apart) g.slot.first[slot[n]] = -1 - at;   // its mentions find the place here
            else slot[n] = at;
        }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < EACH; n++) {
        if (keys[n] <= 0) continue;
        const int x = n * NT + tid, at = apart ? slot[n] : -1 - g.slot.first[slot[n]];
        lim[at * TG + x % TG] = (uint16_t)keys[n];
        atomicMax(&g.pages[at].y, keys[n]);
    }
    __syncthreads();   // the slots' LDS is free for the value tiles
    return base;
}

// A group's rows one by one on the vector ALUs, over the same tiles: where the matrix products of a dense
// cache met a value that is not finite. There a row's weight of 0 times such a value of a page that only
// other rows see is NaN; here a key that a row does not see is not touched. (INT8 values are finite, and
// a key's scales enter its own rows' weights only.) Slow: 9 ms where every group of 512 tokens meets one.
template <int D, typename Params>
__device__ __forceinline__ void group_rows(const Params &p, const int2 *pages, const uint16_t *lim, int tok0, int h, int q0, int q1,
                                           int j0, int j1, int nsp, size_t unit, int w, int nw, int lane) {
    using E = Elt<std::remove_pointer_t<decltype(Params::out)>>;
    constexpr int PER = D / 64;
    for (int r = w; r < p.M; r += nw) {
        const int t = r / p.G, tok = tok0 + t;
        if (tok < q0 || tok >= q1) continue;
        const size_t qrow = (size_t)tok * p.Hq + h * p.G + (r - t * p.G);
        float m = NEG_BIG, l = 0.0f, acc[PER];
#pragma unroll
        for (int k = 0; k < PER; k++) acc[k] = 0.0f;
        for (int j = j0; j < j1; j += 4) {
            const int pos = (j + (lane >> 4)) * 16 + (lane & 15);
            bool see = (j + (lane >> 4)) < j1;
            const int u = see ? pos >> p.pshift : 0, off = pos & (p.P - 1);
            see = see && off < lim[u * p.tg + t];
            const long long row = ((long long)pages[u].x * p.Hk + h) * p.P + off;
            float s = -INFINITY;
            if (see) {
                float dot = 0.0f;
                for (int d = 0; d < D; d++) dot += E::ld(p.q, qrow * D + d) * E::ld(p.kp, row * D + d);
                s = dot * p.scale_log2;
            }
            const float mn = fmaxf(m, wave_max(s));
            const float alpha = fast_exp2(m - mn), pr = see ? fast_exp2(s - mn) : 0.0f;
            m = mn;
            l = l * alpha + wave_sum(pr);
#pragma unroll
            for (int k = 0; k < PER; k++) acc[k] *= alpha;
            for (int i = 0; i < 64; i++) {
                if (!__shfl((int)see, i)) continue;
                const float pi = __shfl(pr, i);
                const long long ri = __shfl(row, i);
#pragma unroll
                for (int k = 0; k < PER; k++) acc[k] += pi * E::ld(p.vp, ri * D + lane + 64 * k);
            }
        }
        if (nsp == 1) {
#pragma unroll
            for (int k = 0; k < PER; k++) E::st(p.out, qrow * D + lane + 64 * k, l == 0.0f ? 0.0f : acc[k] / l);
        } else {
            float *dst = p.part + (unit * (size_t)p.M + r) * (D + 2);
#pragma unroll
            for (int k = 0; k < PER; k++) dst[lane + 64 * k] = acc[k];
            if (lane == 0) {
                dst[D] = m;
                dst[D + 1] = l;
            }
        }
    }
}

}  // namespace ti_group
