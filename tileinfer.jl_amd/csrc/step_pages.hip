// The page bookkeeping of a step on the device: what BlockManager's reserve, slots, truncate and release
// (src/kv/block_manager.jl:58-100) do on the host, for all sequences of a batch in one launch.
//
// Every work-group reads the sequences' lengths and counts and makes their running sums (tokens, pages) in LDS for itself,
// so none waits for another; a token, or a page that changes hands, finds its sequence there by bisection. What the
// work-groups read (lengths, the stack's height) is changed once all of them have read it, by the one that ends last: each
// counts itself in `ticket` behind its work, the last sets it back to 0. Pages on the stack above its height are not
// overwritten by reserve, and release writes above the height and clears table entries that no work-group reads
// but the one that clears them.
//
// Bound: for the tables of a decode step one launch and its chain (lengths -> sums -> page -> slot -> ticket), for prompts
// the slots' bytes and the sums that every work-group makes for itself (256 sequences: 4 steps of 64). Measured: 8 drafted tokens
// for each of 32 sequences reserved and released 7.4 us, both calls (two launches of 1.9 and their chains); 256 prompts of 100 to
// 4096 tokens in pages of 16, 540 thousand slots, 10.6 + 5.4 us.
#include "common.hpp"

using namespace ti;

namespace {

constexpr int MAX_SEQS = 4096, NT = 256;

struct PoolParams {
    ti_page_pool pool;
    int pshift;                       // page_size = 2^pshift, or -1
    const int32_t *counts;            // reserve: more positions; release: positions kept
    int tokens;
    int32_t *positions, *slots, *qsl, *short_of;
};

__device__ __forceinline__ int pages_of(const PoolParams &p, long long positions) {
    return (int)(p.pshift >= 0 ? (positions + p.pool.page_size - 1) >> p.pshift : (positions + p.pool.page_size - 1) / p.pool.page_size);
}

// Running sums of a and b over the sequences, with the totals behind, and what else a sequence is asked for often:
// every thread calls it.
struct Sums {
    int32_t a[MAX_SEQS + 1], b[MAX_SEQS + 1], old[MAX_SEQS];
};
constexpr uint32_t FULL = 0x7fffffff;   // sums stay here once they get here (neither operand is above it: no wrap)
__device__ __forceinline__ uint32_t plus(uint32_t x, uint32_t y) { return min(x + y, FULL); }
template <typename F>
__device__ __forceinline__ void running_sums(Sums &s, int n, uint32_t &total_a, uint32_t &total_b, F &&value) {
    __shared__ uint2 part[NT / 64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t ta = 0, tb = 0;
    for (int i0 = 0; i0 < n; i0 += NT) {
        const int i = i0 + (int)threadIdx.x;
        uint32_t a = 0, b = 0;
        if (i < n) value(i, a, b);
        uint32_t ia = a, ib = b;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t va = __shfl_up(ia, d), vb = __shfl_up(ib, d);
            if (lane >= d) ia = plus(ia, va), ib = plus(ib, vb);
        }
        if (i0 > 0) __syncthreads();   // the last round's parts are read
        if (lane == 63) part[w] = make_uint2(ia, ib);
        __syncthreads();
        uint32_t before_a = ta, before_b = tb;
#pragma unroll
        for (int k = 0; k < NT / 64; k++) {
            const uint2 x = part[k];
            if (k < w) before_a = plus(before_a, x.x), before_b = plus(before_b, x.y);
            ta = plus(ta, x.x), tb = plus(tb, x.y);
        }
        // a sum that is full is of no use to anyone (reserve refuses, release has none)
        if (i < n) s.a[i] = (int32_t)(plus(before_a, ia) - a), s.b[i] = (int32_t)(plus(before_b, ib) - b);
    }
    if (threadIdx.x == 0) s.a[n] = (int32_t)ta, s.b[n] = (int32_t)tb;
    total_a = ta;
    total_b = tb;
    __syncthreads();
}

// The last i with sums[i] <= x: with empty entries at x, the one that x is in.
__device__ __forceinline__ int find(const int32_t *sums, int n, int x) {
    int lo = 0, hi = n;   // sums[lo] <= x < sums[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Whether this work-group is the last of the launch to end (every thread gets the answer; the ticket is 0 again).
__device__ __forceinline__ bool last_to_end(int32_t *ticket) {
    __shared__ int last;
    __syncthreads();   // what the work-group reads of the pool's state is read
    if (threadIdx.x == 0) {
        last = 1;
        if (gridDim.x > 1) {
            // Nothing is handed over through memory, so no fence (one writes an L2 back: 492 work-groups 20 -> 10.6 us):
            // what the others have read is in their registers and LDS.
            const int was = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last = was == (int)gridDim.x - 1;
            if (last) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    __syncthreads();
    return last != 0;
}

__device__ __forceinline__ int32_t clamped(int32_t x, int32_t lo, int32_t hi) { return min(max(x, lo), hi); }

// EACH: neighbouring tokens of a thread.
template <int EACH>
__global__ void __launch_bounds__(NT) reserve_kernel(PoolParams p) {
    __shared__ Sums s;                // tokens, pages
    __shared__ int wide;
    const ti_page_pool &pool = p.pool;
    const int S = pool.num_seqs, P = pool.page_size, have = clamped(pool.free_count[0], 0, pool.num_pages);
    if (threadIdx.x == 0) wide = 0;
    __syncthreads();
    uint32_t tokens, pages;
    running_sums(s, S, tokens, pages, [&](int b, uint32_t &a, uint32_t &n) {
        const long long old = max(pool.lengths[b], 0);
        s.old[b] = (int32_t)old;
        a = max(p.counts[b], 0);
        const long long to = old + a;
        const bool fits = to <= (long long)pool.table_width * P && to <= 0x7fffffffLL;
        if (!fits) wide = 1;
        n = fits ? pages_of(p, to) - pages_of(p, old) : 0;
    });
    const bool outgrown = wide || tokens > (uint32_t)p.tokens || tokens == FULL;
    const bool ok = !outgrown && pages <= (uint32_t)have;
    const int t_all = ok ? (int)tokens : 0;
    const int wg = blockIdx.x, wgs = gridDim.x;
    if (wg == 0) {
        for (int b = threadIdx.x; b <= S; b += NT) p.qsl[b] = ok ? s.a[b] : 0;
        if (threadIdx.x == 0) p.short_of[0] = ok ? 0 : (outgrown ? -1 : (int)(pages - have));
    }
    // page r of the step's: from the top of the stack down
    auto page_at = [&](int r) { return pool.free[have - 1 - r]; };
    if (ok) {
        for (uint32_t r = wg * NT + threadIdx.x; r < pages; r += wgs * NT) {   // (32 bits with no sign: a step further does not wrap)
            const int b = find(s.b, S, r);
            const int held = pages_of(p, s.old[b]);
            pool.tables[(size_t)b * pool.table_width + held + ((int)r - s.b[b])] = page_at((int)r);
        }
    }
    // Neighbouring tokens mostly share a sequence and a page: the chain of loads is walked once for them.
    const bool whole = ((((uintptr_t)p.positions | (uintptr_t)p.slots) & 15) == 0);
    for (uint32_t u0 = EACH * (wg * NT + threadIdx.x); u0 < (uint32_t)p.tokens; u0 += EACH * wgs * NT) {
        const int t0 = (int)u0;
        int pos[EACH], slot[EACH];
#pragma unroll
        for (int e = 0; e < EACH; e++) pos[e] = slot[e] = 0;
        if (t0 < t_all) {
            int b = find(s.a, S, t0), had = -1, base = 0;
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                const int t = t0 + e;
                if (t >= t_all) break;
                while (t >= s.a[b + 1]) b++, had = -1;
                const int old = s.old[b];
                pos[e] = old + (t - s.a[b]);
                const int i = p.pshift >= 0 ? pos[e] >> p.pshift : pos[e] / P;
                if (i != had) {
                    const int held = pages_of(p, old);
                    const int page = i < held ? pool.tables[(size_t)b * pool.table_width + i] : page_at(s.b[b] + i - held);
                    base = (page - 1 - i) * P + 1;
                    had = i;
                }
                slot[e] = base + pos[e];
            }
        }
        if constexpr (EACH == 4) {
            if (whole && t0 <= p.tokens - 4) {
                *reinterpret_cast<int4 *>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
                *reinterpret_cast<int4 *>(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
                continue;
            }
        }
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            if (t0 < p.tokens - e) p.positions[t0 + e] = pos[e], p.slots[t0 + e] = slot[e];
        }
    }
    if (!last_to_end(pool.ticket) || !ok) return;
    for (int b = threadIdx.x; b < S; b += NT) pool.lengths[b] = s.old[b] + (s.a[b + 1] - s.a[b]);
    if (threadIdx.x == 0) pool.free_count[0] = have - (int)pages;
}

// What a sequence gives back: table entries [a0, a1), [b0, b1) and [c0, c1), in this order.
struct Gone {
    int a0, a1, b0, b1, c0, c1, keep, behind;
    __device__ __forceinline__ int count() const { return (a1 - a0) + (b1 - b0) + (c1 - c0); }
    __device__ __forceinline__ int entry(int x) const {
        if (x < a1 - a0) return a0 + x;
        x -= a1 - a0;
        if (x < b1 - b0) return b0 + x;
        return c0 + x - (b1 - b0);
    }
};
__device__ __forceinline__ Gone gone_of(const PoolParams &p, int b) {
    const ti_page_pool &pool = p.pool;
    const int P = pool.page_size, len = max(pool.lengths[b], 0);
    Gone g;
    g.keep = clamped(p.counts[b], 0, len);
    const int held = min(pages_of(p, len), pool.table_width), stay = min(pages_of(p, g.keep), held);
    if (pool.window <= 0) {
        g.a0 = g.a1 = g.b0 = g.b1 = 0;
        g.c0 = stay;
        g.c1 = held;
        g.behind = 0;
        return g;
    }
    // pages [first, was) went back before; a query at `keep` sees positions from keep - window + 1 on
    const int first = min(pages_of(p, pool.sinks), pool.table_width), was = clamped(pool.behind[b], first, max(first, held));
    const long long lo = (long long)g.keep - pool.window + 1;
    const int hid = lo > 0 ? (int)min((long long)stay, p.pshift >= 0 ? lo >> p.pshift : lo / P) : 0;   // pages whole behind it
    const int from = clamped(was, first, max(first, stay));   // a sequence cut into what went back holds nothing there
    g.a0 = min(stay, first);
    g.a1 = min(held, first);
    g.b0 = from;
    g.b1 = max(from, hid);
    g.c0 = max(stay, max(first, was));
    g.c1 = max(g.c0, held);
    g.behind = g.b1;
    return g;
}

__global__ void __launch_bounds__(NT) release_kernel(PoolParams p) {
    __shared__ Sums s;                // pages; kept positions
    const ti_page_pool &pool = p.pool;
    const int S = pool.num_seqs, have = clamped(pool.free_count[0], 0, pool.num_pages);
    uint32_t pages, unused;
    running_sums(s, S, pages, unused, [&](int b, uint32_t &a, uint32_t &n) {
        a = gone_of(p, b).count();
        n = 0;
    });
    const int all = (int)min(pages, (uint32_t)(pool.num_pages - have));   // never above the stack's room
    for (uint32_t r0 = blockIdx.x * NT + threadIdx.x; r0 < (uint32_t)all; r0 += gridDim.x * NT) {
        const int r = (int)r0, b = find(s.a, S, r);
        int32_t *e = pool.tables + (size_t)b * pool.table_width + gone_of(p, b).entry(r - s.a[b]);
        pool.free[have + all - 1 - r] = *e;
        *e = 0;
    }
    if (!last_to_end(pool.ticket)) return;
    for (int b = threadIdx.x; b < S; b += NT) {
        const Gone g = gone_of(p, b);
        pool.lengths[b] = g.keep;
        if (pool.window > 0) pool.behind[b] = g.behind;
    }
    if (threadIdx.x == 0) pool.free_count[0] = have + all;
}

PoolParams params_of(const ti_page_pool *pool, const int32_t *counts) {
    PoolParams p{};
    p.pool = *pool;
    p.pshift = (pool->page_size & (pool->page_size - 1)) == 0 ? __builtin_ctz(pool->page_size) : -1;
    p.counts = counts;
    return p;
}

// Work-groups: one per `each` items, at most `most`.
unsigned groups(long long items, int each, int most) { return (unsigned)max(1LL, min((items + each - 1) / each, (long long)most)); }

}  // namespace

int ti_launch_reserve(const ti_page_pool *pool, const int32_t *counts, int tokens, int32_t *positions, int32_t *slots, int32_t *qsl,
                      int32_t *short_of, hipStream_t s) {
    PoolParams p = params_of(pool, counts);
    p.tokens = tokens;
    p.positions = positions;
    p.slots = slots;
    p.qsl = qsl;
    p.short_of = short_of;
    // one token a thread for steps of a few tokens a sequence, whose chains are the time; four for prompts
    if (tokens < 65536) reserve_kernel<1><<<groups(tokens, NT, 256), NT, 0, s>>>(p);
    else reserve_kernel<4><<<groups(tokens, 4 * NT, 512), NT, 0, s>>>(p);
    return hipGetLastError() == hipSuccess ? TI_OK : TI_ERR_LAUNCH;
}

int ti_launch_release(const ti_page_pool *pool, const int32_t *keep, hipStream_t s) {
    const PoolParams p = params_of(pool, keep);
    release_kernel<<<groups((long long)pool->num_seqs * pool->table_width, 4 * NT, 256), NT, 0, s>>>(p);
    return hipGetLastError() == hipSuccess ? TI_OK : TI_ERR_LAUNCH;
}
