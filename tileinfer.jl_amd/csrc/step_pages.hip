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
// the slots' bytes.
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

// Running sums of a and b over the sequences (b in `sb`, a in `sa`, both with the total behind): every thread calls it.
struct Sums {
    int32_t a[MAX_SEQS + 1], b[MAX_SEQS + 1];
};
template <typename F>
__device__ __forceinline__ void running_sums(Sums &s, int n, long long &total_a, long long &total_b, F &&value) {
    __shared__ long long part[2][NT / 64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    long long ta = 0, tb = 0;
    for (int i0 = 0; i0 < n; i0 += NT) {
        const int i = i0 + (int)threadIdx.x;
        long long a = 0, b = 0;
        if (i < n) value(i, a, b);
        long long ia = a, ib = b;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const long long va = __shfl_up(ia, d), vb = __shfl_up(ib, d);
            if (lane >= d) ia += va, ib += vb;
        }
        __syncthreads();   // the last round's parts are read
        if (lane == 63) part[0][w] = ia, part[1][w] = ib;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NT / 64; k++) {
            if (k < w) ia += part[0][k], ib += part[1][k];
        }
        if (i < n) s.a[i] = (int32_t)min(ta + ia - a, 0x7fffffffLL), s.b[i] = (int32_t)min(tb + ib - b, 0x7fffffffLL);
#pragma unroll
        for (int k = 0; k < NT / 64; k++) ta += part[0][k], tb += part[1][k];
    }
    if (threadIdx.x == 0) s.a[n] = (int32_t)min(ta, 0x7fffffffLL), s.b[n] = (int32_t)min(tb, 0x7fffffffLL);
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
            const int was = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
            last = was == (int)gridDim.x - 1;
            if (last) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    __syncthreads();
    return last != 0;
}

__device__ __forceinline__ int32_t clamped(int32_t x, int32_t lo, int32_t hi) { return min(max(x, lo), hi); }

__global__ void __launch_bounds__(NT) reserve_kernel(PoolParams p) {
    __shared__ Sums s;                // tokens, pages
    __shared__ int wide;
    const ti_page_pool &pool = p.pool;
    const int S = pool.num_seqs, P = pool.page_size, have = clamped(pool.free_count[0], 0, pool.num_pages);
    if (threadIdx.x == 0) wide = 0;
    __syncthreads();
    long long tokens, pages;
    running_sums(s, S, tokens, pages, [&](int b, long long &a, long long &n) {
        const long long old = max(pool.lengths[b], 0);
        a = max(p.counts[b], 0);
        const long long to = old + a;
        const bool fits = to <= (long long)pool.table_width * P && to <= 0x7fffffffLL;
        if (!fits) wide = 1;
        n = fits ? pages_of(p, to) - pages_of(p, old) : 0;
    });
    const bool outgrown = wide || tokens > p.tokens;
    const bool ok = !outgrown && pages <= have;
    const int t_all = ok ? (int)tokens : 0;
    const int wg = blockIdx.x, wgs = gridDim.x;
    if (wg == 0) {
        for (int b = threadIdx.x; b <= S; b += NT) p.qsl[b] = ok ? s.a[b] : 0;
        if (threadIdx.x == 0) p.short_of[0] = ok ? 0 : (outgrown ? -1 : (int)min(pages - have, 0x7fffffffLL));
    }
    // page r of the step's: from the top of the stack down
    auto page_at = [&](int r) { return pool.free[have - 1 - r]; };
    if (ok) {
        for (int r = wg * NT + (int)threadIdx.x; r < (int)pages; r += wgs * NT) {
            const int b = find(s.b, S, r);
            const int held = pages_of(p, max(pool.lengths[b], 0));
            pool.tables[(size_t)b * pool.table_width + held + (r - s.b[b])] = page_at(r);
        }
    }
    for (int t = wg * NT + (int)threadIdx.x; t < p.tokens; t += wgs * NT) {
        int pos = 0, slot = 0;
        if (t < t_all) {
            const int b = find(s.a, S, t), old = max(pool.lengths[b], 0);
            pos = old + (t - s.a[b]);
            const int i = p.pshift >= 0 ? pos >> p.pshift : pos / P, held = pages_of(p, old);
            const int page = i < held ? pool.tables[(size_t)b * pool.table_width + i] : page_at(s.b[b] + i - held);
            slot = (page - 1) * P + (pos - i * P) + 1;
        }
        p.positions[t] = pos;
        p.slots[t] = slot;
    }
    if (!last_to_end(pool.ticket) || !ok) return;
    for (int b = threadIdx.x; b < S; b += NT) pool.lengths[b] = max(pool.lengths[b], 0) + (s.a[b + 1] - s.a[b]);
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
    long long pages, unused;
    running_sums(s, S, pages, unused, [&](int b, long long &a, long long &n) {
        a = gone_of(p, b).count();
        n = 0;
    });
    const int all = (int)min(pages, (long long)(pool.num_pages - have));   // never above the stack's room
    for (int r = blockIdx.x * NT + (int)threadIdx.x; r < all; r += gridDim.x * NT) {
        const int b = find(s.a, S, r);
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
    reserve_kernel<<<groups(tokens, 1024, 256), NT, 0, s>>>(p);
    return hipGetLastError() == hipSuccess ? TI_OK : TI_ERR_LAUNCH;
}

int ti_launch_release(const ti_page_pool *pool, const int32_t *keep, hipStream_t s) {
    const PoolParams p = params_of(pool, keep);
    release_kernel<<<groups((long long)pool->num_seqs * pool->table_width, 16384, 32), NT, 0, s>>>(p);
    return hipGetLastError() == hipSuccess ? TI_OK : TI_ERR_LAUNCH;
}
