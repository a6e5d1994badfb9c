// Writes into 8-bit block caches (TI_KV_FP8): e4m3 values, one power of two per page, KV head and half (keys, values).
//
// A block's scale is the least 2^e with |x| <= 448 2^e over the rows that it was written with (448: the largest e4m3
// value), so a row's place in a block cannot be decided without the block's other rows. One work-group therefore owns a page
// (for some of the KV heads): the one of the page's first token in the call. It finds all tokens of the page, wherever
// they are among the call's, takes the largest magnitude of their keys and values, grows the block's scale if it must (and
// divides the rows that the block already holds), and writes the new rows. Nothing depends on the order of threads: the
// largest magnitude is a maximum, and of two tokens of one slot the later is written.
//
// Bound: a prompt's bytes (2 + 1 per element of k and v), one token's chain slots -> rows -> largest -> rows out. Measured
// (8 heads of 128, bf16): 8192 tokens into pages of 16 16.4 us, 3.05 TB/s (rows stay in registers between the two passes; 34.8 us
// with rows read twice): slots -> page's list -> rows -> largest -> rows out go one after the other in a work-group, and two
// rounds of work-groups fill the CUs; one token for each of 32 sequences 4.0 us, of which 1.9 are a launch. Two forms read full
// pages twice, as their rows do not fit the registers (KEEP below): Float32 rows (26.3 us, 3.2 TB/s) and fused calls, which norm and
// rotate each key twice too (32 query heads, 8192 tokens into pages of 16 84 us, of 64 94, where the dense cache's fused write
// takes 40 and INT8's 47; a token for each of 32 sequences 4.9). A work-group has all of a page, so large pages leave CUs idle: 8192
// tokens into pages of 64 / 128 / 256 / 1024 16.3 / 27 / 47 / 160 us, fused into pages of 1024 655.
//
// The fused kernel rotates queries and keys with every rounding of attention_inputs_v_kernel (kv_write.hip), so it is
// bit-identical to rmsnorm, rope and store_kv in a row: products and sums are rounded one by one.
#pragma clang fp contract(off)

#include <type_traits>

#include "kv_rows.hpp"

using namespace ti;

namespace {

constexpr int MAX_PAGE = 1024, MAX_HEADS = 16;   // keys of a page, KV heads worked on together
constexpr int SHARE = 4;   // pages whose rows are looked for in one pass over the slots

struct Fp8WriteParams {
    const void *k, *v;               // store: [n][Hk][D]
    const void *qkv, *q_norm, *k_norm, *cos_sin;   // fused: [n][nq + 2 Hk][D]
    void *q_out;
    uint8_t *q8;                     // [2][pages][Hk][P][D]
    float *scale;                    // [2][pages][Hk]
    const int32_t *slots, *positions;
    int n, nq, Hk, P, pshift, pages, table_len;
    int chunk, hpg, hgroups, hloop;  // tokens of a work-group; KV heads worked on together, groups of them, groups of a work-group
    int hwgs;                        // work-groups of a chunk of tokens: hgroups / hloop, rounded up
    unsigned page_groups;            // work-groups that write pages; the others rotate queries
    float eps;
};

// The least power of two (2^-120 to 2^120) that 448 times it is no less than `most`.
__device__ __forceinline__ float least_scale(float most) {
    const int x = __builtin_amdgcn_frexp_expf(most);   // most = f 2^x, f in [0.5, 1); 448 = 0.875 2^9
    int e = __builtin_amdgcn_frexp_mantf(most) <= 0.875f ? x - 9 : x - 8;
    e = most > 0.0f ? min(max(e, -120), 120) : -120;
    return __uint_as_float((uint32_t)(e + 127) << 23);
}
__device__ __forceinline__ float inverse(float pow2) { return __uint_as_float((254u << 23) - __float_as_uint(pow2)); }

// Four values in e4m3, to nearest even; what is not finite becomes NaN.
__device__ __forceinline__ uint32_t to_e4m3(const float *x, float mul) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = fabsf(x[e]) < INFINITY ? x[e] * mul : __uint_as_float(0x7fc00000u);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}

// A head's vector with its norm and rotation, as attention_inputs_v_kernel: lane u of the head holds elements
// 4 u .. and D / 2 + 4 u .. .
template <typename T, bool NORM, int D>
__device__ __forceinline__ void rotated(const T *x, const T *w, const T *cs, float eps, int u, float (&y)[8]) {
    constexpr int HALF = D / 2, LPH = D / 8;
    using E = Elt<T>;
    using V = Vec4<T>;
    float a[4], b[4], c1[4], c2[4], s1[4], s2[4];
    V::ld(x + 4 * u, a);
    V::ld(x + HALF + 4 * u, b);
    V::ld(cs + 4 * u, c1);
    V::ld(cs + HALF + 4 * u, c2);
    V::ld(cs + D + 4 * u, s1);
    V::ld(cs + D + HALF + 4 * u, s2);
    if (NORM) {
        float w1[4], w2[4], pp[4];
        V::ld(w + 4 * u, w1);
        V::ld(w + HALF + 4 * u, w2);
#pragma unroll
        for (int e = 0; e < 4; e++) pp[e] = a[e] * a[e] + b[e] * b[e];
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1)
#pragma unroll
            for (int e = 0; e < 4; e++) pp[e] = pp[e] + __shfl_xor(pp[e], o);
        const float ss = (pp[0] + pp[2]) + (pp[1] + pp[3]);
        const float inv_rms = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)D), eps)));
#pragma unroll
        for (int e = 0; e < 4; e++) {
            a[e] = E::rnd(E::rnd(a[e] * inv_rms) * w1[e]);
            b[e] = E::rnd(E::rnd(b[e] * inv_rms) * w2[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        y[e] = E::rnd(E::rnd(a[e] * c1[e]) + E::rnd(-b[e] * s1[e]));
        y[4 + e] = E::rnd(E::rnd(b[e] * c2[e]) + E::rnd(a[e] * s2[e]));
    }
}

template <int N> using IC = std::integral_constant<int, N>;

// Eight elements held between the passes in their own type's bits (a rotated bf16 key is rounded to bf16 already).
template <typename T> struct Held;
template <> struct Held<uint16_t> {
    u32x4 w;
    __device__ __forceinline__ void put(const float (&x)[8]) {
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
    }
    __device__ __forceinline__ void ld(const uint16_t *p) { w = *reinterpret_cast<const u32x4 *>(p); }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 4; e++) x[2 * e] = __uint_as_float(w[e] << 16), x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
};
template <> struct Held<float> {
    f32x4 lo, hi;
    __device__ __forceinline__ void put(const float (&x)[8]) {
#pragma unroll
        for (int e = 0; e < 4; e++) lo[e] = x[e], hi[e] = x[4 + e];
    }
    __device__ __forceinline__ void ld(const float *p) {
        lo = *reinterpret_cast<const f32x4 *>(p);
        hi = *reinterpret_cast<const f32x4 *>(p + 4);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = lo[e], x[4 + e] = hi[e];
    }
};

// FEW: at most a token for each thread, one for each work-group, whose slots are read once, beside the rows of the
// work-group's own token.
template <typename T, bool FUSED, bool NORM, int D, bool FEW>
__global__ void __launch_bounds__(256) fp8_write_kernel(Fp8WriteParams p) {
    constexpr int HALF = D / 2, LPH = D / 8, NT = 256, NG = NT / LPH;
    using V = Vec4<T>;
    __shared__ int srcs[MAX_PAGE];                    // the token that writes each row of up to SHARE pages, or -1
    __shared__ int taken;                             // those of them that a token in front of the chunk's has
    __shared__ uint16_t lists[NT / 64][MAX_PAGE];     // the rows that are written, a copy for each wave
    __shared__ uint32_t most[2 * MAX_HEADS];
    __shared__ float inv[2 * MAX_HEADS], ratio[2 * MAX_HEADS];
    const int tid = threadIdx.x, lane = tid & 63, u = tid % LPH, gid = tid / LPH;
    uint16_t *list = lists[tid >> 6];
    if (FUSED && blockIdx.x >= p.page_groups) {
        const long long item = (long long)(blockIdx.x - p.page_groups) * NG + gid;
        const int t = (int)(item / p.nq), j = (int)(item - (long long)t * p.nq);
        if (t >= p.n) return;   // a whole lane group
        const int pos = p.positions[t];
        if (pos < 0 || pos >= p.table_len) return;
        float y[8];
        rotated<T, NORM, D>((const T *)p.qkv + ((size_t)t * (p.nq + 2 * p.Hk) + j) * D, (const T *)p.q_norm,
                            (const T *)p.cos_sin + (size_t)pos * 2 * D, p.eps, u, y);
        T *dst = (T *)p.q_out + ((size_t)t * p.nq + j) * D;
        const float lo[4] = {y[0], y[1], y[2], y[3]}, hi[4] = {y[4], y[5], y[6], y[7]};
        V::st(dst + 4 * u, lo);
        V::st(dst + HALF + 4 * u, hi);
        return;
    }
    // 0-based page of a slot, -1 for one outside the pool; whether a token writes at all
    const int limit = (int)min((long long)p.pages * p.P, 0x7fffffffLL);
    auto page_of_slot = [&](int s) { return s > 0 && s <= limit ? (s - 1) >> p.pshift : -1; };
    auto writes = [&](int j) {
        if (!FUSED) return true;
        const int pos = p.positions[j];
        return pos >= 0 && pos < p.table_len;
    };
    const int chunk = FEW ? 1 : p.chunk, hloop = FEW ? 1 : p.hloop;
    const int c0 = (int)(blockIdx.x / (unsigned)p.hwgs) * chunk, g0 = (int)(blockIdx.x % (unsigned)p.hwgs) * hloop;
    int h0 = g0 * p.hpg, heads = min(p.hpg, p.Hk - h0);   // of the group of heads that is worked on
    auto load = [&](int t, int hh, Held<T> &x) {
        const int half = hh >= heads, h = h0 + hh - half * heads;
        if constexpr (FUSED) {
            const T *x0 = (const T *)p.qkv + ((size_t)t * (p.nq + 2 * p.Hk) + p.nq + (size_t)half * p.Hk + h) * D;
            if (half) return x.ld(x0 + 8 * u);
            float y[8];
            rotated<T, NORM, D>(x0, (const T *)p.k_norm, (const T *)p.cos_sin + (size_t)p.positions[t] * 2 * D, p.eps, u, y);
            x.put(y);
        } else {
            x.ld((const T *)(half ? p.v : p.k) + ((size_t)t * p.Hk + h) * D + 8 * u);
        }
    };
    const int my_slot = FEW && tid < p.n ? p.slots[tid] : 0;
    // One token a work-group: its rows are on their way while the slots are looked through.
    Held<T> mine;
    if (FEW && (!FUSED || writes(c0))) load(c0, min(gid, 2 * heads - 1), mine);
    // The chunk's tokens (at most 64) that write to another page than the one in front of them: one lane each.
    int first_page = -1;
    if (lane < chunk && c0 + lane < p.n && writes(c0 + lane)) {
        first_page = page_of_slot(p.slots[c0 + lane]);
        if (c0 + lane > 0 && writes(c0 + lane - 1) && page_of_slot(p.slots[c0 + lane - 1]) == first_page) first_page = -1;
    }
    unsigned long long starts = __ballot(first_page >= 0);
    // the next page that begins in the chunk: its first token here
    auto next_start = [&] {
        const int at = __builtin_ctzll(starts);
        starts &= starts - 1;
        return at;
    };
    while (starts) {
        // Up to SHARE pages at a time, whose rows are looked for in one pass over the slots.
        int at[SHARE], first[SHARE], pages = 0;
        unsigned span[SHARE];
        const int fit = FEW ? 1 : min(SHARE, MAX_PAGE >> p.pshift);
#pragma unroll
        for (int k = 0; k < SHARE; k++) {
            at[k] = first[k] = 0;
            span[k] = 0;
            if (k < fit && starts) {
                at[k] = next_start();
                first[k] = (__builtin_amdgcn_readlane(first_page, at[k]) << p.pshift) + 1;   // the page's first slot
                span[k] = (unsigned)min(p.P, limit - first[k] + 1);
                pages = k + 1;
            }
        }
        for (int o = tid; o < pages << p.pshift; o += NT) srcs[o] = -1;
        if (tid == 0) taken = 0;
        // (few tokens: the scales are on their way beside the slots)
        float early = 0.0f;
        if (tid < 2 * heads) {
            const int half = tid >= heads;
            early = p.scale[((size_t)half * p.pages + ((first[0] - 1) >> p.pshift)) * p.Hk + h0 + tid - half * heads];
            most[tid] = 0u;
        }
        __syncthreads();
        // All tokens of the pages, wherever they are; one in front of the chunk's has the page. A slot is of page k where it is
        // less than `span` past the page's first one, as unsigned numbers: none outside the pool is.
        int earlier = 0;
        auto look = [&](auto many) {
            constexpr int N = decltype(many)::value;
            auto take = [&](int s, int j) {
#pragma unroll
                for (int k = 0; k < N; k++) {
                    const unsigned o = (unsigned)s - (unsigned)first[k];
                    if (o < span[k] && writes(j)) {
                        if (j < c0 + at[k]) earlier |= 1 << k;
                        else atomicMax(&srcs[(k << p.pshift) + (int)o], j);
                    }
                }
            };
            if (((uintptr_t)p.slots & 15) == 0) {
                const int quads = p.n >> 2;
                for (int q0 = tid; q0 < quads; q0 += 4 * NT) {
                    int4 s[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) s[e] = reinterpret_cast<const int4 *>(p.slots)[min(q0 + e * NT, quads - 1)];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int j = 4 * (q0 + e * NT);
                        if (q0 + e * NT < quads) take(s[e].x, j), take(s[e].y, j + 1), take(s[e].z, j + 2), take(s[e].w, j + 3);
                    }
                }
                if (tid < (p.n & 3)) take(p.slots[4 * quads + tid], 4 * quads + tid);
            } else {
                for (int j = tid; j < p.n; j += NT) take(p.slots[j], j);
            }
        };
        if constexpr (FEW) {
            const unsigned o = (unsigned)my_slot - (unsigned)first[0];
            if (tid < p.n && o < span[0] && writes(tid)) {
                if (tid < c0) earlier = 1;
                else atomicMax(&srcs[o], tid);
            }
        } else {
            if (pages == 1) look(IC<1>{});
            else look(IC<SHARE>{});
        }
        if (earlier) atomicOr(&taken, earlier);
        __syncthreads();
        const int done = taken;
        for (int k = 0; k < pages; k++) {
            if (done >> k & 1) continue;
            int slot0 = first[0];
#pragma unroll
            for (int j = 1; j < SHARE; j++) slot0 = k == j ? first[j] : slot0;
            const int page = (slot0 - 1) >> p.pshift;
            const int *src = srcs + (k << p.pshift);
            int count = 0;
            for (int o0 = 0; o0 < p.P; o0 += 64) {
                const int o = o0 + lane;
                const bool has = o < p.P && src[o] >= 0;
                const unsigned long long m = __ballot(has);
                if (has) list[count + __popcll(m & ((1ull << lane) - 1))] = (uint16_t)o;
                count += __popcll(m);
            }
            for (int hg = 0; hg < hloop && g0 + hg < p.hgroups; hg++) {
                h0 = (g0 + hg) * p.hpg, heads = min(p.hpg, p.Hk - h0);
                // the blocks' scales, needed below
                float *sp = nullptr;
                float old = 0.0f;
                if (tid < 2 * heads) {
                    const int half = tid >= heads;
                    sp = p.scale + ((size_t)half * p.pages + page) * p.Hk + h0 + tid - half * heads;
                    old = early;
                }
                if (k > 0 || hg > 0) {
                    if (tid < 2 * heads) old = *sp, most[tid] = 0u;
                    __syncthreads();
                }
                // Vectors of the page's new rows: (row, half, head), heads innermost; one per lane group at a time. A lane holds
                // elements 8 u .. 8 u + 7, of a rotated key 4 u .. and D / 2 + 4 u .. .
                const int vectors = count * 2 * heads;
                auto place = [&](int vec, int &row, int &hh) {
                    const int r = vec / (2 * heads);
                    hh = vec - r * 2 * heads;                // half * heads + head
                    row = list[r];
                };
                auto largest = [&](const Held<T> &held, int hh) {
                    float x[8], m = 0.0f;
                    held.get(x);
#pragma unroll
                    for (int e = 0; e < 8; e++) m = fmaxf(m, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.0f);
#pragma unroll
                    for (int o = LPH / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
                    if (u == 0) atomicMax(&most[hh], __float_as_uint(m));   // of no sign: ordered as whole numbers
                };
                uint8_t *base = p.q8 + (((size_t)page * p.Hk + h0) << p.pshift) * D;
                const size_t half_q = (((size_t)p.pages * p.Hk) << p.pshift) * D;
                auto store = [&](const Held<T> &held, int row, int hh) {
                    float x[8];
                    held.get(x);
                    const int half = hh >= heads;
                    uint8_t *dst = base + half * half_q + ((((size_t)(hh - half * heads)) << p.pshift) + row) * D;
                    const uint32_t lo = to_e4m3(x, inv[hh]), hi = to_e4m3(x + 4, inv[hh]);
                    if (FUSED && !half) {
                        *reinterpret_cast<uint32_t *>(dst + 4 * u) = lo;
                        *reinterpret_cast<uint32_t *>(dst + HALF + 4 * u) = hi;
                    } else {
                        *reinterpret_cast<u32x2 *>(dst + 8 * u) = (u32x2){lo, hi};
                    }
                };
                // between the two passes: the blocks' scales, and the rows that they hold already
                auto scales = [&] {
                    __syncthreads();
                    bool grown = false;
                    if (tid < 2 * heads) {
                        const float need = least_scale(__uint_as_float(most[tid]));
                        const bool fresh = src[0] >= 0 || !(old > 0.0f && old < INFINITY);
                        const float now = fresh ? need : fmaxf(old, need);
                        inv[tid] = inverse(now);
                        ratio[tid] = fresh ? 1.0f : old * inverse(now);
                        grown = ratio[tid] < 1.0f;
                        if (now != old) *sp = now;
                    }
                    if (!__syncthreads_or(grown)) return;
                    // 16 bytes at a time
                    for (int c = tid; c < 2 * heads * p.P * (D / 16); c += NT) {
                        const int d16 = c % (D / 16), o = (c / (D / 16)) & (p.P - 1), hh = (c / (D / 16)) >> p.pshift;
                        const float f = ratio[hh];
                        if (src[o] >= 0 || f == 1.0f) continue;
                        const int half = hh >= heads;
                        u32x4 *at16 = reinterpret_cast<u32x4 *>(base + half * half_q + ((((size_t)(hh - half * heads)) << p.pshift) + o) * D) + d16;
                        u32x4 w = *at16;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float x[4] = {__builtin_amdgcn_cvt_f32_fp8((int)w[e], 0), __builtin_amdgcn_cvt_f32_fp8((int)w[e], 1),
                                                __builtin_amdgcn_cvt_f32_fp8((int)w[e], 2), __builtin_amdgcn_cvt_f32_fp8((int)w[e], 3)};
                            w[e] = to_e4m3(x, f);
                        }
                        *at16 = w;
                    }
                };
                // KEEP vectors of a lane group stay in registers between the passes, loaded together; more are read twice (a full page
                // is 8: bf16 rows fit, Float32 and rotated ones do not).
                auto rows = [&](auto keep) {
                    constexpr int KEEP = decltype(keep)::value;
                    Held<T> x[KEEP];
                    int row[KEEP], hh[KEEP];
                    auto read = [&](int v0) {
#pragma unroll
                        for (int k = 0; k < KEEP; k++) {
                            place(min(v0 + k * NG, vectors - 1), row[k], hh[k]);
                            if (KEEP == 1 && FEW && count == 1 && src[row[k]] == c0) x[k] = mine;
                            else load(src[row[k]], hh[k], x[k]);
                        }
                    };
                    for (int v0 = gid; v0 < vectors || v0 == gid; v0 += KEEP * NG) {
                        read(v0);
#pragma unroll
                        for (int k = 0; k < KEEP; k++) largest(x[k], hh[k]);   // (a vector twice is as good as once)
                    }
                    scales();
                    for (int v0 = gid; v0 < vectors; v0 += KEEP * NG) {
                        if (vectors > KEEP * NG) read(v0);
#pragma unroll
                        for (int k = 0; k < KEEP; k++)
                            if (v0 + k * NG < vectors) store(x[k], row[k], hh[k]);
                    }
                };
                if (vectors <= NG) rows(IC<1>{});
                else if (vectors <= 4 * NG || FUSED || sizeof(T) == 4) rows(IC<4>{});
                else rows(IC<8>{});
                __syncthreads();   // the lists and scales are read
            }
            h0 = g0 * p.hpg, heads = min(p.hpg, p.Hk - h0);
        }
        if (starts) __syncthreads();   // `taken` is read
    }
}

constexpr int LONG_GROUPS = 1024;

template <typename T, bool FUSED, bool NORM>
int launch(Fp8WriteParams &p, int D, hipStream_t s) {
    // Tokens of a work-group: one where there are few, a page's rows for prompts. KV heads worked on together: so many that a
    // page's rows are one or eight vectors for each of its lane groups. Few tokens may be one of each sequence or all of
    // one page: two heads up to 32 tokens, one up to 64 (in place of eight: 17 tokens of 3 sequences 17.0 -> 6.5 us, 64
    // of one 39.2 -> 8.2, one each of 32 and 64 5.4 as before, all in a graph of 6 calls).
    const int per = 256 / (D / 8);   // lane groups
    p.chunk = p.n <= 256 ? 1 : min(p.P, 64);
    p.hpg = max(1, min(min(p.Hk, MAX_HEADS), p.n <= 32 ? 2 : p.n <= 64 ? 1 : 4 * per / min(p.P, 64)));
    p.hgroups = (p.Hk + p.hpg - 1) / p.hpg;
    p.hloop = 1;
    auto groups = [&] { return (long long)(p.n + p.chunk - 1) / p.chunk * ((p.hgroups + p.hloop - 1) / p.hloop); };
    // Every work-group looks through all slots, so long prompts have fewer of them, but 1024 at least: all heads, then more
    // pages (32768 tokens in pages of 64 78 -> 52 us, 131072 682 -> 230, in pages of 16 682 -> 329; with 512 8192 take 3 us more).
    while (p.chunk > 1 && p.hloop < p.hgroups && groups() >= 2 * LONG_GROUPS) p.hloop *= 2;
    while (p.chunk > 1 && 2 * p.chunk <= 64 && groups() >= 2 * LONG_GROUPS) p.chunk *= 2;
    p.hwgs = (p.hgroups + p.hloop - 1) / p.hloop;
    const long long pages = groups();
    const long long queries = FUSED ? ((long long)p.n * p.nq + per - 1) / per : 0;
    if ((pages + queries) * 256 > MAX_THREADS) return TI_ERR_UNSUPPORTED;
    p.page_groups = (unsigned)pages;
    const unsigned grid = (unsigned)(pages + queries);
    const bool few = p.chunk == 1;
    if (D == 128 && few) fp8_write_kernel<T, FUSED, NORM, 128, true><<<grid, 256, 0, s>>>(p);
    else if (D == 128) fp8_write_kernel<T, FUSED, NORM, 128, false><<<grid, 256, 0, s>>>(p);
    else if (few) fp8_write_kernel<T, FUSED, NORM, 64, true><<<grid, 256, 0, s>>>(p);
    else fp8_write_kernel<T, FUSED, NORM, 64, false><<<grid, 256, 0, s>>>(p);
    return hipGetLastError() == hipSuccess ? TI_OK : TI_ERR_LAUNCH;
}

Fp8WriteParams params_of(const ti_kv_cache *c, const int32_t *slots, int n) {
    Fp8WriteParams p{};
    p.q8 = (uint8_t *)c->layer_q;
    p.scale = c->layer_scale;
    p.slots = slots;
    p.n = n;
    p.Hk = c->kv_heads;
    p.P = c->page_size;
    p.pshift = __builtin_ctz(c->page_size);
    p.pages = c->num_pages;
    return p;
}

}  // namespace

int ti_launch_store_fp8(int dtype, const ti_kv_cache *c, const void *k, const void *v, const int32_t *slots, int n,
                        hipStream_t s) {
    Fp8WriteParams p = params_of(c, slots, n);
    p.k = k;
    p.v = v;
    return dtype == TI_BF16 ? launch<uint16_t, false, false>(p, c->head_dim, s) : launch<float, false, false>(p, c->head_dim, s);
}

int ti_launch_inputs_fp8(int dtype, void *q_out, const ti_kv_cache *c, const void *qkv, const void *q_norm, const void *k_norm,
                         const void *cos_sin, int table_len, const int32_t *positions, const int32_t *slots, int n,
                         int q_heads, float eps, hipStream_t s) {
    Fp8WriteParams p = params_of(c, slots, n);
    p.qkv = qkv;
    p.q_norm = q_norm;
    p.k_norm = k_norm;
    p.cos_sin = cos_sin;
    p.q_out = q_out;
    p.positions = positions;
    p.nq = q_heads;
    p.table_len = table_len;
    p.eps = eps;
    if (dtype == TI_BF16)
        return q_norm ? launch<uint16_t, true, true>(p, c->head_dim, s) : launch<uint16_t, true, false>(p, c->head_dim, s);
    return q_norm ? launch<float, true, true>(p, c->head_dim, s) : launch<float, true, false>(p, c->head_dim, s);
}
