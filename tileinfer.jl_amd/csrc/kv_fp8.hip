// Writes into 8-bit block caches (TI_KV_FP8): e4m3 values, one power of two per page, KV head and half (keys, values).
//
// A block's scale is the least 2^e with |x| <= 448 2^e over the rows that it was written with (448: the largest e4m3
// value), so a row's place in a block cannot be decided without the block's other rows. One work-group therefore owns a page
// (for some of the KV heads): the one of the page's first token in the call. It finds all tokens of the page, wherever
// they are among the call's, takes the largest magnitude of their keys and values, grows the block's scale if it must (and
// divides the rows that the block already holds), and writes the new rows. Nothing depends on the order of threads: the
// largest magnitude is a maximum, and of two tokens of one slot the later is written.
//
// Bound: a prompt's HBM bytes (2 + 1 per element of k and v), one token's chain slots -> rows -> largest -> rows out.
//
// The fused kernel rotates queries and keys with every rounding of attention_inputs_v_kernel (kv_write.hip), so it is
// bit-identical to rmsnorm, rope and store_kv in a row: products and sums are rounded one by one.
#pragma clang fp contract(off)

#include "kv_rows.hpp"

using namespace ti;

namespace {

constexpr int MAX_PAGE = 1024, MAX_HEADS = 16;   // keys of a page, KV heads of a work-group

struct Fp8WriteParams {
    const void *k, *v;               // store: [n][Hk][D]
    const void *qkv, *q_norm, *k_norm, *cos_sin;   // fused: [n][nq + 2 Hk][D]
    void *q_out;
    uint8_t *q8;                     // [2][pages][Hk][P][D]
    float *scale;                    // [2][pages][Hk]
    const int32_t *slots, *positions;
    int n, nq, Hk, P, pshift, pages, table_len;
    int chunk, hpg, hgroups;         // tokens and KV heads of a work-group, groups of heads
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

template <typename T, bool FUSED, bool NORM, int D>
__global__ void __launch_bounds__(256) fp8_write_kernel(Fp8WriteParams p) {
    constexpr int HALF = D / 2, LPH = D / 8, NT = 256, NG = NT / LPH;
    using V = Vec4<T>;
    __shared__ int src[MAX_PAGE];              // the token that writes each row of the page, or -1
    __shared__ int list[MAX_PAGE];             // the rows that are written
    __shared__ int count;
    __shared__ uint32_t most[2 * MAX_HEADS];
    __shared__ float inv[2 * MAX_HEADS], ratio[2 * MAX_HEADS];
    const int tid = threadIdx.x, u = tid % LPH, gid = tid / LPH;
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
    // 0-based page of token j's slot, -1 where the token writes nothing
    const int limit = (int)min((long long)p.pages * p.P, 0x7fffffffLL);
    auto page_of_token = [&](int j) {
        const int s = p.slots[j];
        bool ok = s > 0 && s <= limit;
        if (FUSED) {
            const int pos = p.positions[j];
            ok = ok && pos >= 0 && pos < p.table_len;
        }
        return ok ? (s - 1) >> p.pshift : -1;
    };
    const int c0 = (int)(blockIdx.x / (unsigned)p.hgroups) * p.chunk, h0 = (int)(blockIdx.x % (unsigned)p.hgroups) * p.hpg;
    const int heads = min(p.hpg, p.Hk - h0), c1 = min(c0 + p.chunk, p.n);
    for (int i = c0; i < c1; i++) {
        const int page = page_of_token(i);
        if (page < 0 || (i > 0 && page_of_token(i - 1) == page)) continue;
        bool earlier = false;
        for (int j = tid; j < i; j += NT) earlier |= page_of_token(j) == page;
        if (__syncthreads_or(earlier)) continue;   // that one's work-group has the page
        for (int o = tid; o < p.P; o += NT) src[o] = -1;
        if (tid < 2 * heads) most[tid] = 0u;
        __syncthreads();
        for (int j = i + tid; j < p.n; j += NT)
            if (page_of_token(j) == page) atomicMax(&src[(p.slots[j] - 1) & (p.P - 1)], j);
        __syncthreads();
        if (tid < 64) {
            int c = 0;
            for (int o0 = 0; o0 < p.P; o0 += 64) {
                const int o = o0 + tid;
                const bool has = o < p.P && src[o] >= 0;
                const unsigned long long m = __ballot(has);
                if (has) list[c + __popcll(m & ((1ull << tid) - 1))] = o;
                c += __popcll(m);
            }
            if (tid == 0) count = c;
        }
        __syncthreads();
        // vectors of the page's new rows: (row, half, head), heads innermost; one per lane group at a time
        const int vectors = count * 2 * heads;
        auto load = [&](int vec, float (&x)[8], int &row, int &hh) {
            const int r = vec / (2 * heads);
            hh = vec - r * 2 * heads;                // half * heads + head
            row = list[r];
            const int t = src[row], half = hh >= heads, h = h0 + hh - half * heads;
            if constexpr (FUSED) {
                const T *x0 = (const T *)p.qkv + ((size_t)t * (p.nq + 2 * p.Hk) + p.nq + h) * D;
                if (!half) {
                    rotated<T, NORM, D>(x0, (const T *)p.k_norm, (const T *)p.cos_sin + (size_t)p.positions[t] * 2 * D, p.eps, u, x);
                    return;
                }
                x0 += (size_t)p.Hk * D;
                float lo[4], hi[4];
                V::ld(x0 + 4 * u, lo);
                V::ld(x0 + HALF + 4 * u, hi);
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = lo[e], x[4 + e] = hi[e];
            } else {
                const T *x0 = (const T *)(half ? p.v : p.k) + ((size_t)t * p.Hk + h) * D;
                float lo[4], hi[4];
                V::ld(x0 + 4 * u, lo);
                V::ld(x0 + HALF + 4 * u, hi);
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = lo[e], x[4 + e] = hi[e];
            }
        };
        for (int vec = gid; vec < vectors; vec += NG) {
            float x[8], m = 0.0f;
            int row, hh;
            load(vec, x, row, hh);
#pragma unroll
            for (int e = 0; e < 8; e++) m = fmaxf(m, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.0f);
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
            if (u == 0) atomicMax(&most[hh], __float_as_uint(m));   // of no sign: ordered as whole numbers
        }
        __syncthreads();
        bool grown = false;
        if (tid < 2 * heads) {
            const int half = tid >= heads, h = h0 + tid - half * heads;
            float *sp = p.scale + ((size_t)half * p.pages + page) * p.Hk + h;
            const float old = *sp, need = least_scale(__uint_as_float(most[tid]));
            const bool fresh = src[0] >= 0 || !(old > 0.0f && old < INFINITY);
            const float now = fresh ? need : fmaxf(old, need);
            inv[tid] = inverse(now);
            ratio[tid] = fresh ? 1.0f : old * inverse(now);
            grown = ratio[tid] < 1.0f;
            if (now != old) *sp = now;
        }
        uint8_t *base = p.q8 + (((size_t)page * p.Hk + h0) << p.pshift) * D;
        const size_t half_q = (((size_t)p.pages * p.Hk) << p.pshift) * D;
        if (__syncthreads_or(grown)) {
            // the held rows of the blocks that grew, 16 bytes at a time
            for (int c = tid; c < 2 * heads * p.P * (D / 16); c += NT) {
                const int d16 = c % (D / 16), o = (c / (D / 16)) & (p.P - 1), hh = (c / (D / 16)) >> p.pshift;
                const float f = ratio[hh];
                if (src[o] >= 0 || f == 1.0f) continue;
                const int half = hh >= heads;
                u32x4 *at = reinterpret_cast<u32x4 *>(base + half * half_q + ((((size_t)(hh - half * heads)) << p.pshift) + o) * D) + d16;
                u32x4 w = *at;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x[4] = {__builtin_amdgcn_cvt_f32_fp8((int)w[e], 0), __builtin_amdgcn_cvt_f32_fp8((int)w[e], 1),
                                        __builtin_amdgcn_cvt_f32_fp8((int)w[e], 2), __builtin_amdgcn_cvt_f32_fp8((int)w[e], 3)};
                    w[e] = to_e4m3(x, f);
                }
                *at = w;
            }
        }
        for (int vec = gid; vec < vectors; vec += NG) {
            float x[8];
            int row, hh;
            load(vec, x, row, hh);
            const int half = hh >= heads;
            uint8_t *dst = base + half * half_q + ((((size_t)(hh - half * heads)) << p.pshift) + row) * D;
            *reinterpret_cast<uint32_t *>(dst + 4 * u) = to_e4m3(x, inv[hh]);
            *reinterpret_cast<uint32_t *>(dst + HALF + 4 * u) = to_e4m3(x + 4, inv[hh]);
        }
        __syncthreads();   // the page's lists are read
    }
}

template <typename T, bool FUSED, bool NORM>
int launch(Fp8WriteParams &p, int D, hipStream_t s) {
    // tokens of a work-group: one where there are few, a page's rows for prompts; KV heads: so many that a page's
    // rows keep its lane groups busy
    p.chunk = p.n <= 256 ? 1 : min(p.P, 64);
    p.hpg = max(1, min(min(p.Hk, MAX_HEADS), 256 / p.chunk));
    p.hgroups = (p.Hk + p.hpg - 1) / p.hpg;
    const long long pages = (long long)(p.n + p.chunk - 1) / p.chunk * p.hgroups;
    const int per = 256 / (D / 8);
    const long long queries = FUSED ? ((long long)p.n * p.nq + per - 1) / per : 0;
    if ((pages + queries) * 256 > MAX_THREADS) return TI_ERR_UNSUPPORTED;
    p.page_groups = (unsigned)pages;
    const unsigned grid = (unsigned)(pages + queries);
    if (D == 128) fp8_write_kernel<T, FUSED, NORM, 128><<<grid, 256, 0, s>>>(p);
    else fp8_write_kernel<T, FUSED, NORM, 64><<<grid, 256, 0, s>>>(p);
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
