// Bounds of the keys of cache pages, and the pages that a query keeps by them.
//
// A page's bounds for one KV head are the largest and the smallest element of its keys in each
// head dimension, as whole multiples of one power of two 2^e, rounded outward into int8:
//   e = least integer in [-126, 127] with |k| <= 127 2^e for every element k of the page's keys
//   hi_d = ceil(max k_d 2^-e), lo_d = floor(min k_d 2^-e)
// Multiplying by a power of two is exact and so are ceil and floor, so the bounds are a function of
// the keys alone, whatever the order they are read in, and no key lies outside them. They depend
// only on what the cache holds below the sequence's length: after a step is taken back (a rejected
// draft) and written again they come out as if it had never been.
#include "common.hpp"

using namespace ti;

namespace {

// The least e in [-126, 127] with a <= 127 2^e, for finite a >= 0: a = f 2^x with f in [0.5, 1), and
// f 2^7 <= 127 takes e = x - 7, else x - 6.
__device__ __forceinline__ int bound_exponent(float a) {
    const int x = __builtin_amdgcn_frexp_expf(a);
    const float f = __builtin_amdgcn_frexp_mantf(a);
    return a > 0.0f ? max(f <= 127.0f / 128.0f ? x - 7 : x - 6, -126) : -126;
}
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

struct BoundsParams {
    const void *kp;
    const int8_t *lq;
    const float *ls, *smooth;
    int8_t *bounds;
    float *scale;
    const int32_t *positions, *qsl, *bt;
    int bt_stride, num_pages, P, Hk, nmax, total;
};

// One wave per (touched page, KV head): LPK = D / E lanes of E elements (16 bytes) hold one key, so
// the wave takes KPW = 64 / LPK keys per load; the running maxima and minima of a lane's dimensions
// are joined across the key groups by xor shuffles. Bound by the read of the pages' keys (values
// are not read); a step of one token per sequence by the latency of its dependent loads (query
// offset, position, page id, keys).
template <typename T, bool INT8, int D>
__global__ void __launch_bounds__(256) key_bounds_kernel(BoundsParams p) {
    constexpr int E = INT8 ? 16 : 16 / (int)sizeof(T);
    constexpr int LPK = D / E, KPW = 64 / LPK;
    const int lane = threadIdx.x & 63;
    const int unit = (int)(blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
    const int idx = unit / p.Hk, h = unit - idx * p.Hk, b = blockIdx.y;
    const int tok0 = p.qsl ? p.qsl[b] : b * p.nmax;
    int nb = p.qsl ? min(p.qsl[b + 1] - tok0, p.nmax) : p.nmax;
    if (tok0 < 0 || tok0 >= p.total || nb <= 0) return;
    nb = min(nb, p.total - tok0);
    const int start = min(max(p.positions[tok0], 0), 0x7fffffff - nb), len = start + nb;
    const int page = start / p.P + idx;
    if (page > (len - 1) / p.P || page >= p.bt_stride) return;
    const int id = p.bt[(size_t)b * p.bt_stride + page] - 1;
    if (id < 0 || id >= p.num_pages) return;   // no such page: nothing is written
    const int held = min(p.P, len - page * p.P);
    const size_t row0 = ((size_t)id * p.Hk + h) * p.P;
    const int kk = lane / LPK, c = (lane % LPK) * E;
    float hi[E], lo[E];
#pragma unroll
    for (int i = 0; i < E; i++) hi[i] = -INFINITY, lo[i] = INFINITY;
    bool fine = true;
    float sm[E];
    if constexpr (INT8) {
#pragma unroll
        for (int i = 0; i < E; i++) sm[i] = p.smooth[c + i];
    }
    // Keys past the last one held re-read it (the join does not change).
    auto take = [&](u32x4 w, float sk) {
        float x[E];
        if constexpr (INT8) {
#pragma unroll
            for (int i = 0; i < E; i++) x[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * sk * sm[i];
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = __uint_as_float(w[i]);
        }
#pragma unroll
        for (int i = 0; i < E; i++) {
            fine &= fabsf(x[i]) < INFINITY;
            hi[i] = fmaxf(hi[i], x[i]);
            lo[i] = fminf(lo[i], x[i]);
        }
    };
    constexpr int U = 4;   // loads in flight per lane
    for (int k0 = 0; k0 < held; k0 += U * KPW) {
        u32x4 w[U];
        float sk[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t row = row0 + min(k0 + u * KPW + kk, held - 1);
            sk[u] = 1.0f;
            if constexpr (INT8) {
                w[u] = *reinterpret_cast<const u32x4 *>(p.lq + row * D + c);
                sk[u] = p.ls[row];
            } else {
                w[u] = *reinterpret_cast<const u32x4 *>((const T *)p.kp + row * D + c);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) take(w[u], sk[u]);
    }
#pragma unroll
    for (int o = LPK; o < 64; o <<= 1)
#pragma unroll
        for (int i = 0; i < E; i++) {
            hi[i] = fmaxf(hi[i], __shfl_xor(hi[i], o));
            lo[i] = fminf(lo[i], __shfl_xor(lo[i], o));
        }
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < E; i++) a = fmaxf(a, fmaxf(fabsf(hi[i]), fabsf(lo[i])));
    a = wave_max(a);
    fine = __all(fine);
    const int e = bound_exponent(fine ? a : 0.0f);
    const float back = power(-e);
    // Lanes of the first key group write hi, those of the second lo (KPW >= 2).
    if (kk < 2) {
        uint32_t w[E / 4];
#pragma unroll
        for (int i = 0; i < E / 4; i++) {
            w[i] = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float x = kk == 0 ? ceilf(hi[4 * i + j] * back) : floorf(lo[4 * i + j] * back);
                const int v = fine ? (int)x : (kk == 0 ? 127 : -127);
                w[i] |= ((uint32_t)v & 255u) << (8 * j);
            }
        }
        uint32_t *dst = reinterpret_cast<uint32_t *>(p.bounds + (((size_t)id * p.Hk + h) * 2 + kk) * D + c);
#pragma unroll
        for (int i = 0; i < E / 4; i++) dst[i] = w[i];
    }
    if (lane == 0) p.scale[(size_t)id * p.Hk + h] = fine ? power(e) : INFINITY;
}

// ---- selection -------------------------------------------------------------------------------
//
// A query row q (one token, one query head) as whole numbers w_d = rint(q_d 2^-e), e as above over
// the row, has with any key inside a page's bounds at most the product
//   2^e 2^e_page sum_d max(w_d hi_d, w_d lo_d) = 2^e 2^e_page (relu(w) . hi + min(w, 0) . lo)
// (of the whole numbers w): one int8 matrix product of depth 2 D, whose sums stay below 2^22 and
// are exact. The score of a page for a token and KV head is the largest over the G query heads, two
// multiplications by powers of two: exact, so equal scores are equal pages' bounds and not
// roundings, and the kept pages do not depend on how the work is split.

struct SelectParams {
    const void *q;
    const int8_t *bounds;
    const float *scale;
    const int32_t *positions, *qsl, *bt;
    int32_t *tables, *lengths;
    uint32_t *keys;   // workspace: order-preserving scores [total][Hk][pitch]
    int bt_stride, num_pages, P, Hk, Hq, G, nmax, total, keep, sinks, window, causal;
    int gp, tp, rblocks;   // rows of a token in a 16-row tile (power of two >= G, at most 16), tokens per tile, 16-row blocks per token
    int pitch, split;      // keys per (token, KV head); work-groups that share a token tile's pages
};

typedef int i32x4 __attribute__((ext_vector_type(4)));

// A sequence's step as the kernels of this file read it; n <= 0: none.
struct Step {
    int tok0, n, start;
};
__device__ __forceinline__ Step step_of(const int32_t *qsl, const int32_t *positions, int b, int nmax, int total) {
    Step s{};
    s.tok0 = qsl ? qsl[b] : b * nmax;
    s.n = qsl ? min(qsl[b + 1] - s.tok0, nmax) : nmax;
    if (s.tok0 < 0 || s.tok0 >= total) s.n = 0;
    s.n = min(s.n, total - s.tok0);
    s.start = s.n > 0 ? min(max(positions[s.tok0], 0), 0x7fffffff - s.n) : 0;
    return s;
}

// Larger score, larger key; NaN (an infinite page scale times 0) counts as the largest.
__device__ __forceinline__ uint32_t order_key(float x) {
    x += 0.0f;   // -0 and 0 are one score
    const uint32_t u = __float_as_uint(x);
    if (x != x) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Scores: grid (Hk x split, token tiles, B), four waves that take the sequence's 16-page tiles in
// turn. S = bounds W on v_mfma_i32_16x16x64_i8 (A: 16 pages, lane l holds page l % 16's bytes
// 16 (l / 16) .. + 16 of each 64; B: 16 query rows, the same way), so lane l gets query row l % 16's
// products with pages 4 (l / 16) .. + 3; the heads of a token are neighbouring lanes.
template <typename T, int D>
__device__ __forceinline__ void score_tile(const SelectParams &p, const Step &st, int b, int h, int part, int w, int lane, int t0) {
    constexpr int NK = D / 64;
    const int r16 = lane & 15, kg = lane >> 4;
    const int tl = min(t0 + p.tp, st.n) - 1;   // the tile's last token
    const int seen = min((st.start + (p.causal ? tl : st.n - 1)) / p.P + 1, p.bt_stride);
    const int ntiles = (seen + 15) >> 4, step = 4 * p.split;
    const int32_t *bt = p.bt + (size_t)b * p.bt_stride;
    const int t = t0 + r16 / p.gp;
    for (int rb = 0; rb < p.rblocks; rb++) {
        const int g = rb * 16 + r16 % p.gp;
        const bool ok = t < st.n && g < p.G;
        float x[NK][16];
        float a = 0.0f;
        const T *qr = (const T *)p.q + ((size_t)(st.tok0 + (ok ? t : t0)) * p.Hq + h * p.G + (ok ? g : 0)) * D;
#pragma unroll
        for (int i = 0; i < NK; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) {
                x[i][j] = Elt<T>::ld(qr, i * 64 + kg * 16 + j);
                a = x[i][j] != x[i][j] ? INFINITY : fmaxf(a, fabsf(x[i][j]));
            }
        a = fmaxf(a, __shfl_xor(a, 16));
        a = fmaxf(a, __shfl_xor(a, 32));
        const bool fine = a < INFINITY;   // a row that is not finite scores 0
        const int e = bound_exponent(fine ? a : 0.0f);
        const float back = power(-e), forth = power(e);
        u32x4 up[NK], dn[NK];
#pragma unroll
        for (int i = 0; i < NK; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t u = 0, d = 0;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int v = fine ? (int)rintf(x[i][4 * j + k] * back) : 0;
                    u |= (uint32_t)max(v, 0) << (8 * k);
                    d |= ((uint32_t)min(v, 0) & 255u) << (8 * k);
                }
                up[i][j] = u;
                dn[i][j] = d;
            }
        for (int j = part * 4 + w; j < ntiles; j += step) {
            const int pg = j * 16 + r16;
            const int id = page_of(bt, min(pg, seen - 1), p.bt_stride, p.num_pages);
            const size_t at = (size_t)id * p.Hk + h;
            const int8_t *bp = p.bounds + at * 2 * D + kg * 16;
            i32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < NK; i++) {
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const i32x4 *>(bp + i * 64),
                                                            __builtin_bit_cast(i32x4, up[i]), acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const i32x4 *>(bp + D + i * 64),
                                                            __builtin_bit_cast(i32x4, dn[i]), acc, 0, 0, 0);
            }
            const float ps = p.scale[at];
            uint32_t key[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float s = ok ? (float)acc[k] * forth : -INFINITY;
                for (int o = 1; o < p.gp; o <<= 1) s = fmaxf(s, __shfl_xor(s, o));
                key[k] = order_key(s * __shfl(ps, 4 * kg + k));
            }
            if (r16 % p.gp == 0 && t < st.n) {
                uint32_t *dst = p.keys + ((size_t)(st.tok0 + t) * p.Hk + h) * p.pitch + j * 16 + 4 * kg;
                u32x4 v = {key[0], key[1], key[2], key[3]};
                if (rb > 0) {   // heads past the sixteenth of a token: the same wave wrote the others
                    const u32x4 o = *reinterpret_cast<const u32x4 *>(dst);
#pragma unroll
                    for (int k = 0; k < 4; k++) v[k] = max(v[k], o[k]);
                }
                *reinterpret_cast<u32x4 *>(dst) = v;
            }
        }
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(256) page_scores_kernel(SelectParams p) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % p.Hk, part = blockIdx.x / p.Hk, b = blockIdx.z;
    const Step st = step_of(p.qsl, p.positions, b, p.nmax, p.total);
    for (int t0 = blockIdx.y * p.tp; t0 < st.n; t0 += gridDim.y * p.tp) score_tile<T, D>(p, st, b, h, part, w, lane, t0);
}

// Kept pages of one (token, KV head): grid (Hk, max_query_len, B), 256 threads. The key of the last
// page kept by score is found by four rounds over its bytes (a histogram of the keys that agree
// in the bytes above, from the workspace), then one pass over the pages in order writes those that
// are forced, above the key, or equal to it while there is room.
__global__ void __launch_bounds__(256) keep_pages_kernel(SelectParams p) {
    __shared__ int hist[256], wsum[2][4];
    __shared__ int pick, left;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int h = blockIdx.x, b = blockIdx.z;
    const Step st = step_of(p.qsl, p.positions, b, p.nmax, p.total);
    for (int t = blockIdx.y; t < st.n; t += gridDim.y) {
    const int last = st.start + (p.causal ? t : st.n - 1);
    const int seen = min(last / p.P + 1, p.bt_stride);
    const size_t pair = (size_t)(st.tok0 + t) * p.Hk + h;
    const uint32_t *keys = p.keys + pair * p.pitch;
    int32_t *out = p.tables + pair * p.keep;
    const int32_t *bt = p.bt + (size_t)b * p.bt_stride;
    const int kept = min(seen, p.keep);
    // candidates by score: pages [c0, c1); the others are forced
    const int c0 = min(p.sinks, seen), c1 = max(c0, seen - p.window);
    const int need = kept - (seen - (c1 - c0));   // pages to keep by score
    uint32_t limit = 0;    // keys above it are kept, and `ties` of those equal to it
    int ties = 0;
    if (need < c1 - c0) {
        ties = need;
        for (int shift = 24; shift >= 0 && ties > 0; shift -= 8) {
            hist[tid] = 0;
            __syncthreads();
            for (int i = c0 + tid; i < c1; i += 256) {
                const uint32_t k = keys[i];
                if (shift == 24 || ((k ^ limit) >> (shift + 8)) == 0) atomicAdd(&hist[(k >> shift) & 255], 1);
            }
            __syncthreads();
            // the byte whose count, with those of the bytes above, first reaches `ties`
            int c = hist[255 - tid], s = c;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(s, o);
                if (lane >= o) s += v;
            }
            if (lane == 63) wsum[0][w] = s;
            __syncthreads();
            for (int i = 0; i < w; i++) s += wsum[0][i];
            if (s >= ties && s - c < ties) {
                pick = 255 - tid;
                left = ties - (s - c);
            }
            __syncthreads();
            limit |= (uint32_t)pick << shift;
            ties = left;
            __syncthreads();
        }
        if (need == 0) limit = 0xffffffffu;   // none by score
    } else {
        ties = c1 - c0;   // every candidate: all are above 0 or equal to it
    }
    int base = 0, eq = 0;
    for (int i0 = 0; i0 < seen; i0 += 256) {
        const int i = i0 + tid;
        const bool in = i < seen, cand = i >= c0 && i < c1;
        const uint32_t k = in && cand ? keys[i] : 0;
        const bool sure = in && (!cand || k > limit), even = in && cand && k == limit;
        const unsigned long long ms = __ballot(sure), me = __ballot(even);
        const unsigned long long below = (1ull << lane) - 1;
        __syncthreads();
        if (lane == 0) {
            wsum[0][w] = __popcll(ms);
            wsum[1][w] = __popcll(me);
        }
        __syncthreads();
        int s = __popcll(ms & below), q = eq + __popcll(me & below), stot = 0, etot = 0;
        for (int j = 0; j < 4; j++) {
            if (j < w) s += wsum[0][j], q += wsum[1][j];
            stot += wsum[0][j];
            etot += wsum[1][j];
        }
        // pages written before this one: the sure ones, and the equal ones while there was room
        const int at = base + s + min(q, ties);
        if ((sure || (even && q < ties)) && at < kept) out[at] = bt[i];
        base += stot;
        eq += etot;
    }
    for (int i = kept + tid; i < p.keep; i += 256) out[i] = 0;
    if (tid == 0) {
        const long long l = (long long)(kept - 1) * p.P + min(last + 1 - (seen - 1) * p.P, p.P);
        p.lengths[pair] = (int)l;
    }
    }
}

}  // namespace

int ti_launch_key_bounds(int dtype, const ti_kv_cache *c, const ti_key_bounds *kb, const int32_t *bt, int bt_stride,
                         const int32_t *positions, const int32_t *qsl, int num_seqs, int nmax, int total, hipStream_t s) {
    BoundsParams p{};
    p.kp = c->k_pages;
    p.lq = c->layer_q;
    p.ls = c->layer_scale;
    p.smooth = c->smooth;
    p.bounds = kb->bounds;
    p.scale = kb->scale;
    p.positions = positions;
    p.qsl = qsl;
    p.bt = bt;
    p.bt_stride = bt_stride;
    p.num_pages = c->num_pages;
    p.P = c->page_size;
    p.Hk = c->kv_heads;
    p.nmax = nmax;
    p.total = total;
    const long long pages = min(((long long)nmax + c->page_size - 2) / c->page_size + 1, (long long)bt_stride);
    const long long groups = (pages * c->kv_heads + 3) / 4;
    if (pages * c->kv_heads > 0x7fffff00LL) return TI_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)groups, num_seqs);
    const bool wide = c->head_dim == 128;
    if (c->kind == TI_KV_INT8) {
        if (wide) key_bounds_kernel<float, true, 128><<<grid, 256, 0, s>>>(p);
        else key_bounds_kernel<float, true, 64><<<grid, 256, 0, s>>>(p);
    } else if (dtype == TI_F32) {
        if (wide) key_bounds_kernel<float, false, 128><<<grid, 256, 0, s>>>(p);
        else key_bounds_kernel<float, false, 64><<<grid, 256, 0, s>>>(p);
    } else {
        if (wide) key_bounds_kernel<uint16_t, false, 128><<<grid, 256, 0, s>>>(p);
        else key_bounds_kernel<uint16_t, false, 64><<<grid, 256, 0, s>>>(p);
    }
    return hipGetLastError() == hipSuccess ? TI_OK : TI_ERR_LAUNCH;
}

size_t ti_select_bytes(const ti_select_args *a) {
    const size_t pitch = ((size_t)a->block_table_stride + 15) / 16 * 16;
    return (size_t)a->total_tokens * a->kv_heads * pitch * sizeof(uint32_t);
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
    p.gp = 1;
    while (p.gp < p.G && p.gp < 16) p.gp <<= 1;
    p.tp = 16 / p.gp;
    p.rblocks = (p.G + 15) / 16;
    p.pitch = (a->block_table_stride + 15) / 16 * 16;
    const int ttiles = (a->max_query_len + p.tp - 1) / p.tp;
    // fewer token tiles than the chip has room for share each tile's pages out
    const long long groups = (long long)ttiles * a->num_seqs * a->kv_heads;
    p.split = 1;
    while (groups * p.split < 512 && p.split * 4 * 16 < a->block_table_stride) p.split <<= 1;
    const dim3 grid(a->kv_heads * p.split, min(ttiles, 32768), a->num_seqs);   // longer steps loop
    if (a->head_dim == 128) {
        if (a->dtype == TI_F32) page_scores_kernel<float, 128><<<grid, 256, 0, s>>>(p);
        else page_scores_kernel<uint16_t, 128><<<grid, 256, 0, s>>>(p);
    } else {
        if (a->dtype == TI_F32) page_scores_kernel<float, 64><<<grid, 256, 0, s>>>(p);
        else page_scores_kernel<uint16_t, 64><<<grid, 256, 0, s>>>(p);
    }
    if (hipGetLastError() != hipSuccess) return TI_ERR_LAUNCH;
    keep_pages_kernel<<<dim3(a->kv_heads, min(a->max_query_len, 32768), a->num_seqs), 256, 0, s>>>(p);
    return hipGetLastError() == hipSuccess ? TI_OK : TI_ERR_LAUNCH;
}
