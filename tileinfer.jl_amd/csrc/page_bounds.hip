// Bounds of the keys of cache pages (page_select.hip keeps pages by them).
//
// A page's bounds for one KV head are the largest and the smallest element of its keys in each
// head dimension, as whole multiples of one power of two 2^e, rounded outward into int8:
//   e = least integer in [-126, 127] with |k| <= 127 2^e for every element k of the page's keys
//   hi_d = ceil(max k_d 2^-e), lo_d = floor(min k_d 2^-e)
// Multiplying by a power of two is exact and so are ceil and floor, so the bounds are a function of
// the keys alone, whatever the order they are read in, and no key lies outside them. They depend
// only on what the cache holds below the sequence's length: after a step is taken back (a rejected
// draft) and written again they come out as if it had never been.
#include "page_bounds.hpp"

using namespace ti;
using namespace ti_pages;

namespace {

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
    const Step st = step_of(p.qsl, p.positions, b, p.nmax, p.total);
    if (st.n <= 0) return;
    const int len = st.start + st.n, page = st.start / p.P + idx;
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
