// Bounds of the keys of cache pages (page_select.hip keeps pages by them).
//
// A page's bounds for one KV head are the largest and the smallest element of its keys in each
// head dimension, as whole multiples of one power of two 2^e, rounded outward into int8:
//   e = least integer in [-126, 127] with |k| <= 127 2^e for every element k of the page's keys
//   hi_d = ceil(max k_d 2^-e), lo_d = floor(min k_d 2^-e)
// Multiplying by a power of two is exact and so are ceil and floor, so the bounds are a function of
// the keys alone, whatever the order they are read in, and no key lies outside them. Divided by powers of two of their
// dimensions first (`channel`, where a few would decide e for all), they stay exact. They depend
// only on what the cache holds below the sequence's length: after a step is taken back (a rejected
// draft) and written again they come out as if it had never been.
#include <type_traits>

#include "page_bounds.hpp"

using namespace ti;
using namespace ti_pages;

namespace {

struct BoundsParams {
    const void *kp;
    const int8_t *lq;
    const float *ls, *smooth, *channel;
    int8_t *bounds;
    float *scale;
    const int32_t *positions, *qsl, *bt;
    int bt_stride, num_pages, P, Hk, nmax, total;
};

// v_permlane32_swap / v_permlane16_swap: the upper half (odd rows of 16 lanes) of a changes places with the
// lower half (even rows) of b. The larger of both then is, in a lane of the lower half (an even row), that
// of a's two lanes 32 (16) apart; in the others that of b's: two values joined across lanes and one left to
// hold, without LDS.
__device__ __forceinline__ float join32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float join16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int CTRL> __device__ __forceinline__ float dpp_max(float x) {
    return fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, false)));
}

// One wave per (touched page, KV head): LPK = D / E lanes of E elements (16 bytes) hold one key, so the
// wave takes KPW = 64 / LPK keys per load and keeps the largest k_d and -k_d of its lanes' keys. The key
// groups' values are joined by lane swaps, each of which halves what a lane still holds, so that in the end
// the lower half of the wave has the largest elements and the upper the negated smallest, E / 2 of them
// per lane (with LDS shuffles the joins bound the kernel: 8 prompts of 4000 tokens 11.2 us). An INT8 key
// is max |q s| first and smoothed once at the end: rounding is monotonic, so that is the same number
// (q s as one fma of the byte + 128).
// Bound by the read of the pages' keys; a step of one token per sequence by the latency of its dependent
// loads (query offset, position, page id, keys).
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
    float up[E], dn[E];   // the largest k_d and -k_d
#pragma unroll
    for (int i = 0; i < E; i++) up[i] = dn[i] = -INFINITY;
    float odd = 0.0f;     // NaN once an element (INT8: a scale) is not finite
    // Keys past the last one held re-read it (the join does not change). `count` loads in flight per lane:
    // a page of 64 keys of 16 bits or less in one round trip, pages of 16 keys without loads past them.
    auto pass = [&](int k0, auto count) {
        constexpr int U = decltype(count)::value;
        u32x4 w[U];
        float sk[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t row = row0 + min(k0 + u * KPW + kk, held - 1);
            if constexpr (INT8) {
                w[u] = *reinterpret_cast<const u32x4 *>(p.lq + row * D + c);
                sk[u] = p.ls[row];
            } else {
                w[u] = *reinterpret_cast<const u32x4 *>((const T *)p.kp + row * D + c);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            float x[E];
            if constexpr (INT8) {
                odd = __builtin_fmaf(sk[u], 0.0f, odd);
#pragma unroll
                for (int i = 0; i < E; i++) {
                    const uint32_t v = w[u][i >> 2] ^ 0x80808080u;
                    x[i] = __builtin_fmaf((float)((v >> (8 * (i & 3))) & 255u), sk[u], -128.0f * sk[u]);
                }
            } else if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[2 * i] = __uint_as_float(w[u][i] << 16);
                    x[2 * i + 1] = __uint_as_float(w[u][i] & 0xffff0000u);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = __uint_as_float(w[u][i]);
            }
#pragma unroll
            for (int i = 0; i < E; i++) {
                if constexpr (!INT8) odd = __builtin_fmaf(x[i], 0.0f, odd);
                up[i] = fmaxf(up[i], x[i]);
                dn[i] = fmaxf(dn[i], -x[i]);
            }
        }
    };
    constexpr int MANY = INT8 ? 8 : 16;
    int k0 = 0;
    for (; held - k0 > 4 * KPW; k0 += MANY * KPW) pass(k0, std::integral_constant<int, MANY>{});
    for (; k0 < held; k0 += 4 * KPW) pass(k0, std::integral_constant<int, 4>{});
    if constexpr (INT8) {
#pragma unroll
        for (int i = 0; i < E; i++) {
            const float s = p.smooth[c + i], a = up[i] * s, b = dn[i] * s;   // s < 0: -k is the larger
            up[i] = s < 0.0f ? -b : a;
            dn[i] = s < 0.0f ? -a : b;
            odd = __builtin_fmaf(a, 0.0f, __builtin_fmaf(b, 0.0f, odd));
        }
    }
    if (p.channel) {   // positive powers of two: the largest key divided is the largest of the divided ones
#pragma unroll
        for (int i = 0; i < E; i++) {
            const float s = 1.0f / p.channel[h * D + c + i];
            up[i] *= s;
            dn[i] *= s;
            odd = __builtin_fmaf(up[i], 0.0f, __builtin_fmaf(dn[i], 0.0f, odd));
        }
    }
    // lanes 0 - 31: up, 32 - 63: dn
    constexpr int N = LPK <= 16 ? E / 2 : E;   // elements a lane is left with
    float v[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        v[i] = join32(up[i], dn[i]);
        if constexpr (LPK <= 16) v[i] = join16(v[i], join32(up[i + N], dn[i + N]));   // odd rows: elements from N on
        if constexpr (LPK <= 8) v[i] = dpp_max<0x128>(v[i]);                          // row_ror 8
        if constexpr (LPK <= 4) v[i] = fmaxf(v[i], __shfl_xor(v[i], 4));
    }
    const bool fine = __all(odd == 0.0f);
    float a = v[0];   // the largest |k_d|: one of k_d and -k_d
#pragma unroll
    for (int i = 1; i < N; i++) a = fmaxf(a, v[i]);
    a = dpp_max<0x140>(dpp_max<0x141>(dpp_max<0x4e>(dpp_max<0xb1>(a))));   // over 16 lanes
    a = join16(a, a);
    a = join32(a, a);
    const int e = bound_exponent(fine ? a : 0.0f);
    const float back = power(-e);
    const bool low = lane >= 32;
    const int d = c + (LPK <= 16 && (lane & 16) ? N : 0);
    if (LPK > 8 || (lane & 15) < LPK) {
        // ceil(hi) and -ceil(-lo) = floor(lo)
        uint32_t w[(N + 3) / 4] = {};
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int x = fine ? (int)ceilf(v[i] * back) : 127;
            w[i >> 2] |= ((uint32_t)(low ? -x : x) & 255u) << (8 * (i & 3));
        }
        int8_t *dst = p.bounds + (((size_t)id * p.Hk + h) * 2 + low) * D + d;
        if constexpr (N == 2) {
            *reinterpret_cast<uint16_t *>(dst) = (uint16_t)w[0];
        } else {
#pragma unroll
            for (int i = 0; i < N / 4; i++) reinterpret_cast<uint32_t *>(dst)[i] = w[i];
        }
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
    p.channel = kb->channel;
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
    if (groups * 256 > MAX_THREADS) return TI_ERR_UNSUPPORTED;
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
