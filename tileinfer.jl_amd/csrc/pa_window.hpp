// Attention with a sliding window and over 8-bit block caches: what the paged kernels share for them.
//
// The query at position p sees the keys in (p - size, p] and the keys below `sinks` (never past p). A work-group's rows
// see, taken together, the sinks and the keys from its first row's window on: it walks the tiles that hold these, a
// first few and then those from the window's on, and masks inside the tiles at the edges.
//
// 8-bit block caches: an e4m3 value times its block's power of two is a bf16 value exactly (v_cvt_scalef32_pk_bf16_fp8),
// so tiles are converted on their way to the matrix cores and everything behind is the dense kernels'.
//
// Masked keys. The matrix products give a masked key the weight 0, and 0 times a value that is not finite is NaN, so
// a NaN in a row of the cache would reach every row that is worked on together with one that sees it. The kernels look at
// what they are about to write: where it is not finite, the work-group's rows are done again one by one over the keys that
// each of them sees (exact_row).
#pragma once

#include <type_traits>

#include "common.hpp"

namespace ti {

// The position of a sequence's first query: a negative one reads as 0, one past all that its block-table row can hold as
// that, so that no count of keys leaves 32 bits and no loop runs on for what no table names.
__device__ __forceinline__ int first_position(int position, int bt_stride, int P) {
    return (int)min((long long)max(position, 0), min((long long)bt_stride * P, 1LL << 30));
}

// Tiles of 2^SHIFT keys that the rows from position `first` on see: `sunk` of them from the cache's start, the others
// `skip` further on.
struct WindowTiles {
    int lo, sunk, skip;
    template <int SHIFT>
    static __device__ __forceinline__ WindowTiles of(int first, int size, int sinks) {
        WindowTiles t;
        t.lo = max(first - size + 1, 0);
        const int from = t.lo >> SHIFT;
        t.sunk = min((min(t.lo, sinks) + (1 << SHIFT) - 1) >> SHIFT, from);
        t.skip = from - t.sunk;
        return t;
    }
    __device__ __forceinline__ int tile(int j) const { return j < sunk ? j : j + skip; }
};

// Whether the query at position `at` sees `key`. Without short circuits: hipcc has made of branches around the choice between
// a matrix product's register and a constant a move of the constant for every lane (attn_f32_kernel's masks, ROCm 7.2).
__device__ __forceinline__ bool window_sees(int key, int at, int size, int sinks) {
    return (key <= at) & ((key > at - size) | (key < sinks));
}

// 8 e4m3 values (two words) times a power of two in bf16.
__device__ __forceinline__ u32x4 e4m3x8_to_bf16(uint32_t x, uint32_t y, float scale) {
    return (u32x4){__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, scale, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, scale, true))};
}

// A wave-uniform float as a scalar load.
__device__ __forceinline__ float sloadf(const float *a, long long idx) {
    const uint64_t at = reinterpret_cast<uint64_t>(a + idx);
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at);
    const uint64_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
    return *(const __attribute__((address_space(4))) float *)((hi << 32) | lo);
}

// One query row over keys v0 .. v1 - 1 of a list on the vector ALUs, by one wave: key_at gives a list entry's key, or
// -1 where the row does not see it; no other key is touched. q: the row, in the activations' type T. Running maximum m (of
// scores in log2 units), sum l, and elements lane + 64 k of the weighted sum. Products as in generic_attention_kernel.
template <int D, bool INT8, bool FP8, typename Params, typename T, typename KeyAt>
__device__ __forceinline__ void exact_row(const Params &p, const int32_t *bt, int h, const T *q, int v0, int v1, KeyAt &&key_at, float &m,
                                          float &l, float (&acc)[D / 64]) {
    using E = Elt<T>;
    const int lane = threadIdx.x & 63;
    const size_t half_q = (size_t)p.num_pages * p.Hk * p.P * D, half_s = (size_t)p.num_pages * p.Hk * p.P;
    m = NEG_BIG;
    l = 0.0f;
#pragma unroll
    for (int k = 0; k < D / 64; k++) acc[k] = 0.0f;
#pragma unroll 1
    for (int c = v0; c < v1; c += 64) {
        const int key = c + lane < v1 ? key_at(c + lane) : -1;
        long long row = 0;
        float s = -INFINITY;
        if (key >= 0) {
            const int i = p.pshift >= 0 ? key >> p.pshift : key / p.P;
            row = ((long long)page_of(bt, i, p.bt_stride, p.num_pages) * p.Hk + h) * p.P + (key - i * p.P);
            float dot = 0.0f;
#pragma unroll 1
            for (int d = 0; d < D; d++) {
                float x;
                if constexpr (FP8) x = __builtin_amdgcn_cvt_f32_fp8((int)(uint8_t)p.lq[row * D + d], 0);
                else if constexpr (INT8) x = (float)p.lq[row * D + d] * p.smooth[d];
                else x = E::ld(p.kp, row * D + d);
                dot += E::ld(q, d) * x;
            }
            if constexpr (FP8) dot *= p.ls[row / p.P];
            if constexpr (INT8) dot *= p.ls[row];
            s = dot * p.scale_log2;
        }
        const float mn = fmaxf(m, wave_max(s));
        const float alpha = fast_exp2(m - mn), pr = key >= 0 ? fast_exp2(s - mn) : 0.0f;
        m = mn;
        l = l * alpha + wave_sum(pr);
#pragma unroll
        for (int k = 0; k < D / 64; k++) acc[k] *= alpha;
#pragma unroll 1
        for (int i = 0; i < 64; i++) {
            if (__shfl(key, i) < 0) continue;
            const float pi = __shfl(pr, i);
            const long long ri = __shfl(row, i);
#pragma unroll
            for (int k = 0; k < D / 64; k++) {
                const int d = lane + 64 * k;
                float x;
                if constexpr (FP8) x = __builtin_amdgcn_cvt_f32_fp8((int)(uint8_t)p.lq[half_q + ri * D + d], 0) * p.ls[(half_s + ri) / p.P];
                else if constexpr (INT8) x = (float)p.lq[half_q + ri * D + d] * p.ls[half_s + ri];
                else x = E::ld(p.vp, ri * D + d);
                acc[k] += pi * x;
            }
        }
    }
}

}  // namespace ti
