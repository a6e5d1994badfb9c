// Attention with a sliding window and over 8-bit block caches: what the paged kernels share for them.
//
// The query at position p sees the keys in (p - size, p] and the keys below `sinks` (never past p). A work-group's rows
// see, taken together, the sinks and the keys from its first row's window on: it walks the tiles that hold these, a
// first few and then those from the window's on, and masks inside the tiles at the edges.
//
// 8-bit block caches: an e4m3 value times its block's power of two is a bf16 value exactly (v_cvt_scalef32_pk_bf16_fp8),
// so tiles are converted on their way to the matrix cores and everything behind is the dense kernels'.
//
// INT8 caches: the prefill kernels multiply fp16 keys (int8 values exactly) by queries that f16_row rounds once, to fp16's
// 11 bits, where a step without a window rounds them to bf16's 8: an output's error is then its own rounding's (1.7e-3 of its
// size, root of the mean square, against 3.3e-3).
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
    // The 32-key tile whose half x no row sees, or -1: with x = 1 the last one of sinks, with x = 0 the window's first. Such a
    // half's page may have been given back and be anyone's, so the other half's is read in its place (halves in pages of more
    // than 16 keys share a page anyhow).
    __device__ __forceinline__ int unseen(int x, int sinks) const {
        const int kt = x ? sunk - 1 : sunk + skip, pos = kt * 32 + 16 * x;
        return kt >= 0 && pos >= sinks && pos + 16 <= lo ? kt : -1;
    }
};

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f16x8_t as_f16x8(u32x4 w) { return __builtin_bit_cast(f16x8_t, w); }

// 8 int8 -> 8 fp16 (exact): the bits 0x6400 | (b + 128) are 1152 + b.
__device__ __forceinline__ u32x4 i8x8_to_f16x8(uint32_t x, uint32_t y) {
    const f16x2_t bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t bits = __builtin_amdgcn_perm(0x64646464u, (e < 2 ? x : y) ^ 0x80808080u, e & 1 ? 0x04030402u : 0x04010400u);
        r[e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, bits) - bias);
    }
    return r;
}

// A lane's N x 8 elements of a query row (bf16; word i holds elements at(i) on) times the keys' smoothing, as fp16 times the
// 2^e that brings the row's largest magnitude into [2^14, 2^15); largest: over the row's lanes. Returns 2^-e.
template <int N, typename At, typename Max>
__device__ __forceinline__ float f16_row(u32x4 (&q)[N], const float *smooth, At &&at, Max &&largest) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            most = fmaxf(most, fmaxf(fabsf(__uint_as_float(q[i][e] << 16) * smooth[at(i) + 2 * e]),
                                     fabsf(__uint_as_float(q[i][e] & 0xffff0000u) * smooth[at(i) + 2 * e + 1])));
    most = largest(most);
    const int e2 = most > 0.0f ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const f32x2 v = {__builtin_ldexpf(__uint_as_float(q[i][e] << 16) * smooth[at(i) + 2 * e], e2),
                             __builtin_ldexpf(__uint_as_float(q[i][e] & 0xffff0000u) * smooth[at(i) + 2 * e + 1], e2)};
            q[i][e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
        }
    return __builtin_ldexpf(1.0f, -e2);
}

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
