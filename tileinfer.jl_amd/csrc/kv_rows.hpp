// What the kernels that write cache pages share: pool rows of slots, and vectors of elements as floats.
#pragma once

#include "common.hpp"

namespace ti {

// Pool row (0-based, in units of D elements) of (1-based slot, KV head h) in a
// [pages][H][P][D] pool: offset + P h + P H page (src/ops/reference.jl:61-70,
// src/ops/tile/elementwise.jl:122-128). Returns -1 for a slot outside the pool.
__device__ __forceinline__ long long slot_row(int32_t slot, int h, int P, int H, int pages) {
    long long s = (long long)slot - 1;
    if (s < 0 || s >= (long long)P * pages) return -1;
    const uint32_t s32 = (uint32_t)s, page = s32 / (uint32_t)P;   // 32-bit division: a slot is an int32
    return (long long)(s32 - page * (uint32_t)P) + (long long)P * h + (long long)P * H * page;
}

// Four consecutive elements of T as floats.
template <typename T> struct Vec4;
template <> struct Vec4<uint16_t> {
    static __device__ __forceinline__ void ld(const uint16_t *p, float (&x)[4]) {
        const uint2 w = *reinterpret_cast<const uint2 *>(p);
        x[0] = __uint_as_float(w.x << 16);
        x[1] = __uint_as_float(w.x & 0xffff0000u);
        x[2] = __uint_as_float(w.y << 16);
        x[3] = __uint_as_float(w.y & 0xffff0000u);
    }
    static __device__ __forceinline__ void st(uint16_t *p, const float (&x)[4]) {
        const uint2 w = make_uint2((uint32_t)f2bf(x[0]) | ((uint32_t)f2bf(x[1]) << 16),
                                   (uint32_t)f2bf(x[2]) | ((uint32_t)f2bf(x[3]) << 16));
        *reinterpret_cast<uint2 *>(p) = w;
    }
};
template <> struct Vec4<float> {
    static __device__ __forceinline__ void ld(const float *p, float (&x)[4]) {
        const float4 w = *reinterpret_cast<const float4 *>(p);
        x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
    }
    static __device__ __forceinline__ void st(float *p, const float (&x)[4]) {
        *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    }
};

// E consecutive elements of T, loaded, stored, or unpacked from 16 bytes.
template <typename T, int E> struct VecE;
template <> struct VecE<float, 4> : Vec4<float> {
    static __device__ __forceinline__ void unpack(uint4 w, float (&x)[4]) {
        x[0] = __uint_as_float(w.x);
        x[1] = __uint_as_float(w.y);
        x[2] = __uint_as_float(w.z);
        x[3] = __uint_as_float(w.w);
    }
};
template <> struct VecE<uint16_t, 4> : Vec4<uint16_t> {};
template <> struct VecE<uint16_t, 8> {
    static __device__ __forceinline__ void ld(const uint16_t *p, float (&x)[8]) {
        unpack(*reinterpret_cast<const uint4 *>(p), x);
    }
    static __device__ __forceinline__ void unpack(uint4 w, float (&x)[8]) {
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[2 * e] = __uint_as_float(ws[e] << 16);
            x[2 * e + 1] = __uint_as_float(ws[e] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void st(uint16_t *p, const float (&x)[8]) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                                   pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    }
};

}  // namespace ti
