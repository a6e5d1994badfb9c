// Whole-number forms of keys and queries, shared by page_bounds.hip and page_select.hip.
#pragma once

#include "common.hpp"

namespace ti_pages {

// The least e in [-126, 127] with a <= 127 2^e, for finite a >= 0: a = f 2^x with f in [0.5, 1), and
// f 2^7 <= 127 takes e = x - 7, else x - 6.
__device__ __forceinline__ int bound_exponent(float a) {
    const int x = __builtin_amdgcn_frexp_expf(a);
    const float f = __builtin_amdgcn_frexp_mantf(a);
    return a > 0.0f ? max(f <= 127.0f / 128.0f ? x - 7 : x - 6, -126) : -126;
}
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// A sequence's step; n <= 0: it has no tokens.
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

}  // namespace ti_pages
