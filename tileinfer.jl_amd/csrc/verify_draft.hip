// Verification of drafted tokens (speculative sampling): sequence b's drafts x_0 .. x_{n-1} are
// accepted in order while
//   u_i q_i(x_i) < p_i(x_i)
// (p the target's probabilities, q the drafter's, 1 where it gives none), a of them; then one more
// token is drawn from the weights
//   w = max(p_a - q_a, 0)      a draft was rejected
//   w = p_a without x_a        a draft was rejected, the drafter gives no probabilities
//   w = p_a                    every draft was accepted
// as the lowest v with w_v > 0 and C(v) > u_N C(V - 1), C the running sum of w. The output then is
// distributed as p for any q.
//
// The test is exact: a product of two floats is one double. The running sums are in double as well:
// the drawn token sits between two of them, and in 32 bits the sum over a large vocabulary is off by
// more than many of its entries. An entry that is not positive and finite has no weight. Weights that
// are all zero (probabilities that contradict each other) fall back to p_a, and a row p_a without
// any weight draws nothing (-1).
//
// Work. All that is read is one value of p and q per draft and then row a of both (V entries).
// sum_kernel: a wave sums pieces of PIECE entries of a sequence's row (PER per lane, 16-byte loads),
// after finding a for itself (the drafts of a sequence one per lane, their loads together); one wave per
// piece, and `rep` pieces per wave where there are more pieces than the chip holds waves. draw_kernel:
// one work-group per sequence takes the piece in which the running sum passes the goal, and scans that
// one piece. Every sum has one fixed order. The sum kernel is bound by the read of the two rows, or where
// that is short by its chain of dependent loads (drafts, their probabilities, the row).
#include "common.hpp"

using namespace ti;

namespace {

constexpr int PIECE = 1024;         // entries summed together: one wave, PER entries per lane
constexpr int PER = PIECE / 64;

struct VerifyParams {
    const void *target, *draft;
    const int32_t *drafted, *counts;
    const float *uniforms;
    int32_t *accepted, *tokens;
    double *sums;   // [B][pieces][2]: the weights' sum and p_a's
    int N, V, pieces, rep;
};

// Accepted drafts of sequence b; every lane gets the count. *count: the sequence's drafts.
template <typename T>
__device__ __forceinline__ int accepted_of(const VerifyParams &p, int b, int lane, int *count) {
    int n = p.N;
    if (p.counts) n = p.counts[b];
    for (int i0 = 0;; i0 += 64) {
        const int i = min(i0 + lane, p.N - 1);   // loads before the count is known stay inside the row
        int x = -1;
        float u = 0.0f;
        if (p.N > 0) {
            x = p.drafted[(size_t)b * p.N + i];
            u = p.uniforms[(size_t)b * (p.N + 1) + i];
        }
        n = min(max(n, 0), p.N);
        *count = n;
        bool ok = false;
        if (i0 + lane < n && x >= 0 && x < p.V) {   // a token that does not exist is not accepted
            const float pv = Elt<T>::ld((const T *)p.target, ((size_t)b * (p.N + 1) + i) * p.V + x);
            const float qv = p.draft ? Elt<T>::ld((const T *)p.draft, ((size_t)b * p.N + i) * p.V + x) : 1.0f;
            ok = (double)u * (double)qv < (double)pv;
        }
        const unsigned long long no = __ballot(!ok);   // lanes past the last draft say no
        if (no) return i0 + __builtin_ctzll(no);
    }
}

__device__ __forceinline__ double positive(double w) { return w > 0.0 && w < INFINITY ? w : 0.0; }

// Four entries from v on (0 past the row's end), one load where all are inside. Rows of an odd
// vocabulary are aligned to their elements only, which a vector load here allows.
template <typename T> __device__ __forceinline__ void load4(const T *row, int v, int V, float (&x)[4]) {
    if (v + 4 <= V) {
        if constexpr (sizeof(T) == 4) {
            typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
            const f32x4u w = *reinterpret_cast<const f32x4u *>(row + v);
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = w[i];
        } else {
            typedef uint16_t u16x4u __attribute__((ext_vector_type(4), aligned(2)));
            const u16x4u w = *reinterpret_cast<const u16x4u *>(row + v);
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = bf2f(w[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = v + i < V ? Elt<T>::ld(row, v + i) : 0.0f;
    }
}

// The rows that the token after a drafts is drawn from: p_a, and q_a or the draft without weight.
template <typename T> struct Rows {
    const T *p, *q;
    int gone, V;
    __device__ Rows(const VerifyParams &v, int b, int a, int n) : V(v.V) {
        p = (const T *)v.target + ((size_t)b * (v.N + 1) + a) * v.V;
        q = a < n && v.draft ? (const T *)v.draft + ((size_t)b * v.N + a) * v.V : nullptr;
        gone = a < n && !v.draft ? v.drafted[(size_t)b * v.N + a] : -1;
    }
};

template <typename T>
__global__ void __launch_bounds__(256) sum_kernel(VerifyParams p) {
    const int lane = threadIdx.x & 63, b = blockIdx.y;
    const int w = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int n;
    const int a = accepted_of<T>(p, b, lane, &n);
    if (w == 0 && lane == 0) p.accepted[b] = a;
    const Rows<T> r(p, b, a, n);
    for (int k = w * p.rep; k < min((w + 1) * p.rep, p.pieces); k++) {
        const int v0 = k * PIECE + 4 * lane;   // entries v0 + 256 j .. + 3
        float pv[PER / 4][4], qv[PER / 4][4];
#pragma unroll
        for (int j = 0; j < PER / 4; j++) load4(r.p, v0 + 256 * j, p.V, pv[j]);
        if (r.q) {
#pragma unroll
            for (int j = 0; j < PER / 4; j++) load4(r.q, v0 + 256 * j, p.V, qv[j]);
        } else {
#pragma unroll
            for (int j = 0; j < PER / 4; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) qv[j][i] = 0.0f;
        }
        double sw = 0.0, sp = 0.0;
#pragma unroll
        for (int j = 0; j < PER / 4; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const double x = pv[j][i];
                sp += positive(x);
                sw += v0 + 256 * j + i == r.gone ? 0.0 : positive(x - (double)qv[j][i]);
            }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            sw += __shfl_xor(sw, o);
            sp += __shfl_xor(sp, o);
        }
        if (lane == 0) {
            double *dst = p.sums + ((size_t)b * p.pieces + k) * 2;
            dst[0] = sw;
            dst[1] = sp;
        }
    }
}

template <int CTRL, int ROWS> __device__ __forceinline__ double dpp_add(double x) {
    union {
        double d;
        int i[2];
    } v{x}, u;
    u.i[0] = __builtin_amdgcn_update_dpp(0, v.i[0], CTRL, ROWS, 0xf, false);   // lanes without a source add 0
    u.i[1] = __builtin_amdgcn_update_dpp(0, v.i[1], CTRL, ROWS, 0xf, false);
    return x + u.d;
}
// Sum of the lanes up to this one: within rows of 16 by shifts, then each row's total into those behind it.
__device__ __forceinline__ double wave_upto(double x) {
    x = dpp_add<0x111, 0xf>(x);   // row_shr 1
    x = dpp_add<0x112, 0xf>(x);   // row_shr 2
    x = dpp_add<0x114, 0xf>(x);   // row_shr 4
    x = dpp_add<0x118, 0xf>(x);   // row_shr 8
    x = dpp_add<0x142, 0xa>(x);   // row_bcast 15 into rows 1 and 3
    return dpp_add<0x143, 0xc>(x);   // row_bcast 31 into rows 2 and 3
}

// Sum of the 256 threads' values before this one's, and of all. part: 4 doubles of LDS of this call's own.
__device__ __forceinline__ double block_before(double own, double *part, int lane, int wv, double *all) {
    const double upto = wave_upto(own);
    if (lane == 63) part[wv] = upto;
    __syncthreads();
    double before = upto - own, total = 0.0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (i < wv) before += part[i];
        total += part[i];
    }
    *all = total;
    return before;
}

// The value (>= 0) of the first thread of the work-group that `has` one, or of the last; -1 where none has.
// cells: 4 words of LDS of this call's own. (An LDS atomic per lane is worked off lane by lane: 3 us each.)
template <bool LAST> __device__ __forceinline__ int end_of(bool has, int v, int *cells, int lane, int wv) {
    const unsigned long long m = __ballot(has);
    const int mine = m ? __builtin_amdgcn_readlane(v, LAST ? 63 - __builtin_clzll(m) : __builtin_ctzll(m)) : -1;
    if (lane == 0) cells[wv] = mine;
    __syncthreads();
    int end = -1;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int c = cells[LAST ? i : 3 - i];
        if (c >= 0) end = c;
    }
    return end;
}

// The drawn token of a sequence, one work-group: bound by its chain of dependent loads (the sums and the
// accepted count, one piece of the rows) and the scans between them, so what does not depend on them is
// loaded in front, and a thread's first piece stays in registers.
template <typename T>
__global__ void __launch_bounds__(256) draw_kernel(VerifyParams p) {
    __shared__ double part[3][4], before_s;
    __shared__ int cells[4][4];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, b = blockIdx.x;
    const double2 *sums = reinterpret_cast<const double2 *>(p.sums) + (size_t)b * p.pieces;
    // thread t holds pieces [t each, (t + 1) each)
    const int each = (p.pieces + 255) / 256, k0 = min(tid * each, p.pieces), k1 = min(k0 + each, p.pieces);
    const double2 s0 = k0 < k1 ? sums[k0] : make_double2(0.0, 0.0);
    const int x0 = tid < p.N ? p.drafted[(size_t)b * p.N + tid] : -1;
    const double u = (double)p.uniforms[(size_t)b * (p.N + 1) + p.N];
    const int a = p.accepted[b];
    const int n = p.counts ? min(max(p.counts[b], 0), p.N) : p.N;
    const Rows<T> r(p, b, a, n);
    double own = s0.x, total, before;
    for (int k = k0 + 1; k < k1; k++) own += sums[k].x;
    before = block_before(own, part[0], lane, wv, &total);
    const bool plain = !(total > 0.0);   // no weight left: the target's own row
    if (plain) {
        own = s0.y;
        for (int k = k0 + 1; k < k1; k++) own += sums[k].y;
        before = block_before(own, part[1], lane, wv, &total);
    }
    const double goal = u * total;
    // the first piece whose running sum passes the goal, or the last with weight where none does
    int mine = -1, top = -1;
    double run = before, mine_before = 0.0, top_before = 0.0;
    for (int k = k0; k < k1; k++) {
        const double2 sk = k == k0 ? s0 : sums[k];
        const double s = plain ? sk.y : sk.x;
        if (s > 0.0) {
            top = k;
            top_before = run;
            if (run + s > goal && mine < 0) {
                mine = k;
                mine_before = run;
            }
        }
        run += s;
    }
    int piece = end_of<false>(mine >= 0, mine, cells[0], lane, wv), token = -1;
    const bool passed = piece >= 0;
    if (!passed) piece = end_of<true>(top >= 0, top, cells[1], lane, wv);
    if (piece >= 0) {
        if (passed ? mine == piece : top == piece) before_s = passed ? mine_before : top_before;
        const int v0 = piece * PIECE + 4 * tid;
        float pv[4], qv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        load4(r.p, v0, p.V, pv);
        if (r.q && !plain) load4(r.q, v0, p.V, qv);
        double w[4], sum = 0.0, all;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            w[i] = !plain && v0 + i == r.gone ? 0.0 : positive((double)pv[i] - (double)qv[i]);
            sum += w[i];
        }
        double c = block_before(sum, part[2], lane, wv, &all) + before_s;
        int hit = -1, held = -1;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c += w[i];
            if (w[i] > 0.0) {
                held = v0 + i;
                if (c > goal && hit < 0) hit = v0 + i;
            }
        }
        // the first entry that passes the goal; the last with weight where rounding leaves none
        token = end_of<false>(hit >= 0, hit, cells[2], lane, wv);
        if (token < 0) token = end_of<true>(held >= 0, held, cells[3], lane, wv);
    }
    for (int i = tid; i <= p.N; i += 256)
        p.tokens[(size_t)b * (p.N + 1) + i] = i < a ? (i == tid ? x0 : p.drafted[(size_t)b * p.N + i]) : (i == a ? token : -1);
}

}  // namespace

size_t ti_verify_bytes(const ti_verify_args *a) {
    return (size_t)a->num_seqs * ((a->vocab + (size_t)PIECE - 1) / PIECE) * 2 * sizeof(double);
}

int ti_launch_verify_draft(const ti_verify_args *a, hipStream_t s) {
    VerifyParams p{};
    p.target = a->target;
    p.draft = a->draft;
    p.drafted = a->draft_tokens;
    p.counts = a->draft_lens;
    p.uniforms = a->uniforms;
    p.accepted = a->accepted;
    p.tokens = a->tokens;
    p.sums = (double *)a->workspace;
    p.N = a->max_drafts;
    p.V = a->vocab;
    p.pieces = (int)((a->vocab + (long long)PIECE - 1) / PIECE);
    // about 16 waves on each of 256 CUs, so that the drafts' chain of loads is paid once
    p.rep = (int)min((long long)p.pieces, max(1LL, (long long)p.pieces * a->num_seqs / 4096));
    const dim3 grid((p.pieces + 4 * p.rep - 1) / (4 * p.rep), a->num_seqs);
    if (a->dtype == TI_F32) {
        sum_kernel<float><<<grid, 256, 0, s>>>(p);
        if (hipGetLastError() != hipSuccess) return TI_ERR_LAUNCH;
        draw_kernel<float><<<a->num_seqs, 256, 0, s>>>(p);
    } else {
        sum_kernel<uint16_t><<<grid, 256, 0, s>>>(p);
        if (hipGetLastError() != hipSuccess) return TI_ERR_LAUNCH;
        draw_kernel<uint16_t><<<a->num_seqs, 256, 0, s>>>(p);
    }
    return hipGetLastError() == hipSuccess ? TI_OK : TI_ERR_LAUNCH;
}
