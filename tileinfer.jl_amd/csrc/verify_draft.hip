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
// Work. All that is read is one value of p and q per draft and then row a of both (V entries), so a
// sequence's row is shared out over work-groups of CHUNK entries: sum_kernel finds a for itself
// (64 drafts per wave step, all loads of a step at once) and sums its chunk, draw_kernel takes the
// chunk in which the sum passes the goal, and scans that. Every sum has one fixed order.
#include "common.hpp"

using namespace ti;

namespace {

constexpr int CHUNK = 4096;    // entries per work-group: 256 threads of 16
constexpr int PER = CHUNK / 256;

struct VerifyParams {
    const void *target, *draft;
    const int32_t *drafted, *counts;
    const float *uniforms;
    int32_t *accepted, *tokens;
    double *sums;   // [B][chunks][2]: the weights' sum and p_a's
    int N, V, chunks;
};

// Accepted drafts of sequence b; every lane gets the count. *n: the sequence's drafts.
template <typename T>
__device__ __forceinline__ int accepted_of(const VerifyParams &p, int b, int lane, int *count) {
    const int n = p.counts ? min(max(p.counts[b], 0), p.N) : p.N;
    *count = n;
    int i0 = 0;
    for (; i0 < n; i0 += 64) {
        const int i = i0 + lane;
        bool ok = false;
        if (i < n) {
            const int x = p.drafted[(size_t)b * p.N + i];
            const float u = p.uniforms[(size_t)b * (p.N + 1) + i];
            if (x >= 0 && x < p.V) {   // a token that does not exist is not accepted
                const float pv = Elt<T>::ld((const T *)p.target, ((size_t)b * (p.N + 1) + i) * p.V + x);
                const float qv = p.draft ? Elt<T>::ld((const T *)p.draft, ((size_t)b * p.N + i) * p.V + x) : 1.0f;
                ok = (double)u * (double)qv < (double)pv;
            }
        }
        const unsigned long long no = __ballot(!ok);   // lanes past the last draft say no
        if (no) return i0 + __builtin_ctzll(no);
    }
    return n;
}

__device__ __forceinline__ double positive(double w) { return w > 0.0 && w < INFINITY ? w : 0.0; }

// PER consecutive entries of row a from v0 on: their weights w and target probabilities pv.
template <typename T>
__device__ __forceinline__ void weights(const VerifyParams &p, int b, int a, int n, int v0, double (&w)[PER], float (&pv)[PER]) {
    const T *row = (const T *)p.target + ((size_t)b * (p.N + 1) + a) * p.V;
    const bool rejected = a < n;
    const T *qrow = rejected && p.draft ? (const T *)p.draft + ((size_t)b * p.N + a) * p.V : nullptr;
    const int gone = rejected && !p.draft ? p.drafted[(size_t)b * p.N + a] : -1;
    float qv[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int v = v0 + i;
        pv[i] = v < p.V ? Elt<T>::ld(row, v) : 0.0f;
        qv[i] = qrow && v < p.V ? Elt<T>::ld(qrow, v) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) w[i] = v0 + i == gone ? 0.0 : positive((double)pv[i] - (double)qv[i]);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(256) sum_kernel(VerifyParams p) {
    __shared__ double part[4][2];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, b = blockIdx.y;
    int n;
    const int a = accepted_of<T>(p, b, lane, &n);
    double w[PER], sw = 0.0, sp = 0.0;
    float pv[PER];
    weights<T>(p, b, a, n, blockIdx.x * CHUNK + tid * PER, w, pv);
#pragma unroll
    for (int i = 0; i < PER; i++) sw += w[i], sp += positive(pv[i]);
    sw = wave_sum64(sw);
    sp = wave_sum64(sp);
    if (lane == 0) part[wv][0] = sw, part[wv][1] = sp;
    __syncthreads();
    if (tid == 0) {
        double *dst = p.sums + ((size_t)b * p.chunks + blockIdx.x) * 2;
        dst[0] = (part[0][0] + part[1][0]) + (part[2][0] + part[3][0]);
        dst[1] = (part[0][1] + part[1][1]) + (part[2][1] + part[3][1]);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) draw_kernel(VerifyParams p) {
    __shared__ double part[4], goal_s, before_s;
    __shared__ int chunk_s, found, last, plain_s;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, b = blockIdx.x;
    int n;
    const int a = accepted_of<T>(p, b, lane, &n);
    const double *sums = p.sums + (size_t)b * p.chunks * 2;
    if (tid == 0) {
        double tw = 0.0, tp = 0.0;
        for (int c = 0; c < p.chunks; c++) tw += sums[2 * c], tp += sums[2 * c + 1];
        const int plain = !(tw > 0.0);   // no weight left: the target's own row
        const double goal = (double)p.uniforms[(size_t)b * (p.N + 1) + p.N] * (plain ? tp : tw);
        double run = 0.0, before = 0.0;
        int chunk = -1;
        for (int c = 0; c < p.chunks; c++) {
            const double s = sums[2 * c + plain];
            if (!(s > 0.0)) continue;
            chunk = c;   // the last chunk with weight, where none passes the goal
            before = run;
            run += s;
            if (run > goal) break;
        }
        goal_s = goal;
        before_s = before;
        chunk_s = chunk;
        plain_s = plain;
        found = CHUNK;
        last = -1;
    }
    __syncthreads();
    const int chunk = chunk_s;
    int token = -1;
    if (chunk >= 0) {
        double w[PER], own = 0.0;
        float pv[PER];
        weights<T>(p, b, a, n, chunk * CHUNK + tid * PER, w, pv);
        int top = -1;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (plain_s) w[i] = positive(pv[i]);
            own += w[i];
            if (w[i] > 0.0) top = tid * PER + i;
        }
        double incl = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double v = __shfl_up(incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 63) part[wv] = incl;
        __syncthreads();
        double run = before_s + (incl - own);
        for (int i = 0; i < wv; i++) run += part[i];
        int hit = CHUNK;
#pragma unroll
        for (int i = PER - 1; i >= 0; i--) {
            double c = run;
#pragma unroll
            for (int j = 0; j <= i; j++) c += w[j];
            if (w[i] > 0.0 && c > goal_s) hit = tid * PER + i;
        }
        if (hit < CHUNK) atomicMin(&found, hit);
        if (top >= 0) atomicMax(&last, top);
        __syncthreads();
        token = chunk * CHUNK + (found < CHUNK ? found : last);
    }
    if (tid == 0) p.accepted[b] = a;
    for (int i = tid; i <= p.N; i += 256)
        p.tokens[(size_t)b * (p.N + 1) + i] = i < a ? p.drafted[(size_t)b * p.N + i] : (i == a ? token : -1);
}

}  // namespace

size_t ti_verify_bytes(const ti_verify_args *a) {
    return (size_t)a->num_seqs * ((a->vocab + (size_t)CHUNK - 1) / CHUNK) * 2 * sizeof(double);
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
    p.chunks = (int)((a->vocab + (long long)CHUNK - 1) / CHUNK);
    const dim3 grid(p.chunks, a->num_seqs);
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
