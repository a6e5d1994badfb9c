// Attention over chosen pages: every query token and KV head has a table of page ids and a number
// of keys of its own (page_select.hip makes them), and the token's G query heads attend to keys
// 0 .. length - 1 through that table.
//
// The kernels are the paged decode kernels with a table row, a length and a split count per
// (token, KV head) pair in place of one per sequence (SPARSE in pa_decode.hpp and
// pa_generic.hip): the keys of a pair are all visible to its rows, so only the last tile is masked.
// Steps of several tokens a sequence (max_query_len > 1) take neighbouring tokens in groups: their tables
// are joined into one list in LDS, and a page that several of them keep is read and multiplied once for
// all their rows (GROUP in pa_decode.hpp). Token by token such a step is bound by the L2's rate (512
// tokens of 2048 keys and 8 KV heads: 4.3 GB in 300 us; 64 us in groups of 16).
//
// Pairs take consecutive work-groups with the KV heads innermost: with 8 KV heads (a multiple of
// the 8 XCDs in general) all tokens of a KV head run on one XCD, and the pages that the tokens of
// a step share are read through one L2.
#include <algorithm>

#include "pa_decode.hpp"

using namespace ti;
using namespace ti_decode;

namespace {

// Merge split partials [pair or group of pairs][splits][rows][D + 2]: one wave per query row. Loads of up to
// SB splits are issued before any arithmetic. A pair without keys writes zeros.
template <int D, typename T, int SB>
__global__ void __launch_bounds__(256) sparse_combine_kernel(DecodeParams p, int rows) {
    constexpr int PER = D / 64;
    const int lane = threadIdx.x & 63;
    const int row = (int)(blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));   // token * Hq + head
    if (row >= rows) return;
    const int tok = row / p.Hq, hq = row - tok * p.Hq, h = hq / p.G, pair = tok * p.Hk + h;
    const int group = tok / p.tg;   // p.tg tokens share a unit of partials, packed rows g + G t
    const int len = table_keys(p.lengths[pair], p.bt_stride * p.P);
    const int q0 = p.qsl ? p.qsl[0] : 0, q1 = p.qsl ? p.qsl[p.B] : tok + 1;
    const int splits = p.min_tiles > 0 && len > 0 ? f32_active_splits((len + 15) >> 4, p.splits, p.min_tiles).active : p.splits;
    const size_t stride = (size_t)p.M * (D + 2);
    const float *base = p.part + ((size_t)group * p.Hk + h) * p.splits * stride +
                        (size_t)(hq - h * p.G + (tok - group * p.tg) * p.G) * (D + 2);
    float mx = NEG_BIG, lsum = 0.0f, acc[PER];
#pragma unroll
    for (int k = 0; k < PER; k++) acc[k] = 0.0f;
    for (int sp0 = 0; sp0 < splits; sp0 += SB) {
        float2 ml[SB];
        float dv[SB][PER];
#pragma unroll
        for (int j = 0; j < SB; j++) {
            const float *src = base + min(sp0 + j, splits - 1) * stride;
            ml[j] = *reinterpret_cast<const float2 *>(src + D);
#pragma unroll
            for (int k = 0; k < PER; k++) dv[j][k] = src[lane + 64 * k];
        }
        float bm = mx;
#pragma unroll
        for (int j = 0; j < SB; j++)
            if (sp0 + j < splits) bm = fmaxf(bm, ml[j].x);
        const float alpha = fast_exp2(mx - bm);
        mx = bm;
        lsum *= alpha;
#pragma unroll
        for (int k = 0; k < PER; k++) acc[k] *= alpha;
#pragma unroll
        for (int j = 0; j < SB; j++) {
            const float wgt = sp0 + j < splits ? fast_exp2(ml[j].x - mx) : 0.0f;
            lsum += ml[j].y * wgt;
#pragma unroll
            for (int k = 0; k < PER; k++) acc[k] += dv[j][k] * wgt;
        }
    }
    if (tok < q0 || tok >= q1) return;         // a row of no sequence
    if (len > 0 && splits == 1) return;        // its one split wrote the output
    T *o = reinterpret_cast<T *>(p.out) + (size_t)row * D;
#pragma unroll
    for (int k = 0; k < PER; k++) Elt<T>::st(o, lane + 64 * k, len > 0 ? acc[k] / lsum : 0.0f);
}

template <int D, typename T>
void launch_combine(const DecodeParams &p, int rows, hipStream_t s) {
    const dim3 grid((rows + 3) / 4);
    if (p.splits <= 2) sparse_combine_kernel<D, T, 2><<<grid, 256, 0, s>>>(p, rows);
    else if (p.splits <= 4) sparse_combine_kernel<D, T, 4><<<grid, 256, 0, s>>>(p, rows);
    else if (p.splits <= 8) sparse_combine_kernel<D, T, 8><<<grid, 256, 0, s>>>(p, rows);
    else sparse_combine_kernel<D, T, 16><<<grid, 256, 0, s>>>(p, rows);
}

template <int D, bool INT8, bool PG16>
void launch_sparse_p(const DecodeParams &p, unsigned grid, hipStream_t s) {
    if constexpr (INT8 && D == 128) {   // the decode launch's rule for joint steps
        if (p.G <= 16 && grid <= 256) {
            decode_kernel<D, 1, INT8, PG16, 4, 1, true, true><<<grid, 256, 0, s>>>(p);
            return;
        }
    }
    if (p.G <= 16) decode_kernel<D, 1, INT8, PG16, 4, 1, false, true><<<grid, 256, 0, s>>>(p);
    else if (p.G <= 32) decode_kernel<D, 2, INT8, PG16, 4, 1, false, true><<<grid, 256, 0, s>>>(p);
    else decode_kernel<D, 2, INT8, PG16, 4, 2, false, true><<<grid, 256, 0, s>>>(p);
}

template <int D>
void launch_sparse_d(const DecodeParams &p, bool int8, unsigned grid, hipStream_t s) {
    const bool pg16 = p.pshift >= 4;
    if (int8) pg16 ? launch_sparse_p<D, true, true>(p, grid, s) : launch_sparse_p<D, true, false>(p, grid, s);
    else pg16 ? launch_sparse_p<D, false, true>(p, grid, s) : launch_sparse_p<D, false, false>(p, grid, s);
}

template <int D, bool INT8, int ROWB>
int launch_group_r(const DecodeParams &p, unsigned grid, hipStream_t s) {
    const size_t lds = (size_t)p.tg * p.tg * p.bt_stride * sizeof(uint16_t);
    auto kernel = decode_kernel<D, ROWB, INT8, true, 4, 1, false, true, true>;
    if (lds > (32u << 10) &&
        hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
        return TI_ERR_LAUNCH;
    kernel<<<grid, 256, lds, s>>>(p);
    return TI_OK;
}

template <int D, bool INT8>
int launch_group_d(const DecodeParams &p, unsigned grid, hipStream_t s) {
    if (p.M <= 16) return launch_group_r<D, INT8, 1>(p, grid, s);
    if constexpr (!INT8)
        if (p.M > 32) return launch_group_r<D, INT8, 4>(p, grid, s);
    return launch_group_r<D, INT8, 2>(p, grid, s);
}

// Steps that are worked on in groups of tokens.
bool groups_allowed(const ti_sparse_attention_args *a, const ti_kv_cache *c) {
    const int P = c->page_size;
    return a->max_query_len > 1 && P >= 16 && P <= 32768 && (P & (P - 1)) == 0 && a->q_heads / c->kv_heads <= 16 &&
           (a->dtype != TI_F32 || ti_sparse_f32_mfma(a, c));
}

// Work-groups below which keys are split, for groups of tg tokens.
long long split_target(bool f32, bool int8, int tg) { return f32 || (int8 && tg > 1) ? 512 : 256; }

// The most splits of a table: at most 16 (Float32 32), of at least four 16-key tiles each.
int most_splits(const ti_sparse_attention_args *a, const ti_kv_cache *c) {
    const long long tiles = ((long long)a->table_width * c->page_size + 15) / 16;
    int s = 1;
    while (s < (a->dtype == TI_F32 ? 32 : 16) && tiles >= 8 * s) s <<= 1;
    return s;
}

}  // namespace

// Tokens worked on together, and splits of their keys.
// Groups: bf16 steps of several tokens a sequence over pages of whole 16-key tiles, as many tokens as fill 16
// query rows. 32 rows read a page for twice the tokens at half the work-groups, and pay once 16 would give
// 256 work-groups (tables of 32 pages of 64 keys: 8 steps of 16 tokens 45 -> 36 us, 256 tokens 72 -> 43, 512 tokens
// 136 -> 80; below it one step of 16 18.5 against 19.0-21.4), INT8 caches 512 (256 tokens 51 -> 48, 512
// tokens 99 -> 72). 64 rows, dense caches only (INT8: 72 -> 118 us for 512
// tokens), are one work-group a CU and pay once 32 would give 512 of them
// (512 tokens 80 -> 64 us, 1024 161 -> 127; 400 tokens 82 and 85, 256 43 and 46), with heads of 64, where two
// work-groups of 32 rows share a CU, 1024 (1024 tokens 82 -> 66; 512 42 and 50). Their tables are joined from at
// most GROUP_PAGES entries; 512 for 32 rows of INT8 caches or heads of 64, two work-groups of which share a CU and its
// LDS (tables of 128 pages of 16 keys: INT8, 16 steps of 16 tokens 53 us, 74 with 1024 entries; dense, 8 steps of 16
// tokens 42 and 37; 128 tokens with heads of 64 22 and 25).
// Splits: while there are fewer work-groups than CUs (twice as many for joined INT8 tables: 8 steps of 16 tokens over
// 128 pages of 16 keys 35.2 -> 32.6 us, 4 over 64 pages of 64 38.5 -> 31.2; dense 39.0 -> 43.5), at most 16 and at
// least four 16-key tiles of a full table each (one per wave).
ti_sparse_plan ti_plan_sparse(const ti_sparse_attention_args *a, const ti_kv_cache *c) {
    const int G = a->q_heads / c->kv_heads, P = c->page_size;
    const bool int8 = c->kind == TI_KV_INT8;
    ti_sparse_plan pl{1, 1};
    auto pairs = [&](int tg) { return ((long long)a->total_tokens + tg - 1) / tg * c->kv_heads; };
    const bool f32 = a->dtype == TI_F32;
    if (groups_allowed(a, c)) {
        auto tokens = [&](int rows, int entries) {
            return max(1, min(min(min(rows / G, 32), a->max_query_len), entries / min(a->table_width, entries + 1)));
        };
        pl.tg = tokens(16, GROUP_PAGES);
        const int wide = tokens(32, int8 || c->head_dim == 64 ? GROUP_PAGES / 2 : GROUP_PAGES);
        if (!f32 && wide > pl.tg && pairs(pl.tg) >= (int8 ? 512 : 256)) pl.tg = wide;
        const int wider = tokens(64, GROUP_PAGES);
        if (!f32 && !int8 && wider > pl.tg && pairs(pl.tg) >= (c->head_dim == 128 ? 512 : 1024)) pl.tg = wider;
    }
    const int most = most_splits(a, c);
    while (pl.splits < most && pairs(pl.tg) * pl.splits < split_target(f32, int8, pl.tg)) pl.splits <<= 1;
    return pl;
}

long long ti_sparse_groups(const ti_sparse_attention_args *a, const ti_kv_cache *c) {
    const ti_sparse_plan pl = ti_plan_sparse(a, c);
    return ((long long)a->total_tokens + pl.tg - 1) / pl.tg * c->kv_heads * pl.splits;
}

size_t ti_sparse_bytes(const ti_sparse_attention_args *a, const ti_kv_cache *c) {
    const ti_sparse_plan pl = ti_plan_sparse(a, c);
    if (pl.splits == 1) return 0;
    const size_t groups = ((size_t)a->total_tokens + pl.tg - 1) / pl.tg;
    return groups * pl.tg * a->q_heads * pl.splits * (c->head_dim + 2) * sizeof(float);
}

// Enough for every plan of at most as many tokens, query tokens a sequence and table entries: one of s > 1 splits has
// fewer than split_target work-groups with s / 2 of them, and no more groups and splits than the largest step.
size_t ti_sparse_bound(const ti_sparse_attention_args *a, const ti_kv_cache *c) {
    const int G = a->q_heads / c->kv_heads, splits = most_splits(a, c);
    const bool f32 = a->dtype == TI_F32, int8 = c->kind == TI_KV_INT8;
    const int rows = f32 ? 16 : int8 ? 32 : 64, most = groups_allowed(a, c) ? max(1, min(min(rows / G, 32), a->max_query_len)) : 1;
    long long tokens = 0;   // times splits
    for (int tg = 1; splits > 1 && tg <= most; tg++) {
        const long long groups = ((long long)a->total_tokens + tg - 1) / tg;
        tokens = std::max(tokens, tg * std::min(groups * splits, (split_target(f32, int8, tg) - 1) / c->kv_heads * 2));
    }
    return (size_t)tokens * a->q_heads * (c->head_dim + 2) * sizeof(float);
}

int ti_launch_sparse_attention(const ti_sparse_attention_args *a, const ti_kv_cache *c, hipStream_t s) {
    DecodeParams p{};
    p.q = (const uint16_t *)a->q;
    p.out = (uint16_t *)a->out;
    p.kp = (const uint16_t *)c->k_pages;
    p.vp = (const uint16_t *)c->v_pages;
    p.lq = c->layer_q;
    p.ls = c->layer_scale;
    p.smooth = c->smooth;
    p.qsl = a->query_start_loc;
    p.B = a->num_seqs;
    p.bt = a->tables;
    p.lengths = a->lengths;
    p.part = (float *)a->workspace;
    p.bt_stride = a->table_width;
    p.num_pages = c->num_pages;
    p.P = c->page_size;
    p.pshift = (c->page_size & (c->page_size - 1)) == 0 ? __builtin_ctz(c->page_size) : -1;
    p.Hk = c->kv_heads;
    p.Hq = a->q_heads;
    const ti_sparse_plan pl = ti_plan_sparse(a, c);
    p.G = a->q_heads / c->kv_heads;
    p.tg = pl.tg;
    p.M = pl.tg * p.G;
    p.total = a->total_tokens;
    p.nmax = 1;
    p.splits = pl.splits;
    p.scale_log2 = a->scale * LOG2E;
    const unsigned grid = (unsigned)ti_sparse_groups(a, c);
    if (a->dtype == TI_F32) {
        p.min_tiles = ti_launch_sparse_f32(a, c, pl, s);
        if (p.min_tiles < 0) return TI_ERR_LAUNCH;
    } else {
        const bool int8 = c->kind == TI_KV_INT8;
        if (pl.tg > 1) {
            int r;
            if (c->head_dim == 128) r = int8 ? launch_group_d<128, true>(p, grid, s) : launch_group_d<128, false>(p, grid, s);
            else r = int8 ? launch_group_d<64, true>(p, grid, s) : launch_group_d<64, false>(p, grid, s);
            if (r != TI_OK) return r;
        } else if (c->head_dim == 128) launch_sparse_d<128>(p, int8, grid, s);
        else launch_sparse_d<64>(p, int8, grid, s);
    }
    if (hipGetLastError() != hipSuccess) return TI_ERR_LAUNCH;
    if (p.splits == 1) return TI_OK;
    const int rows = a->total_tokens * a->q_heads;
    if (c->head_dim == 128) {
        if (a->dtype == TI_F32) launch_combine<128, float>(p, rows, s);
        else launch_combine<128, uint16_t>(p, rows, s);
    } else {
        if (a->dtype == TI_F32) launch_combine<64, float>(p, rows, s);
        else launch_combine<64, uint16_t>(p, rows, s);
    }
    return hipGetLastError() == hipSuccess ? TI_OK : TI_ERR_LAUNCH;
}
