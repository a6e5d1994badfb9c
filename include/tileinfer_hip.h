/*
 * tileinfer_hip.h — C ABI of libtileinfer_hip.so, the MI355X (gfx950) paged
 * flash-attention path of TileInfer.jl.
 *
 * The entry points of paged attention and the cache replace one method each of the reference's
 * op interface (src/ops/interface.jl) for its TileBackend kernels; each declaration cites the
 * reference function it stands in for. Page bounds, page selection, attention over selected pages
 * and draft verification have no counterpart there: they work on the same
 * caches, block tables and steps. All pointers are device pointers unless noted;
 * calls enqueue work on `stream` and return without synchronizing. The library never
 * allocates device memory: the caller owns pools, inputs, outputs and the workspace.
 * Errors are returned as ti_status codes, never thrown; argument checks run on the host
 * before any HIP call, so they work without a GPU.
 *
 * Layouts are C-order, i.e. the reference's column-major shapes reversed, so a Julia
 * array is passed with no copy:
 *   per-head tensors (head_dim, heads, n)               -> [n][heads][head_dim]
 *   dense pools (head_dim, page_size, kv_heads, pages)  -> [pages][kv_heads][page_size][head_dim]
 *   INT8 layer arrays (int8_kv_pools, src/ops/quant.jl:104-109):
 *     layer_q     (D, P, Hk, pages, 2) int8             -> [2][pages][Hk][P][D] (keys first)
 *     layer_scale (P, Hk, pages, 2) Float32             -> [2][pages][Hk][P]
 *     smooth      (D,) Float32 (the keys' smoothing; values use ones)
 *   8-bit block layer arrays (TI_KV_FP8):
 *     layer_q     [2][pages][Hk][P][D] e4m3 (keys first)
 *     layer_scale [2][pages][Hk] Float32 powers of two
 *   rotary table cos_sin (D, 2 max_len)                 -> [max_len][2][D] (cos, then sin)
 *   block tables: int32, 1-based page ids, zero-padded past a sequence's pages
 *   slots: int32, 1-based, slot s = offset (s-1) % P of page (s-1) / P + 1
 *   positions: int32, 0-based
 */
#ifndef TILEINFER_HIP_H
#define TILEINFER_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
    TI_OK = 0,
    TI_ERR_INVALID_ARG = 1,     /* null pointer, non-positive size, mismatched shapes */
    TI_ERR_UNSUPPORTED = 2,     /* a shape or type no kernel covers (e.g. head_dim 96) */
    TI_ERR_WORKSPACE = 3,       /* workspace missing or smaller than ti_attention_workspace_bytes */
    TI_ERR_LAUNCH = 4,          /* the HIP launch failed */
} ti_status;

typedef enum { TI_F32 = 0, TI_BF16 = 1 } ti_dtype;      /* activations / dense pools */
typedef enum { TI_KV_DENSE = 0, TI_KV_INT8 = 1, TI_KV_FP8 = 2 } ti_kv_kind;

/* Path selection for ti_attention. AUTO follows the reference's rule
 * (src/ops/tile/attention.jl:265, :351-352): split-KV decode for short steps, the prefill
 * kernel otherwise. PREFILL takes the prefill family and lets the library pick its
 * variant from host shapes; the last five pin one variant of it (for tests and tuning:
 * every variant gives results within the same tolerances, and pinned variants that the
 * shapes do not allow fall back to the library's pick):
 *   PREFILL_STAGED    four-wave kernel, K/V tiles staged through registers into LDS
 *   PREFILL_DIRECT    four-wave kernel, direct global -> LDS tile loads (bf16 dense cache,
 *                     head_dim 128, pages of 2^k >= 16 tokens; otherwise staged)
 *   PREFILL_PINGPONG  eight-wave ping-pong kernel, 256 packed rows per work-group (bf16 dense
 *                     cache, head_dim 128, pages of 2^k >= 16 tokens, 256 % (q_heads /
 *                     kv_heads) == 0)
 *   PREFILL_PAIRED    four-wave kernel with direct loads whose work-groups each take a
 *                     heavy and a light 32-row q-tile of a causal step (direct-load shapes,
 *                     32 % (q_heads / kv_heads) == 0, the shapes' unsplit two-wave plan)
 *   PREFILL_PAIRED16  the same paired work-groups on sixteen waves of 16 rows each (four
 *                     per SIMD; the default where the paired plan applies and no form of the
 *                     ping-pong kernel is taken) */
typedef enum {
    TI_PATH_AUTO = 0,
    TI_PATH_DECODE = 1,
    TI_PATH_PREFILL = 2,
    TI_PATH_PREFILL_STAGED = 3,
    TI_PATH_PREFILL_DIRECT = 4,
    TI_PATH_PREFILL_PINGPONG = 5,
    TI_PATH_PREFILL_PAIRED = 6,
    TI_PATH_PREFILL_PAIRED16 = 7,
} ti_path;

/* One layer's KV cache: dense pools in the activations' type, an INT8 layer
 * (Int8Pages pair: src/ops/quant.jl:86-92), or an 8-bit block layer. Host struct of device pointers.
 *
 * 8-bit block layers (TI_KV_FP8) hold e4m3 values and one scale for each block, the keys (or the values)
 * of a page and KV head: a value stands for itself times the scale, a power of two between 2^-120 and 2^120.
 * head_dim 64 or 128, pages of 2^k keys from 16 to 1024, block tables of at most 2^30 positions. ti_store_kv and
 * ti_attention_inputs write them, ti_attention, ti_attention_noalloc and ti_window_attention read them; page bounds and sparse
 * attention do not take them (TI_ERR_UNSUPPORTED). `path` names no variants for them: other than TI_PATH_DECODE, the library's pick
 * runs. Where a product meets a value that is not finite, the rows of its work-group are done again key by
 * key over what each of them sees (as in ti_window_attention): slow, and right. */
typedef struct {
    int32_t kind;               /* ti_kv_kind */
    int32_t head_dim;           /* D: 64 or 128 */
    int32_t page_size;          /* P: positions per page (any >= 1; 16 and 64 are tuned) */
    int32_t kv_heads;           /* Hk */
    int32_t num_pages;          /* pages in the pool; page ids are 1..num_pages */
    void *k_pages;              /* dense: [num_pages][Hk][P][D] */
    void *v_pages;
    int8_t *layer_q;            /* int8, fp8: [2][num_pages][Hk][P][D] */
    float *layer_scale;         /* int8: [2][num_pages][Hk][P]; fp8: [2][num_pages][Hk] */
    const float *smooth;        /* int8: [D] keys' smoothing factors */
} ti_kv_cache;

/* Arguments of ti_attention. A batch of `num_seqs` sequences; sequence b owns the query
 * tokens [qsl[b], qsl[b+1]) of q (or [b*max_query_len, (b+1)*max_query_len) when
 * query_start_loc is NULL), its first query sits at positions[qsl[b]] and it attends to
 * keys 0 .. positions[qsl[b]] + n_b - 1 through block table row b. num_seqs = 1 is
 * exactly the reference's one-sequence op.
 * Contract on the device data (not checkable on the host): a row of block_tables must hold
 * at least ceil(len / page_size) page ids for the sequence's len = positions[qsl[b]] + n_b
 * keys, and n_b <= max_query_len. Out of contract, no access leaves the block-table row or
 * the pool (page indices are clamped to [0, block_table_stride), page ids to the pool,
 * n_b to max_query_len), but the output is unspecified. */
typedef struct {
    int32_t dtype;                    /* ti_dtype of q, out (and dense pools) */
    int32_t q_heads;                  /* Hq; Hq % Hk == 0 */
    int32_t num_seqs;                 /* B */
    int32_t max_query_len;            /* max n_b (sizes the grid; host value) */
    int32_t total_tokens;             /* sum n_b (rows of q and out) */
    int32_t block_table_stride;       /* entries per block-table row */
    const void *q;                    /* [total_tokens][Hq][D] */
    void *out;                        /* [total_tokens][Hq][D] */
    const int32_t *positions;         /* [total_tokens] 0-based positions */
    const int32_t *query_start_loc;   /* [B+1] token offsets, or NULL: uniform max_query_len */
    const int32_t *block_tables;      /* [B][block_table_stride] 1-based page ids */
    float scale;                      /* softmax scale, e.g. 1/sqrt(D); finite and > 0 */
    int32_t causal;                   /* 1: key i visible to query t iff i <= pos(t) */
    int32_t path;                     /* ti_path */
    void *workspace;                  /* split-KV partials; may be NULL for the prefill path */
    size_t workspace_bytes;
} ti_attention_args;

/* Library version string, e.g. "tileinfer_hip 0.1.0 gfx950". Host only. */
const char *ti_version(void);

/* Human-readable name of a status code. Host only. */
const char *ti_status_string(int status);

/*
 * Bytes of workspace ti_attention needs for these shapes (0 when the call needs none).
 * Replaces attention_workspace(::TileBackend, q, k_pages) and decode_workspace
 * (src/ops/tile/attention.jl:279-284, :351-352; interface src/ops/interface.jl:275-280).
 * Like the reference's, it depends only on the query shape (dtype, q_heads, num_seqs,
 * max_query_len, path) and the cache, never on the block tables or context length, so
 * a captured graph keeps a fixed workspace. Host only; writes the size to *bytes.
 */
int ti_attention_workspace_bytes(const ti_attention_args *args, const ti_kv_cache *cache,
                                 size_t *bytes);

/*
 * Paged causal (or non-causal) grouped-query attention over the KV cache.
 * Replaces attention!(::TileBackend, out, workspace, q, k_pages, v_pages, block_table,
 * positions, scale; causal) (src/ops/tile/attention.jl:359-366; interface
 * src/ops/interface.jl:152-158) and the allocating attention(...) when the caller
 * provides out and workspace (attention.jl:368-371). Kernels: split-KV decode + combine
 * (attention.jl:185-245) and the causal / chunked / non-causal prefill
 * (attention.jl:130-177), each for dense (bf16, fp32) and INT8 caches.
 * `stream` is a hipStream_t (NULL = default stream).
 */
int ti_attention(const ti_attention_args *args, const ti_kv_cache *cache, void *stream);

/* Bytes of the static device scratch behind ti_attention_noalloc (per GPU). */
#define TI_NOALLOC_SCRATCH_BYTES (32u << 20)

/*
 * ti_attention without a caller workspace and without any allocation: split-KV partials
 * go to a static device array of TI_NOALLOC_SCRATCH_BYTES per GPU (the library's own,
 * held until the process ends). No counterpart in the reference: this is for callers that
 * cannot allocate (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc). It calls no hipMalloc / hipFree and no allocating library routine.
 * Same arguments, kernels and results as ti_attention with a sufficient workspace;
 * args->workspace and args->workspace_bytes are ignored. Where the workspace
 * (ti_attention_workspace_bytes) exceeds the scratch, prefill and fp32 steps run unsplit
 * (as ti_attention does without a workspace) and decode steps, whose workspace is
 * mandatory, are rejected with TI_ERR_WORKSPACE before anything is launched. Every call on
 * one GPU shares that GPU's scratch: calls that overlap on one GPU (several streams,
 * several host threads) race and must be serialized by the caller. Nothing in the scratch
 * needs clearing between calls (every partial a launch reads is written by the same
 * launch). `stream` must belong to the current device (TI_ERR_INVALID_ARG otherwise).
 * The scratch is reserved on every GPU where the library's code object is loaded, whether
 * or not this entry point is called.
 */
int ti_attention_noalloc(const ti_attention_args *args, const ti_kv_cache *cache, void *stream);

/*
 * Write keys and values of n tokens at 1-based slots, bit-exact copies (dense) or
 * quantized per (token, KV head) vector (INT8: q = floor(x 127/max|x| + 1/2),
 * s = max|x|/127, keys divided by smooth first).
 * Replaces store_kv!(::TileBackend, k_pages, v_pages, k, v, slots)
 * (src/ops/tile/elementwise.jl:133-140 and :180-188; reference
 * src/ops/reference.jl:64-74, src/ops/quant.jl:147-159).
 * k, v: [n][Hk][D] in dtype. Slots outside the pool are skipped.
 *
 * 8-bit block layers: a block's scale is the least 2^e (e from -120 to 120) with |x| <= 448 2^e for every finite element
 * that its rows were written with, and a row holds x 2^-e rounded to the nearest e4m3 value (ties to even); an element
 * that is not finite is held as NaN, one of 248 2^120 (3.3e38) or more as 2^128, infinity in 32 bits. Rows are written
 * from a page's first on: a call that writes a page's first row begins the block anew, with the scale of this call's rows
 * alone (other rows of the page then hold nothing). Otherwise the scale only grows; where it does, the rows that the
 * block holds are divided by the growth, which is exact but for values that become subnormal (each time rounded again, by
 * at most 2^-10 of the new scale). The rows of one page may be anywhere among the call's; of two for one slot the later
 * stays.
 */
int ti_store_kv(int dtype, const ti_kv_cache *cache, const void *k, const void *v,
                const int32_t *slots, int n, void *stream);

/*
 * RMS normalization of `rows` rows of `hidden` elements: y = rnd(rnd(x inv_rms) w) with
 * inv_rms = 1 / sqrt(sum x^2 / hidden + eps) in Float32, rnd = round to T (y may alias x).
 * Replaces rmsnorm!(::TileBackend, y, x, w, eps) (src/ops/tile/norm.jl:31-38; interface
 * src/ops/interface.jl:118-122), the q/k norm of the generic attention_inputs! chain
 * (interface.jl:175). Per-head rows (hidden <= 128) are bit-identical to the norm inside
 * ti_attention_inputs. x, y: [rows][hidden], w: [hidden], all in dtype.
 */
int ti_rmsnorm(int dtype, void *y, const void *x, const void *w, int rows, int hidden, float eps,
               void *stream);

/*
 * Rotary embedding ("rotate half") of x [n][heads][D] into y at 0-based positions,
 * rounding to T after every operation as the reference does.
 * Replaces rope!(::TileBackend, y, x, cos, sin, positions)
 * (src/ops/tile/elementwise.jl:10-36; reference src/ops/reference.jl:32-39).
 * cos_table, sin_table: [table_len][D]. Tokens whose position lies outside [0, table_len)
 * are skipped: their rows of y are left untouched (the reference indexes past its table
 * there; a kernel cannot raise, so the row keeps what it held).
 */
int ti_rope(int dtype, void *y, const void *x, const void *cos_table, const void *sin_table,
            int table_len, const int32_t *positions, int n, int heads, int head_dim, void *stream);

/*
 * Everything between the fused qkv projection and attention, in one launch: optional
 * Qwen3 q/k RMSNorm, RoPE at positions, queries into q_out, keys and values into the
 * cache at slots (quantized for an INT8 cache).
 * Replaces attention_inputs!(::TileBackend, q, k_pages, v_pages, qkv, q_norm, k_norm,
 * table, positions, slots, eps) (src/ops/tile/fused.jl:94-130; generic chain
 * src/ops/interface.jl:169-179).
 * qkv: [n][q_heads + 2 Hk][D]; q_out: [n][q_heads][D]; q_norm, k_norm: [D] or both NULL;
 * cos_sin: [table_len][2][D]. A token whose position lies outside [0, table_len) writes
 * nothing (its q_out rows are left untouched and its K/V slot is not written); a token
 * whose slot lies outside the pool writes no K/V row. 8-bit block layers are written as by ti_store_kv.
 */
int ti_attention_inputs(int dtype, void *q_out, const ti_kv_cache *cache, const void *qkv,
                        const void *q_norm, const void *k_norm, const void *cos_sin,
                        int table_len, const int32_t *positions, const int32_t *slots, int n,
                        int q_heads, float eps, void *stream);

/* ---- attention over chosen pages, and draft verification ----------------------------------
 * No counterpart in the reference's ops: a long context read in part, and the end of the verify step
 * that its speculative engine makes of attention calls.
 * Rows of the packed token arrays that belong to no sequence (before query_start_loc[0], from
 * query_start_loc[num_seqs] on) are left as they were by all of them. */

/* Bounds of the keys of a layer's pages, kept beside its cache: for each page and KV head the keys'
 * largest (first row) and smallest element in each dimension, rounded outward to whole multiples
 * of the page's power of two `scale`. 16-byte aligned.
 * One power of two serves all of a head's dimensions, so a few dimensions with keys much larger than the rest
 * leave these a step or two wide, and the selection loses pages for it (ti_select_pages). `channel` takes that out:
 * keys are divided by their dimension's power of two before they are bounded, queries multiplied by it before
 * they are rounded, which leaves every product of the two as it is. The same pointer in both calls. */
typedef struct {
    int8_t *bounds;             /* [num_pages][Hk][2][D] */
    float *scale;               /* [num_pages][Hk] */
    const float *channel;       /* [Hk][D] powers of two, about the dimensions' largest |k|; or NULL: ones */
} ti_key_bounds;

/*
 * Refresh the bounds of the pages that hold the positions of a step (those of the step's queries, as
 * in ti_attention_args: sequence b's n_b positions from positions[qsl[b]] on), from all keys that
 * the cache holds in them up to the step's end. Called after the step's keys are written
 * (ti_attention_inputs, ti_store_kv). The result depends on the cached keys alone, so a step that
 * is taken back and written again needs no other call. For an INT8 cache a key is its value times
 * scale times smoothing, rounded to float after each product; with `channel` a key is what its channel leaves of
 * it (exactly, above 2^-126). A page with a key that is not finite
 * gets bounds 127 and -127 and an infinite scale, and is kept by every selection that reaches
 * its score. Pages whose id lies outside the pool, or past the block-table row, are skipped. Two
 * sequences of a call that write into one page, or two entries of a block-table row that name one,
 * are not supported: each part of the page's bounds is one of the two's.
 * head_dim 64 or 128. dtype: of dense pools.
 */
int ti_update_key_bounds(int dtype, const ti_kv_cache *cache, const ti_key_bounds *bounds,
                         const int32_t *block_tables, int block_table_stride, const int32_t *positions,
                         const int32_t *query_start_loc, int num_seqs, int max_query_len, int total_tokens,
                         void *stream);

/* Arguments of ti_select_pages; the step as in ti_attention_args. */
typedef struct {
    int32_t dtype;                    /* ti_dtype of q */
    int32_t q_heads, kv_heads;        /* q_heads % kv_heads == 0, at most 64 query heads per KV head */
    int32_t head_dim;                 /* 64 or 128 */
    int32_t page_size, num_pages;
    int32_t num_seqs, max_query_len, total_tokens;
    int32_t block_table_stride;
    int32_t keep;                     /* pages kept: the width of a table */
    int32_t sinks, window;            /* the first and last pages always kept: sinks >= 0, window >= 1,
                                         sinks + window <= keep */
    int32_t causal;                   /* 1: a query sees the pages up to its own position's */
    const void *q;                    /* [total_tokens][Hq][D] */
    ti_key_bounds bounds;
    const int32_t *positions, *query_start_loc, *block_tables;
    int32_t *tables;                  /* [total_tokens][Hk][keep]: out */
    int32_t *lengths;                 /* [total_tokens][Hk]: out */
    void *workspace;                  /* 16-byte aligned */
    size_t workspace_bytes;
} ti_select_args;

/*
 * For each query token and KV head the `keep` pages of its sequence whose keys can matter most.
 * A query head (times bounds.channel) is taken as whole numbers w = rint(q / 2^e) (to even), 2^e the least power of two
 * (from 2^-126 on) with |q| <= 127 2^e; a page's score is the largest over the KV head's query heads of
 * 2^e scale sum_d (w_d hi_d where w_d > 0, else w_d lo_d), which no key inside the bounds exceeds with the
 * rounded query 2^e w (it is the sum of max(w_d hi_d, w_d lo_d), since hi_d >= lo_d). With the query itself a key may
 * exceed it by 2^(e - 1) scale sum_d max |hi_d|, |lo_d|, and it may itself exceed the score of unrounded bounds by
 * as much and by scale 2^e sum_d |w_d|: a page that would be kept can be left out for others within these
 * distances. Of 64 pages kept of 512 (random keys about a mean of the page's own, 4 query heads) 62 are
 * those of the unrounded score; with two of 128 dimensions 5 or 10 times as large 49, and 60 to 61 with `channel`.
 * The first `sinks`
 * and the last `window` visible pages are kept, then pages by score, equal ones in order; the sums
 * are exact, so which are kept does not depend on how they are made. A query head with an element
 * that is not finite scores 0 everywhere.
 * tables: the kept pages' ids in order of position, zero-padded; lengths: the keys they hold up to
 * the last visible one, as ti_sparse_attention takes them. All visible pages are kept while there
 * are at most `keep`.
 * The workspace is 4 bytes per token, KV head and (rounded to 256) table entry, up to 128 MiB (at least one token's). It
 * grows with total_tokens and block_table_stride and depends on neither num_seqs nor max_query_len.
 */
int ti_select_pages_workspace_bytes(const ti_select_args *args, size_t *bytes);
int ti_select_pages(const ti_select_args *args, void *stream);

/* Arguments of ti_sparse_attention. */
typedef struct {
    int32_t dtype;                    /* ti_dtype of q, out (and dense pools) */
    int32_t q_heads;                  /* q_heads % kv_heads == 0; bf16: at most 64 per KV head */
    int32_t total_tokens;
    int32_t table_width;              /* entries per table */
    int32_t num_seqs, max_query_len;  /* the step that the tokens are: rows next to each other that belong
                                         to one sequence are worked on together (max_query_len > 1);
                                         results are the same within rounding */
    const void *q;                    /* [total_tokens][Hq][D] */
    void *out;                        /* [total_tokens][Hq][D] */
    const int32_t *tables;            /* [total_tokens][Hk][table_width] 1-based page ids */
    const int32_t *lengths;           /* [total_tokens][Hk] keys, at most table_width * page_size */
    const int32_t *query_start_loc;   /* [num_seqs + 1], or NULL: every row belongs to a sequence */
    float scale;                      /* softmax scale: finite and > 0 */
    void *workspace;                  /* 16-byte aligned */
    size_t workspace_bytes;
} ti_sparse_attention_args;

/*
 * Attention of each query token and KV head over keys 0 .. length - 1 of its own table of pages, all
 * of them visible: the last entry in use may hold fewer than page_size keys. A token without keys
 * (length <= 0) gets zeros; longer lengths read as table_width * page_size. An entry outside the
 * pool is clamped into it, as in ti_attention; a page that a table names twice counts twice.
 * Over INT8 caches a weight (at most 1) times its value's scale is held in 16 bits, as in ti_attention: value
 * scales above 65504 overflow, and products below 2^-14 are rounded to multiples of 2^-24.
 * ti_sparse_attention_workspace_bytes is what a call of exactly these sizes needs: fewer tokens, or another
 * max_query_len, may need more, because keys are split where work-groups are few. ..._workspace_bound is enough
 * for every call with these heads, types and pages of at most total_tokens tokens, max_query_len tokens a sequence
 * and table_width entries, for a workspace that is made once.
 */
int ti_sparse_attention_workspace_bytes(const ti_sparse_attention_args *args, const ti_kv_cache *cache, size_t *bytes);
int ti_sparse_attention_workspace_bound(const ti_sparse_attention_args *args, const ti_kv_cache *cache, size_t *bytes);
int ti_sparse_attention(const ti_sparse_attention_args *args, const ti_kv_cache *cache, void *stream);

/* Arguments of ti_verify_draft. */
typedef struct {
    int32_t dtype;                    /* ti_dtype of target and draft */
    int32_t num_seqs, max_drafts;     /* B, N >= 0 */
    int32_t vocab;                    /* V */
    const int32_t *draft_tokens;      /* [B][N] 0-based */
    const int32_t *draft_lens;        /* [B] drafts of each sequence (clamped to 0 .. N), or NULL: N */
    const void *target;               /* [B][N + 1][V] the target's probabilities */
    const void *draft;                /* [B][N][V] the drafter's, or NULL: it gave its tokens alone */
    const float *uniforms;            /* [B][N + 1] in [0, 1): one per draft, the last for the drawn token */
    int32_t *accepted;                /* [B]: out */
    int32_t *tokens;                  /* [B][N + 1]: out, the accepted drafts, the drawn token, then -1 */
    void *workspace;                  /* 16-byte aligned */
    size_t workspace_bytes;
} ti_verify_args;

/*
 * Speculative sampling: draft i is accepted while u_i q_i(x_i) < p_i(x_i) (q = 1 without a drafter's
 * probabilities); after a of them one token is drawn with the last uniform from max(p_a - q_a, 0), or
 * p_a without x_a, where a draft was rejected, and from p_a where none was: the lowest token with
 * weight whose running sum exceeds u times the sum of all. Products and sums in double. Entries that
 * are not positive and finite have no weight; without any weight p_a itself is taken, and -1 where
 * that has none. A draft token outside [0, V) is rejected.
 */
int ti_verify_draft_workspace_bytes(const ti_verify_args *args, size_t *bytes);
int ti_verify_draft(const ti_verify_args *args, void *stream);

/* ---- attention with a sliding window ----------------------------------------------------------
 *
 * ti_attention with causal = 1, where the query at position p sees the keys p - window + 1 .. p and the keys
 * 0 .. sinks - 1 (never past p): window >= 1, sinks >= 0. Arguments, caches and steps as in ti_attention (path:
 * TI_PATH_AUTO; workspace of ti_window_attention_workspace_bytes, which depends on the window too, mandatory
 * where that is not 0; block tables of at most 2^30 positions). Block-table entries of pages that hold no visible key of any
 * of the sequence's queries are not used: their pages may have been given back. Rows of q and out that belong to no sequence are left as they were.
 *
 * A key that a query does not see leaves its output as it is whatever the cache holds there, NaN and infinities
 * among it. The rows of a work-group are worked on together, so where a product is not finite they are done
 * again row by row over the keys that each sees: right, but slow (a cache with NaN in it takes hundreds of times as long).
 */
int ti_window_attention_workspace_bytes(const ti_attention_args *args, int window, int sinks, const ti_kv_cache *cache,
                                        size_t *bytes);
int ti_window_attention(const ti_attention_args *args, int window, int sinks, const ti_kv_cache *cache, void *stream);

/* ---- the page bookkeeping of a step, on the device ----------------------------------------------
 *
 * The pages of a pool and the sequences that hold them, as device arrays: what BlockManager (src/kv/block_manager.jl:39-100)
 * keeps on the host. A step can be reserved, run and taken back in one captured graph.
 * Page i of sequence b (positions i P .. i P + P - 1) is tables[b][i]. With a window, release gives back the pages that
 * no later query can see, those from page ceil(sinks / P) up to behind[b]; their entries are 0. (behind[b] starts as
 * ceil(sinks / P). Over tables of which pages went back before, it counts them: entries in front of it are not given back again.)
 * Calls on one pool must not overlap. `ticket` is 0 between calls. */
typedef struct {
    int32_t num_pages, page_size;
    int32_t num_seqs;                 /* S: 1 to 4096 */
    int32_t table_width;              /* W */
    int32_t window, sinks;            /* of the attention over the pool: window 0: none, every page is kept */
    int32_t *free;                    /* [num_pages] stack of free page ids, 1-based, the next one on top */
    int32_t *free_count;              /* [1] ids on the stack */
    int32_t *tables;                  /* [S][W] page ids, 0 where none */
    int32_t *lengths;                 /* [S] positions */
    int32_t *behind;                  /* [S]; NULL without a window */
    int32_t *ticket;                  /* [1] */
} ti_page_pool;

/*
 * counts[b] more positions for each sequence (a negative count is 0): pages off the stack in order of sequence and position
 * into the tables, lengths moved on, and the step's arrays: query_start_loc [S + 1]; positions and slots [tokens]
 * of the step's tokens, 0 behind them (slot 0 writes nothing).
 * short_of [1]: 0; or the pages that were missing; or -1 where a sequence would outgrow its table or the step
 * `tokens`. Unless it is 0 nothing is reserved: pool unchanged, query_start_loc, positions and slots 0.
 */
int ti_reserve_pages(const ti_page_pool *pool, const int32_t *counts, int tokens, int32_t *positions, int32_t *slots,
                     int32_t *query_start_loc, int32_t *short_of, void *stream);

/*
 * Sequences cut to keep[b] positions (0 .. lengths[b]; others are clamped): pages that only later positions use
 * go back, and with a window those that a query at position keep[b] or later does not see. The stack gets them in
 * the opposite order to that in which ti_reserve_pages takes them, so a step taken back whole leaves the pool as it was.
 * A sequence must not be cut to below a position whose window reaches into pages given back before.
 */
int ti_release_pages(const ti_page_pool *pool, const int32_t *keep, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* TILEINFER_HIP_H */
