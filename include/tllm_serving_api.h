/*
 * tllm_serving_api.h - operators of a quantised serving step, for programs that keep many requests in little memory.
 *
 * Where GPTAttention (tllm_plugin_api.h) keeps its cache in 8 bits under one scale per tensor, takes its block tables from the host
 * and has as many key heads as query heads, these operators work on a PACKED batch (the step's tokens of all requests back to back) and
 *   - take the pages that the tokens go to from a free list in device memory, so that a step needs no host work (tllm_paged_plan);
 *   - hold the cache in int8 or OCP e4m3 with a scale for each page and head, which grows with what the page holds (tllm_paged_append);
 *   - attend to it, grouped heads, causal with an optional window, single tokens and portions of prompts alike (tllm_paged_attention);
 *   - multiply by 4-bit weights with a scale for each group of a row (tllm_group_matmul).
 *
 * Conventions are those of tllm_plugin_api.h: device pointers unless stated otherwise, work is enqueued on `stream`, which has to belong to the
 * current device, nothing synchronises or allocates, 0 on success and non-zero with tllm_last_error() otherwise; every call can be
 * captured into a graph.  Nothing is kept from one call for the next.  Type codes: TLLM_HALF (1), TLLM_INT8 (2), TLLM_FP8 (6: e4m3, largest
 * value 448, no infinity) and 7 for bfloat16.
 */
#ifndef TLLM_SERVING_API_H
#define TLLM_SERVING_API_H

#include "tllm_plugin_api.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TLLM_BF16 7

/* ------------------------------------------------------------------------------------------------
 * One step's pages.  Request b holds lens[b] tokens in the pages block_table[b][0 .. ceil(lens[b] / page_size)) and brings new_lens[b]
 * tokens (0: none); a negative new_lens[b] ends it.  The free blocks are ring[(head + i) mod num_blocks], i < count, with
 * ring_state = {head, count}.  New pages are taken from the ring's front in the order of the requests and of their pages, an ended
 * request's pages go behind its end in that order (they can be taken from the next step on).  Written:
 *   block_table   the new pages' entries (an ended request's row stays as it is, its length becomes 0), ring: the returned blocks;
 *   cu_tokens     [n_seqs + 1] the packed rows of request b are cu_tokens[b] .. cu_tokens[b + 1];
 *   slot_map      [n_rows] block * page_size + offset of each row's token, -1 behind the last row;
 *   positions     [n_rows] its position in its request, -1 behind the last row;
 *   lens_out, ring_state_out: the state behind the step; they may be lens and ring_state themselves (no other two tensors may overlap);
 *   status        [1] 0, or a sum of 1: a request needs more than max_blocks pages, 2: the ring has too few blocks, 4: the step has more than
 *                 n_rows tokens, 8: a negative length, or a ring_state that cannot be (or would hold more than num_blocks).  A step
 *                 with a status changes no table, ring or state, and has no rows: cu_tokens is 0, every slot -1.
 * At most 4096 requests, 2^19 rows, 2^19 pages a request; num_blocks * page_size < 2^31; page_size 16, 32, 64 or 128.
 * Two overlapping calls on the same ring or tables are the caller's mistake.
 * ---------------------------------------------------------------------------------------------- */
typedef struct
{
    int32_t n_seqs, n_rows, page_size, num_blocks, max_blocks;
    int64_t table_stride; /* entries from one request's row of block_table to the next (>= max_blocks) */
    const int32_t* lens;
    const int32_t* new_lens;
    int32_t* ring;
    const int32_t* ring_state;
    int32_t* block_table;
    int32_t* cu_tokens;
    int32_t* slot_map;
    int32_t* positions;
    int32_t* lens_out;
    int32_t* ring_state_out;
    int32_t* status;
} tllm_paged_plan_params_t;

int32_t tllm_paged_plan(const tllm_paged_plan_params_t* p, tllm_stream_t stream);

/* ------------------------------------------------------------------------------------------------
 * Keys and values into the cache, keys (and queries) rotated on the way.  The cache of a layer:
 *   pool   [num_blocks][2][kv_heads][page_size * head_size] elements of 8 bits: keys of a page and head [page_size][head_size], values
 *          [head_size][page_size];
 *   scales fp32 [num_blocks][2][kv_heads]: an element stands for its value times its page's and head's scale.
 * Row t goes to slot slot_map[t]; a negative slot, or one behind the pool's end, is passed over.  A page is filled in order, and the tokens that
 * one call brings to it are consecutive rows: offset 0 starts it anew, with o > 0 its first o tokens are kept.  With
 * a = max(largest magnitude of the call's values for the page and head, 2^-100) and top = 127 (int8) or 448 (e4m3) the scale becomes
 * a / top, or stays what it was if that is larger and o > 0; where it grows the tokens held before are brought to it (rounded once
 * more: half a step of the new scale each time).  Values are rounded to nearest even; infinities count as the largest finite value of the
 * input's type, NaN is stored as 0.  No slot twice in one call, and no two calls on one page at a time.
 * rot_dim > 0: dimensions 0 .. rot_dim of every key, and of every query if there are any, are rotated by rope[position]:
 * (cos, sin)[rot_dim / 2] of fp32, rope_len positions; pairs (i, i + rot_dim / 2), or (2 i, 2 i + 1) with rope_pairs = 1.  A row whose
 * position is not in the table is passed over.  The key is rounded once, from the rotated fp32 value to 8 bits.  q_out may be q, with its strides, and lies on
 * no place of q, k or v otherwise, nor with two rows on one place; rows that are passed over stay as they were.
 * Strides count elements; the last dimension is contiguous; k, v, q and q_out are 16-byte aligned with strides that are multiples of 8.
 * head_size 64, 128 or 256; rot_dim a multiple of 16, at most head_size; page_size as above; n_rows at most 2^19.
 * ---------------------------------------------------------------------------------------------- */
typedef struct
{
    int32_t n_rows, kv_heads, q_heads, head_size, page_size, num_blocks; /* q_heads 0: no queries */
    int32_t dtype, cache_type;                                          /* TLLM_HALF | TLLM_BF16, TLLM_INT8 | TLLM_FP8 */
    int32_t rot_dim, rope_pairs, rope_len;
    const void* k;
    const void* v;
    const void* q;
    void* q_out;
    int64_t k_row, k_head, v_row, v_head, q_row, q_head, q_out_row, q_out_head;
    const int32_t* slot_map;
    const int32_t* positions; /* rot_dim > 0 */
    const float* rope;        /* rot_dim > 0 */
    void* pool;
    float* scales;
} tllm_paged_append_params_t;

int32_t tllm_paged_append(const tllm_paged_append_params_t* p, tllm_stream_t stream);

/* ------------------------------------------------------------------------------------------------
 * Attention of the step's queries to that cache: o = sum_j softmax_j(scale q . k_j) v_j.  Request b has the rows cu_tokens[b] ..
 * cu_tokens[b + 1] of q and out and kv_lens[b] cached tokens, its own rows' keys the last of them: its i-th of n rows is the token at
 * kv_lens[b] - n + i and sees the keys up to itself, the last `window` of them if window > 0.  A row that sees none (a length shorter than its
 * rows) is 0.  Query head h reads key head h / (q_heads / kv_heads).  Rows that belong to no request stay as they were.
 * scale >= 0.  Scores, softmax and sums in fp32.  Two things are rounded on the way: the weights enter the second product as fp16, each to 2^-11 of itself, or to
 * 2^-32 of the row's largest product of weight and page's value scale where its own is below 2^-21 of that; bfloat16 queries enter the first one as fp16 under a
 * power of two per row, exactly down to 2^-17 of the row's largest value and to 2^-25 of it below.  What a row does not see has no part in either.
 * Scores are below 2^24 in magnitude (fp32 has no fraction beyond); a row with larger ones may be NaN.
 *   max_new  no request has more rows (rows behind that many are not computed);
 *   max_kv   an expectation of the longest kv_lens, for how the work is split; any kv_lens up to max_blocks * page_size is right.
 * Table entries that are no block of the pool count as masked.  Lengths beyond the table are cut to it.
 * out may be q itself, with its strides, and lies on no place of it otherwise, nor with two rows on one place.
 * At most 4096 requests and 2^19 rows; n_seqs * kv_heads * ceil(max_new * (q_heads / kv_heads) / 128) is at most 2^25 (64 for 128 with heads of 256): the work is
 * laid out as if every request had max_new rows, and what none has costs a workgroup's start.
 * Workspace: tllm_paged_attention_workspace() bytes, 16-byte aligned, not shared by calls that may overlap.
 * ---------------------------------------------------------------------------------------------- */
typedef struct
{
    int32_t n_seqs, n_rows, q_heads, kv_heads, head_size, page_size, num_blocks, max_blocks;
    int32_t dtype, cache_type, max_new, max_kv, window;
    float scale;
    int64_t table_stride, q_row, q_head, out_row, out_head;
    const void* q;
    const void* pool;
    const float* scales;
    const int32_t* block_table;
    const int32_t* cu_tokens;
    const int32_t* kv_lens;
    void* out;
} tllm_paged_attention_params_t;

/* bytes, 0 when the call needs none; -1 on parameters that the call would refuse */
int64_t tllm_paged_attention_workspace(const tllm_paged_attention_params_t* p);
int32_t tllm_paged_attention(const tllm_paged_attention_params_t* p, void* workspace, tllm_stream_t stream);

/* ------------------------------------------------------------------------------------------------
 * y[m, n] = sum_k x[m, k] q[n, k] s[n, k / group], q in -8 .. 7, group 32, 64 or 128, K a multiple of 32 (the last group may be
 * shorter).  x, y and s fp16 or bfloat16 (one type), sums in fp32.
 * bfloat16 rows hold values below 2^113; a row with larger ones or infinities gives NaN (in fp16 an infinity gives what q x gives: an infinity, or NaN for q = 0).
 * The weights are packed once (tensorrt_llm.quantization.group does it):
 *   packed  [ceil(N / 16)][ceil(K / 128)][64][16] bytes: lane l = 16 g + r of a tile holds, in its 32-bit word j, row r's eight
 *           elements k = 32 j + 8 g + e of the tile, as nibbles q + 8 in the order e = 0 2 4 6 1 3 5 7; padding is 8 (zero);
 *   scales  [ceil(K / group)][16 * ceil(N / 16)], padding 0.
 * x rows start 16-byte aligned (ldx a multiple of 8); y rows 2-byte aligned; no row of y lies on one of x or on the weights (rows of both may alternate).
 * ---------------------------------------------------------------------------------------------- */
typedef struct
{
    int32_t rows, n, k, group, dtype;
    int64_t ldx, ldy; /* elements */
    const void* x;
    const void* packed;
    const void* scales;
    void* y;
} tllm_group_matmul_params_t;

int32_t tllm_group_matmul(const tllm_group_matmul_params_t* p, tllm_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif
