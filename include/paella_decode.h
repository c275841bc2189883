/*
 * paella_decode.h -- C-ABI of the operators of a decoding step over a paged cache, hand-written for gfx950: appending
 * keys and values (with the norms and the rotation of queries and keys on the way), attention for sequences that share
 * a prefix, and beam search's selection and reordering.  No counterpart in the reference, whose models are CNNs; the
 * entry points follow paella_ops.h (stream or direct-dispatch queue, job_id and notifier hooks, return codes, launch
 * shapes for the scheduler, one launch per call but for attention plans of two stages), so a job definition issues them like any other operator.
 *
 * The cache of one layer is two tensors [num_pages][kv_heads][page_size][head_dim], keys and values, on 16-byte
 * boundaries.  A sequence's own token i lies in slot i % page_size of page tables[sequence][i / page_size]; the shared
 * prefix lies the same way in the pages of prefix_table.  All lengths and tables are device data, so a captured graph
 * follows them.  Offsets into the cache are 64-bit; attention sees a sequence's first 2^30 own tokens.
 *
 * Device data that the host cannot check is checked where it is used: a page number outside the cache, or a token
 * beyond its row of the table, is never written and takes no part in attention; a negative length counts as 0; no
 * access leaves the tensors whatever the numbers are.  `starts` has to begin with 0 and must not decrease, nor grow by more than
 * max_new from one entry to the next; the outputs of a call that breaks this are undefined, and so is the workspace of an attention
 * call (fill it with zeros again).
 */
#ifndef PAELLA_DECODE_H
#define PAELLA_DECODE_H

#include <stddef.h>
#include <stdint.h>

#include "paella_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

enum paella_dtype { PAELLA_F32 = 0, PAELLA_BF16 = 1, PAELLA_F16 = 2 };

typedef struct paella_kv_cache {
    void* k;
    void* v;
    int dtype;                   /* enum paella_dtype: of the cache and of the queries, keys, values and outputs beside it */
    int num_pages, kv_heads, page_size, head_dim;   /* page_size and head_dim: multiples of 8; head_dim at most 512; a page under 2 GiB */
} paella_kv_cache;

/* The new tokens of a batch.  Row t of queries, keys, values and outputs belongs to sequence b for starts[b] <= t <
 * starts[b + 1] (starts NULL: every sequence has max_new rows); as new token j = t - starts[b] it is the sequence's own
 * token past[b] + j, at position prefix_len + past[b] + j.  Rows behind the last sequence are neither read nor written. */
typedef struct paella_kv_batch {
    int sequences;
    int max_new;                 /* most new tokens of any sequence */
    int tokens;                  /* rows; sequences * max_new where starts is NULL */
    int max_pages;               /* entries of a sequence's row of the table */
    int prefix_len;              /* tokens of the shared prefix; 0: there is none and prefix_table is not looked at */
    const int32_t* starts;       /* [sequences + 1] or NULL */
    const int32_t* past;         /* [sequences]: own tokens in the cache before this step */
    const int32_t* tables;       /* [sequences][max_pages] */
    const int32_t* prefix_table; /* [ceil(prefix_len / page_size)] */
} paella_kv_batch;

/* ---------------------------------------------------------------- append */

typedef struct paella_kv_append_desc {
    int heads;                   /* query heads; 0: keys and values only */
    int rotary_dim;              /* leading values of a head that are rotated: a multiple of 16, at most head_dim; 0: none */
    int interleaved;             /* pairs are (2i, 2i + 1); 0: (i, i + rotary_dim / 2) */
    float eps;                   /* of the norms */
    int64_t q_stride, k_stride, v_stride;  /* values from one row to the next, multiples of 8; heads lie side by side, so views of one packed projection do */
} paella_kv_append_desc;

/* Per head x' = x / sqrt(mean(x * x) + eps) * weight[head_dim] (where q_weight / k_weight is given), then pair i turned by
 * the angle position * inv_freq[i] (a product taken in 64 bits, so far positions keep their angle), in 32 bits with one rounding
 * at the end.  Queries go to q_out [tokens][heads][head_dim] (which may be q where q_stride is heads * head_dim), keys and, as
 * they are, values to the cache.  q, q_out: NULL where heads is 0; inv_freq: [rotary_dim / 2], NULL where rotary_dim is 0.
 * Two sequences of one call must not share the page that either appends to.  q_out must not overlap k, v or the cache; q, k and v must not lie in places of
 * the cache that the call writes. */
int paella_kv_append_dims(const paella_kv_append_desc* desc, const paella_kv_cache* cache, const paella_kv_batch* batch, paella_launch_dims* dims);
int paella_kv_append_launch(const paella_kv_append_desc* desc, const paella_kv_cache* cache, const paella_kv_batch* batch, const void* q, const void* k,
                            const void* v, const float* q_weight, const float* k_weight, const float* inv_freq, void* q_out, void* stream,
                            uint32_t job_id, void* notifier);
/* The same where positions are not places in the cache, as after an eviction (paella_long_cache.h): new token j of sequence b is at position positions[b] + j (device data, [sequences]; NULL:
 * prefix_len + past[b] + j).  q_out must not overlap positions. */
int paella_kv_append_at_launch(const paella_kv_append_desc* desc, const paella_kv_cache* cache, const paella_kv_batch* batch, const int32_t* positions, const void* q,
                               const void* k, const void* v, const float* q_weight, const float* k_weight, const float* inv_freq, void* q_out, void* stream,
                               uint32_t job_id, void* notifier);

/* ---------------------------------------------------------------- attention over a shared prefix and each sequence's own tokens */

typedef struct paella_prefix_attention_plan {
    int dtype, heads, kv_heads, head_dim, page_size;
    int sequences, max_new, tokens, max_pages, prefix_len;
    float scale;                 /* of the products of queries and keys; set by the plan to 1 / sqrt(head_dim) where 0 is asked for */
    int prefix_rows, own_rows;   /* query rows (a head of a token each) of a workgroup over the prefix / over a sequence's own tokens */
    int prefix_splits, own_splits;  /* workgroups that share a row's keys, each */
    int stages;                  /* launches of a call: 2 where the parts of a row's keys are joined by a launch of their own */
    size_t workspace_bytes;      /* 0 where one workgroup does all of a row's keys */
    paella_launch_dims dims;
    double flops;                /* algorithmic, every sequence as long as its table: 4 * head_dim per query head and key */
    double bytes;                /* prefix once, own tokens as long as the tables, queries and outputs */
} paella_prefix_attention_plan;

/* out[t][h] = sum_i softmax_i(scale * q[t][h] . k_i[h / (heads / kv_heads)]) v_i over the prefix and the own tokens 0 .. past + j of
 * row t.  The prefix is walked once for all rows that share it, tile by tile.  Scores, maxima, sums and outputs are kept in 32 bits; of 16-bit types the weights
 * softmax_i are rounded to the type ahead of their product with v_i (which takes both in one type) and divided by the sum of the rounded ones, so a result
 * is off by one more half step of the type than its own rounding.  A row whose every key is excluded (pages outside the cache) gives zeros.  Keys and values in excluded places may hold anything; those of a sequence's later new tokens must be finite.
 * head_dim 64, 128 or 256 (PAELLA_ENOSUP otherwise).  Pure host arithmetic; of the cache and the batch, only the extents are looked at. */
int paella_prefix_attention_plan_make(const paella_kv_cache* cache, const paella_kv_batch* batch, int heads, float scale, paella_prefix_attention_plan* plan);
/* Launch shape of a stage with the register count and LDS of the kernel that is launched (the plan's own figures without a device). */
int paella_prefix_attention_dims(const paella_prefix_attention_plan* plan, int stage, paella_launch_dims* dims);
/* q: rows of heads * head_dim values, q_stride (a multiple of 8) from one row to the next; out: [tokens][heads][head_dim], not
 * overlapping q or the cache.  Cache and batch must have the plan's extents.  workspace: workspace_bytes, zero-filled once before its first use,
 * private to the request (launches that share it must not overlap); NULL where workspace_bytes is 0.  Issues all stages in order, the last
 * of which reports to `notifier`; PAELLA_ENOSUP for two stages on a queue that keeps no order: there the caller issues them one after
 * the other with paella_prefix_attention_launch_stage, the second once the first has finished. */
int paella_prefix_attention_launch(const paella_prefix_attention_plan* plan, const paella_kv_cache* cache, const paella_kv_batch* batch, const void* q,
                                   int64_t q_stride, void* out, void* workspace, void* stream, uint32_t job_id, void* notifier);
int paella_prefix_attention_launch_stage(const paella_prefix_attention_plan* plan, int stage, const paella_kv_cache* cache, const paella_kv_batch* batch,
                                         const void* q, int64_t q_stride, void* out, void* workspace, void* stream, uint32_t job_id, void* notifier);

/* ---------------------------------------------------------------- beam search */

typedef struct paella_beam_select_plan {
    int dtype;                   /* of the logits */
    int groups, beams, vocab, count;  /* beams <= 32, vocab <= 524288, count <= 64, beams * ceil(vocab / 8192) <= 1024 (PAELLA_ENOSUP beyond) */
    int values, splits;          /* logits per thread; workgroups per beam */
    size_t workspace_bytes;
    paella_launch_dims dims;
    double flops, bytes;
} paella_beam_select_plan;

/* Per group (request) the `count` best continuations of its beams, best first.  Continuation (w, t) is worth scores[w] + x[w][t] -
 * log(sum_u exp(x[w][u])); of equals the lower w * vocab + t comes first.  Worths are added and compared in 64 bits, the exponentials and their sums over up
 * to 8192 logits are 32-bit: within a beam the order is that of the logits, between beams that of worths whose logarithms carry such sums' roundings.  A beam with finished[w] != 0 has one continuation, pad_token, worth
 * scores[w]; its logits are not read.  A NaN logit counts as -inf, a row that holds +inf has no continuations, and what is worth an infinity or NaN is no
 * continuation: where fewer than `count` are left, the rest of the outputs are -inf, -1 and -1.  out_scores, out_parents (w), out_tokens (t):
 * [groups][count], overlapping neither each other nor any input; but out_scores may be scores where count == beams, and may overlap them where groups == 1.
 * logits: rows of vocab values, row_stride apart; finished (bytes) may be NULL.  workspace as for attention. */
int paella_beam_select_plan_make(int dtype, int groups, int beams, int vocab, int count, paella_beam_select_plan* plan);
int paella_beam_select_dims(const paella_beam_select_plan* plan, paella_launch_dims* dims);
int paella_beam_select_launch(const paella_beam_select_plan* plan, const void* logits, int64_t row_stride, const float* scores, const uint8_t* finished,
                              int pad_token, float* out_scores, int32_t* out_parents, int32_t* out_tokens, void* workspace, void* stream,
                              uint32_t job_id, void* notifier);

/* The paged caches of a group's beams after a selection.  Child c of group g continues beam p = parents[g][c], row r = g * beams + p of
 * tables and past: its row g * count + c of tables_out names the parent's full pages (shared, not copied) and then the page of its next
 * token -- for the first child of p the parent's half-filled page itself, for every further one spare[g * count + c], to which that page's tokens are
 * copied; where the parent's pages are all full, the spare page for every child.  Entries behind that page are left as they were; past_out = past[r]. A
 * parent outside 0 .. beams - 1 gives past_out 0 and an untouched row.  tables_out and past_out must overlap neither each other nor any input; the spare pages must be
 * named by no table.  Several layers: one call for each layer's cache with the same tables. */
typedef struct paella_beam_reorder_desc {
    int groups, beams, count, max_pages;
} paella_beam_reorder_desc;
int paella_beam_reorder_dims(const paella_beam_reorder_desc* desc, const paella_kv_cache* cache, paella_launch_dims* dims);
int paella_beam_reorder_launch(const paella_beam_reorder_desc* desc, const paella_kv_cache* cache, const int32_t* parents, const int32_t* past,
                               const int32_t* tables, const int32_t* spare, int32_t* tables_out, int32_t* past_out, void* stream, uint32_t job_id,
                               void* notifier);

#ifdef __cplusplus
}
#endif
#endif
