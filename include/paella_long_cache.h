/*
 * paella_long_cache.h -- C-ABI of the operators that keep a long paged cache (paella_decode.h) from being read whole and from being
 * kept whole, hand-written for gfx950: bounds of each page's keys, the pages whose bounds allow the largest products with a
 * query, attention over the pages that were picked, the attention weight that each token gathers, and the eviction of the tokens that
 * gathered least.  No counterpart in the reference, whose models are CNNs; conventions (stream or direct-dispatch queue, job_id and
 * notifier hooks, return codes, launch shapes, plans of several stages, workspaces) as in paella_decode.h.
 *
 * Pages are counted along a sequence: page e < P = ceil(prefix_len / page_size) is the shared prefix's prefix_table[e], page P + i the
 * sequence's own tables[sequence][i].  New token j of a sequence sees the prefix and the own tokens 0 .. past + j; a page is visible to it that
 * holds such a token.
 *
 * Device data that the host cannot check is checked where it is used, as there: pages outside the cache take no part, tokens beyond the
 * table are none, a negative length counts as 0, no access leaves the tensors whatever the numbers are; tables of 2^30 tokens and more are refused (PAELLA_ENOSUP).  What `starts` has to hold to is said there.
 */
#ifndef PAELLA_LONG_CACHE_H
#define PAELLA_LONG_CACHE_H

#include <stddef.h>
#include <stdint.h>

#include "paella_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------- bounds of a page's keys */

/* bounds [num_pages][kv_heads][2][head_dim], of the cache's type: the least and the largest value that a page's keys have in each dimension, over the page's tokens
 * up to the last new one.  Of every page that holds a new token of the batch both rows are made anew from all of them, so what was there does not matter: a page that drafts
 * were taken back from, or that was copied, needs no more than its next call.  (A prefix: a sequence of its own, with past 0 and max_new as long as it.)  A NaN counts as no value; bounds of a page without
 * any are +inf and -inf.  Two sequences of one call must not share a page that either appends to.  bounds: on a 16-byte boundary, not over the cache or the batch's
 * tensors. */
int paella_page_bounds_dims(const paella_kv_cache* cache, const paella_kv_batch* batch, paella_launch_dims* dims);
int paella_page_bounds_launch(const paella_kv_cache* cache, const paella_kv_batch* batch, void* bounds, void* stream, uint32_t job_id, void* notifier);

/* ---------------------------------------------------------------- the pages that a new token reads */

typedef struct paella_page_select_plan {
    int dtype, heads, kv_heads, head_dim, page_size;
    int sequences, max_new, tokens, max_pages, prefix_len;
    int count, first, last;      /* pages of a new token and key head; of them the sequence's first and last visible ones, whatever their bounds */
    int splits;                  /* workgroups that share a row's pages */
    int stages;                  /* launches of a call */
    size_t workspace_bytes;
    size_t zero_bytes;           /* the first bytes of the workspace that have to be 0 ahead of its first call; what the others hold does not matter */
    paella_launch_dims dims;
    double flops, bytes;         /* algorithmic, every sequence as long as its table */
} paella_page_select_plan;

/* pages [tokens][kv_heads][count]: the visible pages with the largest worth, ascending, -1 behind the last where there are fewer than count.  Worth of a page: the largest, over
 * the query heads of the key head, of sum_d max(q_d low_d, q_d high_d), which no product of the query with a key between the bounds exceeds.  The first `first` and the last `last`
 * visible pages (last >= 1) are taken whatever they are worth; of equals the lower page is taken, and a worth that is no number counts as the largest.  Worths are computed and compared in 64 bits.
 * Bounds have to be those of the keys (paella_page_bounds_launch).  head_dim 64, 128 or 256 (PAELLA_ENOSUP otherwise). */
int paella_page_select_plan_make(const paella_kv_cache* cache, const paella_kv_batch* batch, int heads, int count, int first, int last, paella_page_select_plan* plan);
int paella_page_select_dims(const paella_page_select_plan* plan, int stage, paella_launch_dims* dims);
/* q as for attention; of the cache only the extents are read.  pages and the workspace must not overlap q, bounds, the cache, the batch's tensors or each other.  Stages and queues as for
 * paella_prefix_attention_launch, and the workspace but for the plan's zero_bytes, here and below. */
int paella_page_select_launch(const paella_page_select_plan* plan, const paella_kv_cache* cache, const paella_kv_batch* batch, const void* q, int64_t q_stride,
                              const void* bounds, int32_t* pages, void* workspace, void* stream, uint32_t job_id, void* notifier);
int paella_page_select_launch_stage(const paella_page_select_plan* plan, int stage, const paella_kv_cache* cache, const paella_kv_batch* batch, const void* q,
                                    int64_t q_stride, const void* bounds, int32_t* pages, void* workspace, void* stream, uint32_t job_id, void* notifier);

/* ---------------------------------------------------------------- attention over picked pages */

typedef struct paella_page_attention_plan {
    int dtype, heads, kv_heads, head_dim, page_size;
    int sequences, max_new, tokens, max_pages, prefix_len;
    int count;                   /* entries of a row's list */
    float scale;                 /* set by the plan to 1 / sqrt(head_dim) where 0 is asked for */
    int splits;                  /* workgroups that share a list */
    int stages;                  /* 2 where their parts are joined by a launch of its own */
    size_t workspace_bytes;      /* 0 where one workgroup does a list */
    size_t zero_bytes;
    paella_launch_dims dims;
    double flops, bytes;         /* algorithmic, lists full and of different pages */
} paella_page_attention_plan;

/* out[t][h] = sum_i softmax_i(scale * q[t][h] . k_i) v_i over the tokens that row t sees of the pages in pages[t][h / (heads / kv_heads)] (int32 [tokens][kv_heads][count], as
 * paella_page_select writes it; entries outside the sequence's pages, and pages outside the cache, are passed over wherever they stand, and a page listed twice counts twice).  Scores, maxima, sums and outputs are kept in 32 bits;
 * of 16-bit types a weight is taken as the sum of two numbers of the type, divided by the sum of those, so that a result is off by little more than its own rounding; a row without any token gives zeros, and what lies in places that a row does not see may be anything.  head_dim 64, 128 or 256. */
int paella_page_attention_plan_make(const paella_kv_cache* cache, const paella_kv_batch* batch, int heads, int count, float scale, paella_page_attention_plan* plan);
int paella_page_attention_dims(const paella_page_attention_plan* plan, int stage, paella_launch_dims* dims);
int paella_page_attention_launch(const paella_page_attention_plan* plan, const paella_kv_cache* cache, const paella_kv_batch* batch, const void* q, int64_t q_stride,
                                 const int32_t* pages, void* out, void* workspace, void* stream, uint32_t job_id, void* notifier);
int paella_page_attention_launch_stage(const paella_page_attention_plan* plan, int stage, const paella_kv_cache* cache, const paella_kv_batch* batch, const void* q,
                                       int64_t q_stride, const int32_t* pages, void* out, void* workspace, void* stream, uint32_t job_id, void* notifier);

/* ---------------------------------------------------------------- the attention weight that tokens gather */

typedef struct paella_key_weights_plan {
    int dtype, heads, kv_heads, head_dim, page_size;
    int sequences, max_new, tokens, max_pages, prefix_len;
    float scale;
    int splits, own_splits;      /* workgroups that share a sequence's keys in the first and in the second stage */
    int stages;
    size_t workspace_bytes;
    size_t zero_bytes;
    paella_launch_dims dims;
    double flops, bytes;
} paella_key_weights_plan;

/* weights [sequences][kv_heads][max_pages * page_size], float, on a 16-byte boundary: to each own token i of a sequence is added sum softmax_i(scale * q[t][h] . k) over the sequence's new tokens t that
 * see it and the query heads h of the key head, the softmax taken over the prefix and the own tokens that t sees.  The sequence's new tokens (i >= past) start from 0 whatever was there; places behind them, and all of a sequence
 * without new tokens, are left as they were.  Everything is kept in 32 bits; sums are taken in the same order in every run, and
 * the old weight is added once, to the sum of the call's.  The workspace holds the scores of all own tokens where a sequence has 16 rows (new tokens by heads of a key head)
 * at most and they are 1 GB at most by the tables' width, and those sums, 4 bytes a place, where it has many.  head_dim 64, 128 or 256. */
int paella_key_weights_plan_make(const paella_kv_cache* cache, const paella_kv_batch* batch, int heads, float scale, paella_key_weights_plan* plan);
int paella_key_weights_dims(const paella_key_weights_plan* plan, int stage, paella_launch_dims* dims);
int paella_key_weights_launch(const paella_key_weights_plan* plan, const paella_kv_cache* cache, const paella_kv_batch* batch, const void* q, int64_t q_stride,
                              float* weights, void* workspace, void* stream, uint32_t job_id, void* notifier);
int paella_key_weights_launch_stage(const paella_key_weights_plan* plan, int stage, const paella_kv_cache* cache, const paella_kv_batch* batch, const void* q,
                                    int64_t q_stride, float* weights, void* workspace, void* stream, uint32_t job_id, void* notifier);

/* ---------------------------------------------------------------- eviction */

typedef struct paella_kv_evict_desc {
    int sequences, max_pages;
    int keep;                    /* tokens that stay of a longer sequence, for each key head */
    int first, recent;           /* of them its first and its last ones, whatever they weigh; first + recent <= keep */
} paella_kv_evict_desc;

/* Of each sequence with past > keep every key head keeps its first `first` tokens, its last `recent` ones and the heaviest of those between (of equals the lower one; a NaN weighs least), which move,
 * in their order, to its places 0 .. keep - 1: keys, values and weights.  kept [sequences][kv_heads][keep]: which they were (0, 1, .. for a shorter sequence, -1 behind its last token); past_out = min(past, keep), which
 * may be past.  Heads keep different tokens: rotate keys ahead of the cache (paella_kv_append_launch does), and give later tokens their positions (paella_kv_append_at_launch).  What lay behind the places kept is left as it
 * was, the pages there are the caller's again.  Bounds of the pages have to be made anew.  No page may be named twice, by one sequence or two, and none by a prefix that is still used; a token whose page lies outside the cache is neither read
 * nor written.  Two launches (stages); on a queue that keeps no order the caller issues them one after the other.  kept and past_out must overlap neither each other nor weights, tables or the cache. */
int paella_kv_evict_dims(const paella_kv_evict_desc* desc, const paella_kv_cache* cache, int stage, paella_launch_dims* dims);
int paella_kv_evict_launch(const paella_kv_evict_desc* desc, const paella_kv_cache* cache, float* weights, const int32_t* past, const int32_t* tables, int32_t* kept,
                           int32_t* past_out, void* stream, uint32_t job_id, void* notifier);
int paella_kv_evict_launch_stage(const paella_kv_evict_desc* desc, int stage, const paella_kv_cache* cache, float* weights, const int32_t* past, const int32_t* tables,
                                 int32_t* kept, int32_t* past_out, void* stream, uint32_t job_id, void* notifier);

#ifdef __cplusplus
}
#endif
#endif
