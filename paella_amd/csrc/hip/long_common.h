#pragma once
// What the operators over long caches (paella_long_cache.h) share beyond decode_common.h: a sequence's new tokens, the pages along a sequence, and the host's
// checks of plans.

#include "decode_common.h"
#include "paella_long_cache.h"

namespace paella {

struct NewTokens {
    int first, count, past;  // rows, and own tokens ahead of them
};

// Of sequence `seq`, the same for the whole wave.
__device__ __forceinline__ NewTokens new_tokens(const int* __restrict__ starts, const int* __restrict__ past, int seq, int max_new, int tokens) {
    NewTokens n{seq * max_new, max_new, 0};
    if (starts) {
        n.first = min(max(__builtin_amdgcn_readfirstlane(starts[seq]), 0), tokens);
        n.count = max(min(min(__builtin_amdgcn_readfirstlane(starts[seq + 1]), tokens) - n.first, max_new), 0);
    }
    n.past = max(__builtin_amdgcn_readfirstlane(past[seq]), 0);
    return n;
}

// Two floats in one store that goes through to memory.
__device__ __forceinline__ void put_pair(f32x2* p, float a, float b) {
    __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), (unsigned long long)as_word(b) << 32 | as_word(a), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Own pages that new token j of a sequence sees.
__device__ __forceinline__ int own_pages(int past, int j, Divisor page_size, int max_pages) {
    return (int)min(divide((unsigned)max(past, 0) + (unsigned)j, page_size).q + 1, (unsigned)max_pages);
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline bool over_batch(const paella_kv_batch* b, int page_size, const void* at, double bytes) {
    const double n = b->sequences;
    return overlap(b->past, 4 * n, at, bytes) || overlap(b->tables, 4 * n * b->max_pages, at, bytes) || (b->starts && overlap(b->starts, 4 * n + 4, at, bytes)) ||
           (b->prefix_len && b->prefix_table && overlap(b->prefix_table, 4.0 * ceil_div(b->prefix_len, page_size), at, bytes));
}

inline bool keeps_no_order(void* stream) {
    const DirectQueue* const queue = direct_queue_lookup(stream);
    return queue && !direct_queue_ordered(queue);
}

// The extents that all plans hold.
template <typename Plan>
void plan_extents(Plan* p, const paella_kv_cache* c, const paella_kv_batch* b, int heads) {
    p->dtype = c->dtype; p->heads = heads; p->kv_heads = c->kv_heads; p->head_dim = c->head_dim; p->page_size = c->page_size;
    p->sequences = b->sequences; p->max_new = b->max_new; p->tokens = b->tokens; p->max_pages = b->max_pages; p->prefix_len = b->prefix_len;
}

template <typename Plan>
bool planned_extents_ok(const Plan* p) {
    if (p->dtype < PAELLA_F32 || p->dtype > PAELLA_F16 || p->page_size <= 0 || p->page_size % 8 || p->sequences <= 0 || p->max_new <= 0 || p->max_new >= 1 << 30 || p->tokens <= 0 ||
        p->max_pages <= 0 || p->prefix_len < 0 || p->prefix_len >= 1 << 30 || p->heads <= 0 || p->kv_heads <= 0 || p->heads % p->kv_heads || p->head_dim <= 0)
        return false;
    if ((double)p->kv_heads * p->page_size * p->head_dim * element_bytes(p->dtype) >= 2147483648.0) return false;
    // 32-bit offsets of a call's rows and 32-bit numbers of own tokens
    return (double)p->tokens * p->heads * p->head_dim < 1073741824.0 && (double)p->max_new * p->heads < 1073741824.0 && (double)p->max_pages * p->page_size < 1073741824.0 &&
           (double)p->sequences * p->max_pages < 2147483648.0 && (double)p->sequences * p->max_new < 2147483648.0;
}

// Whether a cache and a batch are what a plan was made for, with everything that a launch reads.
template <typename Plan>
bool planned_for(const Plan* p, const paella_kv_cache* c, const paella_kv_batch* b) {
    return cache_ok(c) && batch_ok(b) && c->dtype == p->dtype && c->kv_heads == p->kv_heads && c->head_dim == p->head_dim && c->page_size == p->page_size &&
           b->sequences == p->sequences && b->max_new == p->max_new && b->tokens == p->tokens && b->max_pages == p->max_pages && b->prefix_len == p->prefix_len &&
           (!b->prefix_len || b->prefix_table);
}

}  // namespace paella
