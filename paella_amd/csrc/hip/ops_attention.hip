// Attention of a decoding step: planning and launch (the kernels: prefix_attention.h).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "prefix_attention.h"

namespace {

using namespace paella;

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

AttentionKernel kernel_of(const paella_prefix_attention_plan* p) {
    const int rp = p->prefix_rows, ro = p->own_rows;
    return p->dtype == PAELLA_F32 ? attention_kernel_f32(p->head_dim, rp, ro)
                                  : p->dtype == PAELLA_BF16 ? attention_kernel_bf16(p->head_dim, rp, ro) : attention_kernel_f16(p->head_dim, rp, ro);
}

AttentionKernel join_of(const paella_prefix_attention_plan* p) {
    return p->dtype == PAELLA_F32 ? attention_join_f32(p->head_dim) : p->dtype == PAELLA_BF16 ? attention_join_bf16(p->head_dim) : attention_join_f16(p->head_dim);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Grid {
    int64_t prefix_tiles, own_tiles, prefix_items, all;
};

Grid grid_of(const paella_prefix_attention_plan* p) {
    const int64_t per_kv = p->heads / p->kv_heads;
    Grid g;
    g.prefix_tiles = p->prefix_len ? ceil_div(p->tokens * per_kv, p->prefix_rows) : 0;
    g.own_tiles = ceil_div(p->max_new * per_kv, p->own_rows);
    g.prefix_items = g.prefix_tiles * p->kv_heads * p->prefix_splits;
    g.all = g.prefix_items + p->sequences * g.own_tiles * p->kv_heads * p->own_splits;
    return g;
}

bool extents_ok(const paella_prefix_attention_plan* p) {
    if (p->heads <= 0 || p->kv_heads <= 0 || p->heads % p->kv_heads) return false;
    // 32-bit offsets of outputs and parts
    return (double)p->tokens * p->heads * p->head_dim < 1073741824.0 && (double)p->max_new * p->heads < 1073741824.0;
}

bool plan_ok(const paella_prefix_attention_plan* p) {
    if (!p || p->dtype < PAELLA_F32 || p->dtype > PAELLA_F16 || p->page_size <= 0 || p->page_size % 8 || p->sequences <= 0 || p->max_new <= 0 || p->tokens <= 0 ||
        p->max_pages <= 0 || p->prefix_len < 0 || !(p->scale >= 0.f) || !(p->scale < INFINITY) || !extents_ok(p) || !kernel_of(p))
        return false;
    if (p->own_splits <= 0 || p->own_splits > 64 || p->prefix_splits < 0 || p->prefix_splits > 64 || (p->prefix_splits > 0) != (p->prefix_len > 0)) return false;
    const Grid g = grid_of(p);
    return (double)g.all <= kMostWorkgroups;
}

// Whether the workgroup that arrives last at a row joins it, or a launch of its own does: where its lanes have all of the outputs at once and request all parts
// together.  (Rows of heads of 128 in 5 parts, twice as many as that, 12.3 us against 10.5 with the other launch, 12 in 21 parts 16.2 against 10.8; 2 sequences of 4
// rows in 8 parts 9.8 against 10.3.)
int stages_of(const paella_prefix_attention_plan* p) {
    const int parts = p->prefix_splits + p->own_splits;
    if (parts == 1) return 1;
    const int64_t per_kv = p->heads / p->kv_heads;
    const int64_t own = std::min<int64_t>(p->own_rows, p->max_new * per_kv), shared = p->prefix_splits ? std::min<int64_t>(p->prefix_rows, p->tokens * per_kv) : 0;
    return std::max(own, shared) * p->head_dim / 4 <= 256 && parts <= kJoined ? 1 : 2;
}

size_t counter_pitch(const paella_prefix_attention_plan* p) { return up256((size_t)p->tokens * (p->heads / p->kv_heads) * 4) / 4; }

size_t workspace_of(const paella_prefix_attention_plan* p) {
    const size_t parts = (size_t)p->prefix_splits + p->own_splits, rows = (size_t)p->tokens * p->heads;
    return parts == 1 ? 0 : p->kv_heads * counter_pitch(p) * 4 + up256(parts * rows * 8) + parts * rows * p->head_dim * 4;
}

}  // namespace

extern "C" {

int paella_prefix_attention_plan_make(const paella_kv_cache* c, const paella_kv_batch* b, int heads, float scale, paella_prefix_attention_plan* p) {
    if (!p || !cache_extents_ok(c) || !batch_extents_ok(b) || heads <= 0 || heads % c->kv_heads || !(scale >= 0.f) || !(scale < INFINITY)) return PAELLA_EINVAL;
    *p = paella_prefix_attention_plan{};
    p->dtype = c->dtype; p->heads = heads; p->kv_heads = c->kv_heads; p->head_dim = c->head_dim; p->page_size = c->page_size;
    p->sequences = b->sequences; p->max_new = b->max_new; p->tokens = b->tokens; p->max_pages = b->max_pages; p->prefix_len = b->prefix_len;
    p->scale = scale > 0.f ? scale : 1.f / std::sqrt((float)c->head_dim);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return PAELLA_ENOSUP;
    if (!extents_ok(p)) return PAELLA_ENOSUP;
    const int64_t per_kv = heads / c->kv_heads, size = element_bytes(c->dtype), row_bytes = c->head_dim * size;
    const int step = size == 4 ? 16 : 32;
    // Rows of a workgroup.  Where a key head has few, 16: its waves split the keys.  Else 64 or 128: each wave has rows of its own, the keys are read once
    // for all of them.  That is no gain up to some number of steps by 16 rows, where latency counts.  fp32, heads of 128, by 16 rows / by 64: 4 key heads, 96 rows each over 1600
    // keys, 192 over 1200 / 1500 / 2200 / 3000 (2400, 3600 / 4512 / 6624 / 9024 steps) 15.7 / 18.7 us, 19.6 / 20.4, 20.8 / 21.0, 23.2 / 21.7, 32.0 / 23.1; 96 over 3000 (4512)
    // 21.2 / 20.2.  bf16, by 16 / by 128: 96 over 1600, 192 over 1200 / 2000 / 3000 (1200, 1824 / 3024 / 4512) 10.4 / 15.3, 12.6 / 14.6, 13.7 / 16.2, 16.8 / 16.6, but 8 key
    // heads, 36 rows over 3000 / 8000 (2256 / 6000) 12.9 / 12.3 and 21.2 / 17.0.  Heads of 256 hold few keys' loads beside 16 rows: 24 rows over 187 keys 16.8 against 13.0.
    const bool small_heads = c->head_dim <= 128;
    auto rows = [&](int64_t n) { return n <= 64 || !small_heads || row_bytes > 256 ? 64 : 128; };
    const int64_t own = std::min(b->max_new, b->tokens) * per_kv, shared = b->tokens * per_kv;  // no sequence has more than all rows, whatever max_new leaves room for
    p->own_rows = own <= (small_heads ? 32 : 16) ? 16 : rows(own);
    p->prefix_rows = p->own_rows;
    if (p->prefix_len) {
        const double steps = (double)ceil_div(shared, 16) * c->kv_heads * ceil_div(p->prefix_len, step);
        const bool few = shared <= 16 || (small_heads && steps <= (size == 4 ? 4500 : 2048));
        p->prefix_rows = few && p->own_rows == 16 ? 16 : rows(shared);
    }
    if (p->own_rows == 64 && p->prefix_rows == 128) p->own_rows = 128;
    // A row's keys are shared by so many workgroups that three are there for each compute unit, or eight where many sequences' lengths have to even out (64
    // sequences of up to 4000 tokens in 2 / 3 / 4 parts, beside a prefix, 190 / 186 / 182 us; 32 of 1000 and 5 new in 2 / 3 / 4 / 6 49 / 45 / 44 / 49; but 10 of 1500 in
    // 7 / 10 15 / 19).  A workgroup of 16 rows has 256 keys at least (28 rows a key head in fp32 over 3000 keys in 12 / 24 parts 18.4 / 23.7 us), one of more eight steps
    // (96 rows in fp32 over 3000 in 12 / 24 33 / 24), or, of few workgroups, a step for each wave as
    // long as the parts are at most seven (one step against two, 4 sequences over 130 + 100 keys in fp32: 7.8 against 8.9 us).
    auto splits = [&](int64_t want, int64_t undivided, int64_t keys, int least) {
        int64_t n = ceil_div(keys, least);
        if (undivided < 128) n = std::max(n, std::min<int64_t>(ceil_div(keys, 4 * step), 7));
        n = std::min(want, n);
        return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
    };
    const int64_t own_keys = (int64_t)b->max_pages * c->page_size;
    p->own_splits = 1;
    Grid g = grid_of(p);
    const int64_t undivided = b->sequences * g.own_tiles * c->kv_heads;
    p->own_splits = splits(ceil_div(undivided < 128 ? 768 : 2048, undivided), undivided, own_keys, 256);
    if (p->prefix_len) {
        // Workgroups over the prefix start first.  Those of many rows are bound by the products, those over own tokens by memory: one of the first to a
        // compute unit, the second beside it, is best where the own tokens are half as many as the prefix's, by tiles, or more; where they are fewer, two, if that leaves
        // each 512 keys (of heads of 128); a unit holds one with heads of 256 anyway.  One more than fits them all costs a whole round.  (bf16, heads of 128, 256 against 512 workgroups:
        // 64 sequences over 65536 + 4000 / 2000 / 1000 / 500 keys 186 / 129 / 118 / 120 against 216 / 145 / 117 / 105 us, 32 of up to 5 tokens over 8190 + 1000
        // / 300 39 / 34 against 47 / 38; 7 over 20000 + 60 25 against 28, heads of 64, 74 over 11439 + 108 28 against 25; 528 in place of 504: 39.7 against 37.8; fp32, 48 over 3000 + 60, 252 in place of 288: 23
        // against 30; heads of 256 with hardly any own tokens 32 against 39.)
        const int64_t tiles = g.prefix_tiles * c->kv_heads;
        const bool beside = 2.0 * b->sequences * own_keys >= (double)g.prefix_tiles * b->prefix_len;
        const bool two = c->head_dim <= 128 && !beside && (double)b->prefix_len * tiles >= 2048.0 * c->head_dim;
        p->prefix_splits = splits(p->prefix_rows > 16 ? (two ? 512 : 256) / tiles : ceil_div(768, tiles), tiles, b->prefix_len, p->prefix_rows > 16 ? 8 * step : 256);
    }
    if (!plan_ok(p)) return PAELLA_ENOSUP;
    g = grid_of(p);
    p->workspace_bytes = workspace_of(p);
    p->stages = stages_of(p);
    set_launch_dims(&p->dims, (unsigned)g.all, 256, 0, 256);
    const double keys = (double)b->max_pages * c->page_size;
    p->flops = 4.0 * c->head_dim * b->tokens * heads * (p->prefix_len + keys);
    p->bytes = 2.0 * (p->prefix_len + b->sequences * keys) * c->kv_heads * row_bytes + 2.0 * b->tokens * heads * row_bytes;
    return 0;
}

int paella_prefix_attention_dims(const paella_prefix_attention_plan* p, int stage, paella_launch_dims* dims) {
    if (!plan_ok(p) || !dims || stage < 0 || stage >= stages_of(p)) return PAELLA_EINVAL;
    if (stage) set_launch_dims(dims, (unsigned)ceil_div((int64_t)p->tokens * p->heads, kJoinRows / p->head_dim), 256, 0, 64);
    else set_launch_dims(dims, (unsigned)grid_of(p).all, 256, 0, 256);
    loaded_dims((const void*)(stage ? join_of(p) : kernel_of(p)), dims);
    return 0;
}

int paella_prefix_attention_launch_stage(const paella_prefix_attention_plan* p, int stage, const paella_kv_cache* c, const paella_kv_batch* b, const void* q,
                                         int64_t q_stride, void* out, void* workspace, void* stream, uint32_t job_id, void* notifier) {
    if (!plan_ok(p) || !cache_ok(c) || !batch_ok(b) || !q || !out || stage < 0 || stage >= stages_of(p)) return PAELLA_EINVAL;
    if (c->dtype != p->dtype || c->kv_heads != p->kv_heads || c->head_dim != p->head_dim || c->page_size != p->page_size || b->sequences != p->sequences ||
        b->max_new != p->max_new || b->tokens != p->tokens || b->max_pages != p->max_pages || b->prefix_len != p->prefix_len)
        return PAELLA_EINVAL;
    if (p->prefix_len && !b->prefix_table) return PAELLA_EINVAL;
    const int64_t size = element_bytes(c->dtype), row = (int64_t)p->heads * c->head_dim;
    if (q_stride < row || q_stride % 8 || (((uintptr_t)q | (uintptr_t)out) & 15)) return PAELLA_EINVAL;
    if (overlap(q, ((double)(b->tokens - 1) * q_stride + row) * size, out, (double)b->tokens * row * size)) return PAELLA_EINVAL;
    const size_t need = workspace_of(p);
    if (need && (!workspace || ((uintptr_t)workspace & 15))) return PAELLA_EINVAL;
    const double out_bytes = (double)b->tokens * row * size;
    if (over_cache(c, out, out_bytes)) return PAELLA_EINVAL;
    if (need && (over_cache(c, workspace, (double)need) || overlap(out, out_bytes, workspace, (double)need) ||
                 rows_overlap(q, b->tokens, q_stride * size, row * size, workspace, (double)need)))
        return PAELLA_EINVAL;
    const Grid g = grid_of(p);
    AttentionArgs a;
    a.q = (const char*)q; a.k_cache = (const char*)c->k; a.v_cache = (const char*)c->v; a.out = (char*)out;
    a.starts = b->starts; a.past = b->past; a.tables = b->tables; a.prefix_table = b->prefix_table;
    a.q_stride = q_stride * size;
    a.sequences = b->sequences; a.max_new = b->max_new; a.tokens = b->tokens; a.max_pages = b->max_pages; a.prefix_len = b->prefix_len;
    a.prefix_pages = (int)ceil_div(b->prefix_len, c->page_size);
    a.heads = p->heads; a.page_size = c->page_size; a.num_pages = c->num_pages;
    a.kv_heads = divisor((unsigned)p->kv_heads); a.per_kv = divisor((unsigned)(p->heads / p->kv_heads)); a.page_blocks = divisor((unsigned)c->page_size / 8);
    a.scale_log2 = p->scale * 1.44269504088896340736f;
    const int step = size == 4 ? 16 : 32;  // keys
    a.eight_tiles = divisor((unsigned)g.prefix_tiles * 8); a.prefix_splits = divisor((unsigned)p->prefix_splits);
    a.own_tiles = divisor((unsigned)g.own_tiles); a.own_splits = divisor((unsigned)p->own_splits);
    a.prefix_per = p->prefix_splits ? (int)ceil_div(ceil_div(p->prefix_len, step), p->prefix_splits) : 0;
    a.prefix_pairs = p->kv_heads * p->prefix_splits;
    a.prefix_items = (unsigned)g.prefix_items;
    const size_t parts = (size_t)p->prefix_splits + p->own_splits, rows = (size_t)p->tokens * p->heads;
    a.counters = need && stages_of(p) == 1 ? (unsigned*)workspace : nullptr;
    a.counter_pitch = (unsigned)counter_pitch(p);
    a.ml = need ? (f32x2*)((char*)workspace + p->kv_heads * counter_pitch(p) * 4) : nullptr;
    a.acc = need ? (float*)((char*)a.ml + up256(parts * rows * 8)) : nullptr;
    a.job_id = job_id; a.notifier = (Notifier*)notifier;
    const unsigned grid = stage ? (unsigned)ceil_div((int64_t)rows, kJoinRows / p->head_dim) : (unsigned)g.all;
    launch(stage ? join_of(p) : kernel_of(p), dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

int paella_prefix_attention_launch(const paella_prefix_attention_plan* p, const paella_kv_cache* c, const paella_kv_batch* b, const void* q, int64_t q_stride,
                                   void* out, void* workspace, void* stream, uint32_t job_id, void* notifier) {
    if (!plan_ok(p)) return PAELLA_EINVAL;
    const int stages = stages_of(p);
    if (stages > 1) {
        const DirectQueue* queue = direct_queue_lookup(stream);
        if (queue && !direct_queue_ordered(queue)) return PAELLA_ENOSUP;
        if (int rc = paella_prefix_attention_launch_stage(p, 0, c, b, q, q_stride, out, workspace, stream, job_id, nullptr)) return rc;
    }
    return paella_prefix_attention_launch_stage(p, stages - 1, c, b, q, q_stride, out, workspace, stream, job_id, notifier);
}

}  // extern "C"
