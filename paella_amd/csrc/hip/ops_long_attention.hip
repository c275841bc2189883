// Attention over picked pages and the attention weight that tokens gather: planning and launch (the kernels: long_attention.h).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "long_attention.h"

namespace {

using namespace paella;

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
bool scale_ok(float scale) { return scale >= 0.f && scale < INFINITY; }
bool dim_ok(int dim) { return dim == 64 || dim == 128 || dim == 256; }

// ------------------------------------------------------------------------------------------ attention over picked pages

using PagePlan = paella_page_attention_plan;

PageAttentionKernel kernel_of(const PagePlan* p) {
    return p->dtype == PAELLA_F32 ? page_attention_f32(p->head_dim) : p->dtype == PAELLA_BF16 ? page_attention_bf16(p->head_dim) : page_attention_f16(p->head_dim);
}
AttentionKernel join_of(const PagePlan* p) {
    return p->dtype == PAELLA_F32 ? attention_join_f32(p->head_dim) : p->dtype == PAELLA_BF16 ? attention_join_bf16(p->head_dim) : attention_join_f16(p->head_dim);
}

int64_t tiles_of(const PagePlan* p) { return ceil_div(p->heads / p->kv_heads, 16); }
int64_t grid_of(const PagePlan* p) { return p->tokens * tiles_of(p) * p->kv_heads * p->splits; }

bool plan_ok(const PagePlan* p) {
    return p && planned_extents_ok(p) && dim_ok(p->head_dim) && p->count > 0 && p->count < 1 << 24 && p->scale > 0.f && scale_ok(p->scale) && p->splits > 0 && p->splits <= 64 &&
           (double)p->tokens * tiles_of(p) * p->kv_heads * p->splits <= kMostWorkgroups && (double)p->tokens * p->kv_heads * p->count < 2147483648.0;
}

// As in the decoding step's attention: the workgroup that arrives last joins a row's parts where its lanes have all outputs at once and request all parts together.
int stages_of(const PagePlan* p) {
    if (p->splits == 1) return 1;
    return std::min<int64_t>(16, p->heads / p->kv_heads) * p->head_dim / 4 <= 256 && p->splits <= kJoined ? 1 : 2;
}

size_t counters_of(const PagePlan* p) { return stages_of(p) == 1 ? up256((size_t)p->tokens * tiles_of(p) * p->kv_heads * 32 * 4) : 0; }
size_t workspace_of(const PagePlan* p) {
    const size_t parts = p->splits, rows = (size_t)p->tokens * p->heads;
    return parts == 1 ? 0 : counters_of(p) + up256(parts * rows * 8) + parts * rows * p->head_dim * 4;
}

// ------------------------------------------------------------------------------------------ the weight that tokens gather

using WeighPlan = paella_key_weights_plan;

// Few rows: the first pass stores the scores, which the second one reads in place of the keys.  That pays while a token's scores, written and read, 8 bytes a row, are less than its key, and costs nothing where they
// are as much: a tile of 16 rows and a key of 128 bytes.  (32 sequences of 4096 to 8192 tokens, 8 key heads, stored / keys read again, us: bf16 heads of 64, 4 / 8 / 16 rows 48 / 56 / 77, 77; of 128 99 / 105 / 119,
// 147; of 256 180 / 185 / 200, 309; fp32 heads of 64 95 / 103 / 124, 187; of 256 322 / 337 / 357, 653.  A small call, 4 bf16 sequences of 4096 tokens of 2 heads of 64, 16 rows, 12.0 / 11.5.)  Scores go by the
// tables' width, the plan not knowing the lengths, and each stream that the plan is used on has its own: up to 1 GB in all, where 32 sequences of 65536 tokens, 16 rows of bf16 heads of 128, take 970 / 1252.
constexpr double kMostScores = 1073741824.0;
bool few_rows(const WeighPlan* p) {
    const int64_t rows = (int64_t)std::min(p->max_new, p->tokens) * (p->heads / p->kv_heads);
    return rows <= 16 && 4.0 * p->sequences * p->kv_heads * (double)rows * p->max_pages * p->page_size <= kMostScores;
}
int chunk_rows(const WeighPlan* p) {
    if (few_rows(p)) return 16;
    return 16 * std::min(8, 32768 / (16 * p->head_dim * element_bytes(p->dtype)));
}
int64_t chunks_of(const WeighPlan* p) { return ceil_div((int64_t)std::min(p->max_new, p->tokens) * (p->heads / p->kv_heads), chunk_rows(p)); }

WeighKernel kernel_of(const WeighPlan* p, int stage) {
    const bool few = few_rows(p);
    const int d = p->head_dim;
    if (stage) return p->dtype == PAELLA_F32 ? key_weights_f32(d, few) : p->dtype == PAELLA_BF16 ? key_weights_bf16(d, few) : key_weights_f16(d, few);
    return p->dtype == PAELLA_F32 ? key_sums_f32(d, few) : p->dtype == PAELLA_BF16 ? key_sums_bf16(d, few) : key_sums_f16(d, few);
}

int64_t grid_of(const WeighPlan* p, int stage) { return stage ? (int64_t)p->sequences * p->kv_heads * p->own_splits : p->sequences * chunks_of(p) * p->kv_heads * p->splits; }

bool plan_ok(const WeighPlan* p) {
    return p && planned_extents_ok(p) && dim_ok(p->head_dim) && p->scale > 0.f && scale_ok(p->scale) && p->splits > 0 && p->splits <= 64 && p->own_splits > 0 &&
           (double)p->prefix_len + (double)p->max_pages * p->page_size < 1073741824.0 - 1048576.0 && p->page_size <= 1 << 20 &&
           (double)p->sequences * chunks_of(p) * p->kv_heads * p->splits <= kMostWorkgroups && (double)p->sequences * p->kv_heads * p->own_splits <= kMostWorkgroups;
}

size_t parts_of(const WeighPlan* p) { return up256((size_t)p->splits * p->tokens * p->heads * 8); }
int score_rows(const WeighPlan* p) { return few_rows(p) ? std::min(p->max_new, p->tokens) * (p->heads / p->kv_heads) : 0; }
// Floats that are kept of an own token: its scores, or the sum over the rows so far (as much memory as the weights themselves).
int kept_of(const WeighPlan* p) { return few_rows(p) ? score_rows(p) : chunks_of(p) > 1 ? 1 : 0; }
size_t workspace_of(const WeighPlan* p) { return parts_of(p) + (size_t)p->sequences * p->kv_heads * kept_of(p) * p->max_pages * p->page_size * 4; }

}  // namespace

extern "C" {

int paella_page_attention_plan_make(const paella_kv_cache* c, const paella_kv_batch* b, int heads, int count, float scale, paella_page_attention_plan* p) {
    if (!p || !cache_extents_ok(c) || !batch_extents_ok(b) || heads <= 0 || heads % c->kv_heads || count <= 0 || !scale_ok(scale)) return PAELLA_EINVAL;
    *p = paella_page_attention_plan{};
    plan_extents(p, c, b, heads);
    p->count = count;
    p->scale = scale > 0.f ? scale : 1.f / std::sqrt((float)c->head_dim);
    p->splits = 1;
    if (!plan_ok(p)) return PAELLA_ENOSUP;
    const int64_t undivided = grid_of(p), keys = (int64_t)count * c->page_size, pages = std::min<int64_t>(count, ceil_div(b->prefix_len, c->page_size) + b->max_pages);
    // Lists are equally long, and have no more pages than the sequence: no more parts than the device holds at once, three workgroups to a compute unit or, of heads of 256, one, and of 256 keys at least.
    // (8 key heads of 128 in bf16: 512 lists of 4096 tokens in 1 / 2 / 3 parts 178 / 187 / 199 us, 120 of 1600 in 6 / 7 18.4 / 20.7, 64 of 4096 in 12 / 16 26.0 / 27.9; of 256: 64 of 4096 in 4 / 8 / 12
    // 43 / 48 / 52, 192 in 1 / 4 135 / 147; 122 fp32 lists of 44 entries, of which sequences of 3 pages fill 3, in 1 / 6 7.2 / 15.2.)
    const int64_t resident = c->head_dim > 128 ? 256 : 768;
    p->splits = (int)std::max<int64_t>(1, std::min<int64_t>({resident / undivided, ceil_div(pages * c->page_size, 256), pages, 64}));
    if (!plan_ok(p)) return PAELLA_ENOSUP;
    p->stages = stages_of(p);
    p->workspace_bytes = workspace_of(p);
    p->zero_bytes = p->workspace_bytes ? counters_of(p) : 0;
    set_launch_dims(&p->dims, (unsigned)grid_of(p), 256, 0, 256);
    const double size = element_bytes(c->dtype), rows = (double)p->tokens * p->kv_heads;
    p->flops = 4.0 * p->head_dim * p->tokens * heads * (double)keys;
    p->bytes = 2.0 * rows * keys * p->head_dim * size + 2.0 * p->tokens * heads * p->head_dim * size + 4.0 * rows * count;
    return 0;
}

int paella_page_attention_dims(const paella_page_attention_plan* p, int stage, paella_launch_dims* dims) {
    if (!plan_ok(p) || !dims || stage < 0 || stage >= stages_of(p)) return PAELLA_EINVAL;
    if (stage) set_launch_dims(dims, (unsigned)ceil_div((int64_t)p->tokens * p->heads, kJoinRows / p->head_dim), 256, 0, 64);
    else set_launch_dims(dims, (unsigned)grid_of(p), 256, 0, 256);
    loaded_dims(stage ? (const void*)join_of(p) : (const void*)kernel_of(p), dims);
    return 0;
}

int paella_page_attention_launch_stage(const paella_page_attention_plan* p, int stage, const paella_kv_cache* c, const paella_kv_batch* b, const void* q, int64_t q_stride,
                                       const int32_t* pages, void* out, void* workspace, void* stream, uint32_t job_id, void* notifier) {
    if (!plan_ok(p) || stage < 0 || stage >= stages_of(p) || !planned_for(p, c, b) || !q || !pages || !out || ((uintptr_t)pages & 3)) return PAELLA_EINVAL;
    const int64_t size = element_bytes(c->dtype), row = (int64_t)p->heads * c->head_dim;
    if (q_stride < row || q_stride % 8 || (((uintptr_t)q | (uintptr_t)out) & 15)) return PAELLA_EINVAL;
    const size_t need = workspace_of(p);
    if (need && (!workspace || ((uintptr_t)workspace & 15))) return PAELLA_EINVAL;
    const double out_bytes = (double)b->tokens * row * size, list_bytes = 4.0 * p->tokens * p->kv_heads * p->count;
    const struct { const void* at; double bytes; } outs[2] = {{out, out_bytes}, {workspace, (double)need}};
    for (const auto& o : outs)
        if (o.bytes > 0 && (rows_overlap(q, p->tokens, q_stride * size, row * size, o.at, o.bytes) || overlap(pages, list_bytes, o.at, o.bytes) || over_cache(c, o.at, o.bytes) ||
                            over_batch(b, c->page_size, o.at, o.bytes)))
            return PAELLA_EINVAL;
    if (need && overlap(out, out_bytes, workspace, (double)need)) return PAELLA_EINVAL;
    PageAttentionArgs a{};
    a.c.q = (const char*)q; a.c.k_cache = (const char*)c->k; a.c.v_cache = (const char*)c->v; a.c.out = (char*)out;
    a.c.starts = b->starts; a.c.past = b->past; a.c.tables = b->tables; a.c.prefix_table = b->prefix_table;
    a.c.q_stride = q_stride * size;
    a.c.sequences = b->sequences; a.c.max_new = b->max_new; a.c.tokens = b->tokens; a.c.max_pages = b->max_pages; a.c.prefix_len = b->prefix_len;
    a.c.prefix_pages = (int)ceil_div(b->prefix_len, c->page_size);
    a.c.heads = p->heads; a.c.page_size = c->page_size; a.c.num_pages = c->num_pages;
    a.c.kv_heads = divisor((unsigned)p->kv_heads); a.c.per_kv = divisor((unsigned)(p->heads / p->kv_heads)); a.c.page_blocks = divisor((unsigned)c->page_size / 8);
    a.c.scale_log2 = p->scale * 1.44269504088896340736f;
    a.c.prefix_splits = divisor(0); a.c.own_splits = divisor((unsigned)p->splits);
    const size_t rows = (size_t)p->tokens * p->heads, counters = counters_of(p);
    a.c.counters = need && counters ? (unsigned*)workspace : nullptr;
    a.c.ml = need ? (f32x2*)((char*)workspace + counters) : nullptr;
    a.c.acc = need ? (float*)((char*)a.c.ml + up256(p->splits * rows * 8)) : nullptr;
    a.c.job_id = job_id; a.c.notifier = (Notifier*)notifier;
    a.pages = pages; a.count = p->count; a.per = (int)ceil_div(p->count, p->splits);
    a.tiles = divisor((unsigned)tiles_of(p)); a.splits = divisor((unsigned)p->splits); a.max_new = divisor((unsigned)p->max_new);
    if (stage) launch(join_of(p), dim3((unsigned)ceil_div((int64_t)rows, kJoinRows / p->head_dim)), dim3(256), 0, (hipStream_t)stream, a.c);
    else launch(kernel_of(p), dim3((unsigned)grid_of(p)), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

int paella_page_attention_launch(const paella_page_attention_plan* p, const paella_kv_cache* c, const paella_kv_batch* b, const void* q, int64_t q_stride, const int32_t* pages,
                                 void* out, void* workspace, void* stream, uint32_t job_id, void* notifier) {
    if (!plan_ok(p)) return PAELLA_EINVAL;
    const int stages = stages_of(p);
    if (stages > 1) {
        if (keeps_no_order(stream)) return PAELLA_ENOSUP;
        if (int rc = paella_page_attention_launch_stage(p, 0, c, b, q, q_stride, pages, out, workspace, stream, job_id, nullptr)) return rc;
    }
    return paella_page_attention_launch_stage(p, stages - 1, c, b, q, q_stride, pages, out, workspace, stream, job_id, notifier);
}

int paella_key_weights_plan_make(const paella_kv_cache* c, const paella_kv_batch* b, int heads, float scale, paella_key_weights_plan* p) {
    if (!p || !cache_extents_ok(c) || !batch_extents_ok(b) || heads <= 0 || heads % c->kv_heads || !scale_ok(scale)) return PAELLA_EINVAL;
    *p = paella_key_weights_plan{};
    plan_extents(p, c, b, heads);
    p->scale = scale > 0.f ? scale : 1.f / std::sqrt((float)c->head_dim);
    p->splits = p->own_splits = 1;
    if (!plan_ok(p)) return PAELLA_ENOSUP;
    const int64_t own = (int64_t)c->page_size * b->max_pages, keys = own + b->prefix_len;
    const int64_t sums = grid_of(p, 0), weights = grid_of(p, 1);
    // Few rows: memory bounds it, and parts are as many as even out the sequences' lengths (32 sequences of 8192 to 16384 tokens of 8 heads of 128 in bf16 in 16 / 32 / 48 / 64 parts 181 / 174 / 177 / 182 us).
    // Many rows: as many workgroups as the device holds at once, two to a compute unit in the first stage (4 sequences, 128 rows over 17000 keys of 8 heads, in 12 / 16 / 24 parts 35 / 29 / 45 us) and three
    // in the second.
    // The second pass over stored scores: eight workgroups to a compute unit, of 1024 tokens at least (64 sequences of 2048 to 4096 tokens, 16 rows, 8 heads by 1024 / 2048 / 4096 workgroups 80.2 / 77.4 / 77.5 us for
    // the call; 2 of 60000 tokens, 8 rows, one head, by 512 / 1024 / 2048 tokens 19.9 / 20.2 / 21.7, 3 of 900 9.8 / 9.4 / 9.6).
    const bool few = few_rows(p);
    p->splits = (int)std::max<int64_t>(1, std::min<int64_t>({ceil_div(few ? 8192 : 512, sums), ceil_div(keys, 256), 64}));
    p->own_splits = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(few ? 2048 : 768, weights), ceil_div(own, few ? 1024 : 256)));
    if (!plan_ok(p)) return PAELLA_ENOSUP;
    p->stages = 2;
    p->workspace_bytes = workspace_of(p);
    set_launch_dims(&p->dims, (unsigned)grid_of(p, 0), 256, 0, 256);
    const double size = element_bytes(c->dtype);
    p->flops = 2.0 * p->head_dim * p->tokens * heads * (double)keys;
    p->bytes = (p->prefix_len + (double)p->sequences * own) * p->kv_heads * p->head_dim * size + (double)p->tokens * heads * p->head_dim * size + 8.0 * p->sequences * own * p->kv_heads;
    return 0;
}

int paella_key_weights_dims(const paella_key_weights_plan* p, int stage, paella_launch_dims* dims) {
    if (!plan_ok(p) || !dims || stage < 0 || stage > 1) return PAELLA_EINVAL;
    set_launch_dims(dims, (unsigned)grid_of(p, stage), 256, 0, 256);
    loaded_dims((const void*)kernel_of(p, stage), dims);
    return 0;
}

int paella_key_weights_launch_stage(const paella_key_weights_plan* p, int stage, const paella_kv_cache* c, const paella_kv_batch* b, const void* q, int64_t q_stride, float* weights,
                                    void* workspace, void* stream, uint32_t job_id, void* notifier) {
    if (!plan_ok(p) || stage < 0 || stage > 1 || !planned_for(p, c, b) || !q || !weights || !workspace || (((uintptr_t)q | (uintptr_t)weights | (uintptr_t)workspace) & 15))
        return PAELLA_EINVAL;
    const int64_t size = element_bytes(c->dtype), row = (int64_t)p->heads * c->head_dim;
    if (q_stride < row || q_stride % 8) return PAELLA_EINVAL;
    const double space = (double)workspace_of(p), weight_bytes = 4.0 * p->sequences * p->kv_heads * p->max_pages * p->page_size;
    const struct { const void* at; double bytes; } outs[2] = {{weights, weight_bytes}, {workspace, space}};
    for (const auto& o : outs)
        if (rows_overlap(q, p->tokens, q_stride * size, row * size, o.at, o.bytes) || over_cache(c, o.at, o.bytes) || over_batch(b, c->page_size, o.at, o.bytes)) return PAELLA_EINVAL;
    if (overlap(weights, weight_bytes, workspace, space)) return PAELLA_EINVAL;
    WeighArgs a{};
    a.q = (const char*)q; a.k_cache = (const char*)c->k; a.weights = weights;
    a.starts = b->starts; a.past = b->past; a.tables = b->tables; a.prefix_table = b->prefix_table; a.q_stride = q_stride * size;
    a.sequences = b->sequences; a.max_new = b->max_new; a.tokens = b->tokens; a.max_pages = b->max_pages; a.prefix_len = b->prefix_len;
    a.prefix_pages = (int)ceil_div(b->prefix_len, c->page_size); a.num_pages = c->num_pages; a.page_size = c->page_size; a.heads = p->heads;
    a.kv_heads = divisor((unsigned)p->kv_heads); a.per_kv = divisor((unsigned)(p->heads / p->kv_heads)); a.page_blocks = divisor((unsigned)c->page_size / 8);
    a.splits = divisor((unsigned)p->splits); a.own_splits = divisor((unsigned)p->own_splits); a.chunks = divisor((unsigned)chunks_of(p));
    a.scale_log2 = p->scale * 1.44269504088896340736f; a.rise = kRise / a.scale_log2; a.ml = (f32x2*)workspace;
    a.scores = a.sums = (float*)((char*)workspace + parts_of(p)); a.score_rows = score_rows(p);
    a.job_id = job_id; a.notifier = (Notifier*)notifier;
    launch(kernel_of(p, stage), dim3((unsigned)grid_of(p, stage)), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

int paella_key_weights_launch(const paella_key_weights_plan* p, const paella_kv_cache* c, const paella_kv_batch* b, const void* q, int64_t q_stride, float* weights, void* workspace,
                              void* stream, uint32_t job_id, void* notifier) {
    if (!plan_ok(p)) return PAELLA_EINVAL;
    if (keeps_no_order(stream)) return PAELLA_ENOSUP;
    if (int rc = paella_key_weights_launch_stage(p, 0, c, b, q, q_stride, weights, workspace, stream, job_id, nullptr)) return rc;
    return paella_key_weights_launch_stage(p, 1, c, b, q, q_stride, weights, workspace, stream, job_id, notifier);
}

}  // extern "C"
