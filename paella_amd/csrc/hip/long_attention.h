#pragma once
// Attention over the pages that were picked for a token, and the attention weight that the tokens of a cache gather.  Included by one translation unit per
// element type.  Operands of the products as in prefix_attention.h: lane l of a wave holds query row l % 16, lane group l / 16 the scores of TPL keys that follow each other.

#include "long_common.h"
#include "prefix_attention.h"

namespace paella {

// ------------------------------------------------------------------------------------------ attention over picked pages
// A workgroup per new token, 16 heads of a key head at most, and part of the list.  It turns its part of the list into places of the cache and the tokens that are seen there, in LDS, and
// then walks the keys as the decoding step's attention walks a sequence's: each wave every fourth step, keys and values straight from memory into registers.
struct PageAttentionArgs {
    AttentionArgs c;
    const int* pages;  // [tokens][kv_heads][count]
    int count, per;    // entries of a workgroup
    Divisor tiles, splits, max_new;
};

constexpr int kListed = 512;  // entries that a workgroup looks up at a time

template <typename T, int D>
struct ListWalk : NarrowWalk<T, D> {
    using Narrow = NarrowWalk<T, D>;
    using Rows = typename Narrow::Rows;
    static constexpr bool F = Rows::F;
    static constexpr int TPL = Rows::TPL, STEP = Rows::STEP;

    int off, seen;            // of the step whose keys are loaded next: the lane group's first key in its page, and how many tokens of the page are seen

    // list: (page, tokens seen), n entries
    __device__ __forceinline__ void find(const Keys& s, const u32x2* list, int n, unsigned b8, bool even, int lane) {
        auto at = [&](unsigned block) {
            const Quotient p = divide(block, s.page_blocks);
            return Keys::Place{p.q, p.r};
        };
        auto get = [&](unsigned entry) { return entry < (unsigned)n ? list[entry] : u32x2{0u, 0u}; };
        const int group = lane >> 4;
        if (even) {
            const Keys::Place p = at(__builtin_amdgcn_readfirstlane(b8));
            const u32x2 e = get(p.entry);
            this->page_k = this->page_v = (int)e.x;
            this->in_k = this->in_v = p.in;
            seen = (int)e.y;
            off = (int)p.in * 8 + group * TPL;
        } else {
            constexpr int BLOCK_LANES_K = F ? 8 : 4;
            const Keys::Place k = at(b8 + (unsigned)(lane & 15) / BLOCK_LANES_K), v = at(b8 + (unsigned)group * TPL / 8);
            const u32x2 ek = get(k.entry), ev = get(v.entry);
            this->page_k = (int)ek.x;
            this->page_v = (int)ev.x;
            this->in_k = k.in;
            this->in_v = v.in;
            seen = (int)ev.y;
            off = (int)v.in * 8 + (F ? (group & 1) * 4 : 0);
        }
    }

    // One step, whose places are (here, held).  next(true) is called once K is no longer needed, next(false) once V is.
    template <typename Next>
    __device__ __forceinline__ void step(Rows& rows, int here, int held, float scale, Next next) {
        f32x4 x[1][Rows::NT];
        rows.scores(x, [&](int t, int c) { return this->k[t][c]; });
        next(true);
        if (__any(here + TPL > held)) {
            const int limit[1] = {held};
            Rows::mask(x, here, false, limit);
#pragma unroll
            for (int u = 0; u < TPL; ++u)  // what lies in places that no row may see can be anything
                if (here + u >= held) {
#pragma unroll
                    for (int w = 0; w < Rows::GRP * Rows::VW; ++w) this->v[u][w] = 0;
                }
        }
        // In two parts, so that results are off by little more than their own rounding: memory bounds the walk, and the second product's units have room.  (One / two parts: 64 bf16 lists of 4096 tokens of 8
        // heads of 128 179.8 / 179.9 us, 30 fp16 ones of 1600 20.2 / 20.3, 3 of 256 tokens of 2 heads of 256 8.6 / 9.0.)
        unsigned p[F ? 1 : 2][1][4];
        rows.weigh(x, scale, p);
        rows.add_values(this->v, p);
        next(false);
    }
};

// Steps wave, wave + 4, ... of the list's n entries, the next one's keys and values in flight while one is worked on.  Nothing is requested under a condition within the loop, and nothing that is not
// there: a request that may not have been made turns every wait for older ones into one for all, and the workgroup waits for all of them in the end.
template <typename T, int D>
__device__ __forceinline__ void walk_list(AttentionRows<T, D, 1, false>& rows, const Keys& s, const u32x2* list, int n, float scale, int wave, int lane) {
    using Walk = ListWalk<T, D>;
    constexpr int BLOCKS = Walk::STEP / 8;
    const int steps = (n * (int)s.page_blocks.d + BLOCKS - 1) / BLOCKS;
    if (wave >= steps) return;
    const bool even = s.page_blocks.d % BLOCKS == 0;
    Walk walk;
    walk.find(s, list, n, (unsigned)wave * BLOCKS, even, lane);
    walk.load_k(s, even, lane);
    walk.load_v(s, even, lane);
    int at = wave;
    for (; at + 4 < steps; at += 4) {
        const int here = walk.off, held = walk.seen;
        walk.step(rows, here, held, scale, [&](bool k_is_free) {
            if (k_is_free) {
                walk.find(s, list, n, (unsigned)(at + 4) * BLOCKS, even, lane);
                walk.load_k(s, even, lane);
            } else {
                walk.load_v(s, even, lane);
            }
        });
    }
    walk.step(rows, walk.off, walk.seen, scale, [](bool) {});
}

template <typename T, int D>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void page_attention_kernel(PageAttentionArgs p) {
    const AttentionArgs& a = p.c;
    hook_entry(a.notifier, a.job_id);
    using Fm = Form<1, false>;
    __shared__ __attribute__((aligned(16))) char lds[attention_lds<T, D, Fm>()];
    __shared__ u32x2 list[kListed];
    __shared__ int row_id[16], done[16], ends[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int head_bytes = D * T::bytes;
    const Quotient by_head = divide(blockIdx.x, a.kv_heads), by_split = divide(by_head.q, p.splits), by_tile = divide(by_split.q, p.tiles);
    const int h = (int)by_head.r, split = (int)by_split.r, tile = (int)by_tile.r, t = (int)by_tile.q, per_kv = (int)a.per_kv.d;
    int seq, j;
    if (row_owner(a.starts, a.sequences, p.max_new, t, lane, &seq, &j)) {
        const int64_t places = (int64_t)a.max_pages * a.page_size;
        const int visible = (int)min((int64_t)max(__builtin_amdgcn_readfirstlane(a.past[seq]), 0) + j + 1, places);  // own tokens
        const int* const table = a.tables + (size_t)seq * a.max_pages;
        const int* const entries = p.pages + ((size_t)t * a.kv_heads.d + h) * p.count;
        const int first_row = tile * 16;
        if (threadIdx.x < 16) row_id[threadIdx.x] = first_row + (int)threadIdx.x < per_kv ? t * a.heads + h * per_kv + first_row + (int)threadIdx.x : -1;
        Keys s;
        s.page_bytes = (size_t)a.kv_heads.d * a.page_size * head_bytes;
        s.page_blocks = a.page_blocks;
        s.num_pages = (unsigned)a.num_pages;
        s.k = a.k_cache + (size_t)h * a.page_size * head_bytes;
        s.v = a.v_cache + (size_t)h * a.page_size * head_bytes;
        AttentionRows<T, D, 1, false> rows;
        rows.begin();
        rows.load_q(0, a.q + t * a.q_stride + (size_t)(h * per_kv + min(first_row + (lane & 15), per_kv - 1)) * head_bytes, lane);
        const int end = min((split + 1) * p.per, p.count);
        for (int first = split * p.per; first < end; first += kListed) {
            const int n = min(end - first, kListed);
            __syncthreads();
            int last = 0;  // lane 0: behind the wave's last entry of which something is seen
            for (int i = threadIdx.x; i < n; i += 256) {
                const int e = entries[first + i], o = e < 0 ? e : e - a.prefix_pages;
                int page = 0, seen = 0;
                if (e >= 0 && o < 0) {
                    page = a.prefix_table[e];
                    seen = a.prefix_len - e * a.page_size;
                } else if (e >= 0 && o < a.max_pages) {
                    page = table[o];
                    seen = visible - o * a.page_size;
                }
                if ((unsigned)page >= (unsigned)a.num_pages) seen = 0;
                list[i] = u32x2{(unsigned)page, (unsigned)max(min(seen, a.page_size), 0)};
                const unsigned long long who = __ballot(seen > 0);
                if (who) last = i - lane + 64 - __clzll(who);
            }
            if (lane == 0) ends[wave] = last;
            __syncthreads();
            const int some = __builtin_amdgcn_readfirstlane(max(max(ends[0], ends[1]), max(ends[2], ends[3])));  // (lists of short sequences end in entries of no page)
            walk_list<T, D>(rows, s, list, some, a.scale_log2, __builtin_amdgcn_readfirstlane(wave), lane);
        }
        leave<T, D, Fm>(a, rows, split, row_id, lds);
        if (a.counters) join_last<T, D, 16>(a, row_id, (unsigned)(((size_t)t * p.tiles.d + tile) * a.kv_heads.d + h) * 32, min(per_kv - first_row, 16), done);
    }
    hook_exit(a.notifier, a.job_id);
}

using PageAttentionKernel = void (*)(PageAttentionArgs);

template <typename T>
PageAttentionKernel page_attention_kernel_of(int dim) {
    return dim == 64 ? page_attention_kernel<T, 64> : dim == 128 ? page_attention_kernel<T, 128> : dim == 256 ? page_attention_kernel<T, 256> : nullptr;
}

// ------------------------------------------------------------------------------------------ the weight that tokens gather
// weights[i] += sum over rows r of exp2(x_ri - m_r) / l_r, x = scale q . k in powers of two.  A first launch leaves each row's maximum and sum over its part of the keys, a second one
// puts the parts together and adds the rows' weights up, key by key.  A wave has a step's keys in registers and takes the rows through, 16 at a time, from LDS.  Where a key head has 16 rows at most, as
// in a step of single tokens, memory bounds both: the first launch leaves the scores, too, 4 bytes a row and key, and the second reads those instead of the keys.
struct WeighArgs {
    const char *q, *k_cache;
    float* weights;
    const int *starts, *past, *tables, *prefix_table;
    int64_t q_stride;  // bytes
    int sequences, max_new, tokens, max_pages, prefix_len, prefix_pages, num_pages, page_size, heads;
    Divisor kv_heads, per_kv, page_blocks, splits, own_splits, chunks;  // chunks: of a sequence's rows
    float scale_log2, rise;  // rise: of scores that are not yet scaled
    f32x2* ml;         // [splits][tokens * heads]: maximum and sum of each part
    float* scores;     // q . k: [sequences][kv_heads][score_rows][max_pages * page_size], -inf where a row does not see the token
    int score_rows;
    float* sums;       // what a call's rows so far give each token, where a workgroup takes them through in several chunks: [sequences][kv_heads][max_pages * page_size]
    uint32_t job_id;
    Notifier* notifier;
};

constexpr int kOnce = 2;  // for stores: not to be kept in the caches (the scores of 32 sequences of up to 16384 tokens: 174.6 us without, 170.6 with)
constexpr float kRise = 8.f;  // how far scores may be above the running maximum before it moves
constexpr float kLowest = -3.4028234663852886e38f;  // the maximum of no scores: what is not seen, -inf, is below it

// Rows that a workgroup has in LDS: 32 KB of queries.
template <typename T, int D>
constexpr int weigh_tiles() { return 32768 / (16 * D * T::bytes) > 8 ? 8 : 32768 / (16 * D * T::bytes); }

// Tiles of 16 rows that a wave takes through at once: the products and exponentials of one go on while those of the other are waited for.  (The sums of 128 rows, as below, one by
// one / two by two 33.4 / 31.3 us.)
template <int TILES>
constexpr int side_by_side() { return TILES % 2 ? 1 : 2; }

// The keys of one key head, step by step: the prefix's pages, then the sequence's own.  Places count along those pages, the prefix's last one to its end.
template <typename T, int D>
struct KeyWalk {
    using Rows = AttentionRows<T, D, 1, false>;
    static constexpr bool F = Rows::F;
    static constexpr int ROW = Rows::ROW, TPL = Rows::TPL, STEP = Rows::STEP, NT = Rows::NT, KC = Rows::KC;

    const int *prefix, *own;
    unsigned prefix_pages, all_pages, num_pages;
    const char* k;
    size_t page_bytes;
    Divisor page_blocks;

    u32x4 keys[NT][KC];  // of the step that is worked on next
    bool absent;         // the lane group's lie in no page

    // Where the blocks of a wave's steps lie, some steps ahead: lane i has block i % BLOCKS of step i / BLOCKS.  A request that follows keys' requests is answered after them: looked up
    // step by step, pages would have each step's keys wait for those of the one before.
    static constexpr int BLOCKS = STEP / 8, STEPS = 64 / BLOCKS;
    int page, page_behind;        // of this window, and of the next
    unsigned in, in_behind;       // the blocks' places in the pages
    int left;                     // steps of the window that have not been asked for

    __device__ __forceinline__ void look(int step, int lane, int* page, unsigned* in) const {
        const Quotient at = divide((unsigned)(step + lane / BLOCKS * 4) * BLOCKS + lane % BLOCKS, page_blocks);
        const unsigned e = min(at.q, all_pages - 1);
        *page = *(e < prefix_pages ? prefix + e : own + (e - prefix_pages));  // (one load: two that meet are waited for)
        *in = at.r;
    }
    __device__ __forceinline__ void begin(int step, int lane) {
        look(step, lane, &page, &in);
        look(step + STEPS * 4, lane, &page_behind, &in_behind);
        left = STEPS;
    }
    // Asks for the keys of `step`, the steps in turn.
    __device__ __forceinline__ void request(u32x4 (&to)[NT][KC], bool& gone, int step, int lane) {
        if (left == 0) {
            page = page_behind;
            in = in_behind;
            look(step + STEPS * 4, lane, &page_behind, &in_behind);
            left = STEPS;
        }
        const int mm = lane & 15, first = (STEPS - left) * BLOCKS, mine = first + mm / (F ? 8 : 4);
        --left;
        gone = (unsigned)__shfl(page, first + (lane >> 4) * TPL / 8, 64) >= num_pages;
        const unsigned p = (unsigned)__shfl(page, mine, 64), row = (unsigned)__shfl((int)in, mine, 64) * 8 + (F ? mm & 7 : mm & 3);
        const char* const from = k + (p < num_pages ? p : 0u) * page_bytes + (size_t)(row * ROW + (lane >> 4) * 16);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < KC; ++c) to[t][c] = *reinterpret_cast<const u32x4*>(from + t * 4 * ROW + c * 64);
    }

    // Asks for a wave's first step, ahead of all else that a workgroup has to fetch: any step may be asked for.
    __device__ __forceinline__ void start(int step, int lane) {
        begin(step, lane);
        request(keys, absent, step, lane);
    }

    // x = K q^T for SIDE tiles of 16 rows, whose pieces lie in LDS in the order of the lanes
    template <int SIDE>
    __device__ __forceinline__ void scores(f32x4 (&x)[SIDE][NT], const u32x4* q, int lane) const {
#pragma unroll
        for (int i = 0; i < SIDE; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t) x[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < SIDE; ++i) {
                const u32x4 piece = q[(i * KC + c) * 64 + lane];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if constexpr (F) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[i][t] = mfma_f32(as_float(keys[t][c][e]), as_float(piece[e]), x[i][t]);
                    } else {
                        x[i][t] = Mfma<T>::go(keys[t][c], piece, x[i][t]);
                    }
                }
            }
    }
};

template <typename T, int D>
__device__ __forceinline__ KeyWalk<T, D> key_walk(const WeighArgs& a, int seq, int h) {
    KeyWalk<T, D> k;
    k.prefix = a.prefix_table;
    k.own = a.tables + (size_t)seq * a.max_pages;
    k.prefix_pages = (unsigned)a.prefix_pages;
    k.all_pages = (unsigned)(a.prefix_pages + a.max_pages);
    k.num_pages = (unsigned)a.num_pages;
    k.page_bytes = (size_t)a.kv_heads.d * a.page_size * D * T::bytes;
    k.k = a.k_cache + (size_t)h * a.page_size * D * T::bytes;
    k.page_blocks = a.page_blocks;
    return k;
}

// Queries of a workgroup's rows from `first` on, piece by piece as the lanes want them in LDS; behind the sequence's last row the last one again.  All are requested before any is put
// there (4 sequences, 128 rows over 17000 bf16 keys of 8 heads of 128: the sums 31.3 us one after the other, 28.9 so).
template <typename T, int D, int TILES>
struct StagedQueries {
    static constexpr int KC = D * T::bytes / 64, PIECES = TILES * KC * 64, EACH = (PIECES + 255) / 256;
    u32x4 piece[EACH];

    __device__ __forceinline__ void request(const WeighArgs& a, int token, int h, int first, int rows) {
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
            const int i = min(u * 256 + (int)threadIdx.x, PIECES - 1), lane = i & 63, c = i / 64 % KC, tile = i / 64 / KC;
            const Quotient at = divide((unsigned)min(first + tile * 16 + (lane & 15), rows - 1), a.per_kv);
            piece[u] = *reinterpret_cast<const u32x4*>(a.q + (token + (int)at.q) * a.q_stride + (size_t)(h * (int)a.per_kv.d + (int)at.r) * D * T::bytes + c * 64 + (lane >> 4) * 16);
        }
    }
    __device__ __forceinline__ void put(u32x4* to) const {
#pragma unroll
        for (int u = 0; u < EACH; ++u)
            if (PIECES % 256 == 0 || u * 256 + (int)threadIdx.x < PIECES) to[u * 256 + threadIdx.x] = piece[u];
    }
};

// Steps over the keys [begin, end) of `walk`, every fourth one for each wave.  each(x, tile, first): scores of a tile for the step's keys, those of keys that a row does not see
// -inf; close(first): behind a step's last tile; open(): ahead of a step's requests.
template <typename T, int D, int TILES, int SIDE, typename Open, typename Each, typename Close>
__device__ __forceinline__ void walk_keys(const WeighArgs& a, KeyWalk<T, D>& walk, const u32x4* q, int first_row, int rows, int past, int begin, int end, int wave, int lane, Open open,
                                          Each each, Close close) {
    using Walk = KeyWalk<T, D>;
    int at = begin + wave;
    if (at >= end) return;
    const int behind = a.prefix_pages * a.page_size;  // the first own token's place
    const int places = min(a.max_pages * a.page_size, 1 << 30);
    const int least = behind + min(past + (int)divide((unsigned)first_row, a.per_kv).q + 1, places);  // the first place that some row does not see
    auto work = [&](bool absent) {
        const int first = at * Walk::STEP, mine = first + (lane >> 4) * Walk::TPL;
        const bool whole = (first + Walk::STEP <= a.prefix_len || (first >= behind && first + Walk::STEP <= least)) && !__any(absent);
#pragma unroll
        for (int tile = 0; tile < TILES; tile += SIDE) {
            if (first_row + tile * 16 >= rows) break;
            f32x4 x[SIDE][Walk::NT];
            walk.scores(x, q + tile * Walk::KC * 64, lane);
            if (!whole) {
#pragma unroll
                for (int i = 0; i < SIDE; ++i) {
                    const int row = min(first_row + (tile + i) * 16 + (lane & 15), rows - 1);
                    const int limit = mine < behind ? a.prefix_len : behind + min(past + (int)divide((unsigned)row, a.per_kv).q + 1, places);
#pragma unroll
                    for (int t = 0; t < Walk::NT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (absent || mine + t * 4 + e >= limit) x[i][t][e] = -INFINITY;
                }
            }
            each(x, tile, first);
        }
        close(first);
    };
    using Held = u32x4[Walk::NT][Walk::KC];
    auto move = [](Held& to, const Held& from) {
#pragma unroll
        for (int t = 0; t < Walk::NT; ++t)
#pragma unroll
            for (int c = 0; c < Walk::KC; ++c) to[t][c] = from[t][c];
    };
    // A step's keys are requested one step ahead.  Not under a condition: a request that may not have been made turns every wait for older ones into one for all.  (Two steps ahead: no faster, 180 us
    // for 32 sequences of up to 16384 tokens of 8 heads of 128 in bf16 in 16 parts either way.)
    Held next;
    bool absent_next;
    for (; at + 4 < end; at += 4) {
        open();
        walk.request(next, absent_next, at + 4, lane);
        work(walk.absent);
        move(walk.keys, next);
        walk.absent = absent_next;
    }
    open();
    work(walk.absent);
}

template <typename T, int D, int TILES>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void key_sums_kernel(WeighArgs a) {
    hook_entry(a.notifier, a.job_id);
    using Walk = KeyWalk<T, D>;
    __shared__ u32x4 q[TILES * Walk::KC * 64];
    constexpr int SIDE = side_by_side<TILES>();
    __shared__ f32x2 sums[4][TILES * 16];
    __shared__ __attribute__((aligned(16))) float stored[TILES == 1 ? 4 * 16 * Walk::STEP : 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const Quotient by_head = divide(blockIdx.x, a.kv_heads), by_split = divide(by_head.q, a.splits), by_chunk = divide(by_split.q, a.chunks);
    const int h = (int)by_head.r, split = (int)by_split.r, seq = (int)by_chunk.q, first_row = (int)by_chunk.r * TILES * 16;
    const NewTokens its = new_tokens(a.starts, a.past, seq, a.max_new, a.tokens);
    const int rows = its.count * (int)a.per_kv.d;
    if (first_row < rows) {
        const int last_row = min(first_row + TILES * 16, rows) - 1;
        const int places = min(a.max_pages * a.page_size, 1 << 30), past = min(its.past, places);
        const int keys = a.prefix_pages * a.page_size + min(past + (int)divide((unsigned)last_row, a.per_kv).q + 1, places);
        const int steps = (keys + Walk::STEP - 1) / Walk::STEP, per = (int)divide((unsigned)steps + a.splits.d - 1, a.splits).q;
        const int begin = min(split * per, steps), end = min(begin + per, steps);
        Walk walk = key_walk<T, D>(a, seq, h);
        walk.start(begin + wave, lane);
        StagedQueries<T, D, TILES> staged;
        staged.request(a, its.first, h, first_row, rows);
        staged.put(q);
        float m[TILES], l[TILES], limit[TILES];  // limit: what scores, not yet scaled, may rise to
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            m[i] = kLowest;
            limit[i] = -INFINITY;
            l[i] = 0.f;
        }
        __syncthreads();
        const int behind = a.prefix_pages * a.page_size, places_all = a.max_pages * a.page_size;
        const __amdgpu_buffer_rsrc_t to_scores = descriptor(TILES == 1 ? a.scores + ((size_t)seq * a.kv_heads.d + h) * a.score_rows * (size_t)places_all : nullptr);
        // Scores leave through LDS, so that whole lines do, 16 bytes of a row's per lane, and a step late, ahead of the requests of the next: a wait for keys waits for the stores ahead of them as well.
        float* const mine = stored + (TILES == 1 ? wave * (16 * Walk::STEP) : 0);
        int waiting = -1;
        auto put_scores = [&]() {
            if constexpr (TILES == 1) {
                constexpr int PIECES = Walk::STEP / 4;
                if (waiting < 0) return;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
                for (int u = 0; u < 16 * PIECES / 64; ++u) {
                    const int i = u * 64 + lane, row = i / PIECES, at = waiting + i % PIECES * 4 - behind;
                    if (row < rows && at >= 0 && at < places_all)
                        __builtin_amdgcn_raw_buffer_store_b128(*reinterpret_cast<const u32x4*>(mine + i * 4), to_scores, (row * places_all + at) * 4, 0, kThrough | kOnce);
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
        };
        walk_keys<T, D, TILES, SIDE>(
            a, walk, q, first_row, rows, past, begin, end, wave, lane, put_scores,
            [&](const f32x4 (&x)[SIDE][Walk::NT], int tile, int first) {
                float top[SIDE];
                bool rises = false;
#pragma unroll
                for (int i = 0; i < SIDE; ++i) {
                    top[i] = x[i][0][0];
#pragma unroll
                    for (int t = 0; t < Walk::NT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) top[i] = fmaxf(top[i], x[i][t][e]);
                    rises |= top[i] > limit[tile + i];
                }
                if (__any(rises)) {  // (until then the exponentials have room above 1)
#pragma unroll
                    for (int i = 0; i < SIDE; ++i) {
                        const float now = fmaxf(m[tile + i], top[i] * a.scale_log2);
                        l[tile + i] *= m[tile + i] == now ? 1.f : __builtin_amdgcn_exp2f(m[tile + i] - now);
                        m[tile + i] = now;
                        limit[tile + i] = fmaxf(limit[tile + i], top[i] + a.rise);
                    }
                }
#pragma unroll
                for (int i = 0; i < SIDE; ++i)
#pragma unroll
                    for (int t = 0; t < Walk::NT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) l[tile + i] += __builtin_amdgcn_exp2f(__builtin_fmaf(x[i][t][e], a.scale_log2, -m[tile + i]));
                if constexpr (TILES == 1) {
#pragma unroll
                    for (int t = 0; t < Walk::NT; ++t) *reinterpret_cast<f32x4*>(mine + (lane & 15) * Walk::STEP + (lane >> 4) * Walk::TPL + t * 4) = x[0][t];
                    waiting = first;
                }
            },
            [](int) {});
        put_scores();
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
#pragma unroll
            for (int off = 16; off < 64; off <<= 1) {
                const float other = __shfl_xor(m[i], off, 64), more = __shfl_xor(l[i], off, 64), now = fmaxf(m[i], other);
                l[i] = l[i] * (m[i] == now ? 1.f : __builtin_amdgcn_exp2f(m[i] - now)) + more * (other == now ? 1.f : __builtin_amdgcn_exp2f(other - now));
                m[i] = now;
            }
            if (lane < 16) sums[wave][i * 16 + lane] = f32x2{m[i], l[i]};
        }
        __syncthreads();
        const int row = first_row + (int)threadIdx.x;
        if ((int)threadIdx.x < TILES * 16 && row < rows) {
            float top = -INFINITY, total = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) top = fmaxf(top, sums[w][threadIdx.x].x);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const f32x2 s = sums[w][threadIdx.x];
                total += s.y * (s.x == top ? 1.f : __builtin_amdgcn_exp2f(s.x - top));
            }
            const Quotient at = divide((unsigned)row, a.per_kv);
            const size_t id = (size_t)split * a.tokens * a.heads + (size_t)(its.first + (int)at.q) * a.heads + h * (int)a.per_kv.d + (int)at.r;
            put_pair(a.ml + id, top, total);
        }
    }
    hook_exit(a.notifier, a.job_id);
}

// Of each of ROWS rows from `first` on: maximum and one over the sum, the parts put together in their order.  Behind the last row, and where a row sees nothing, what gives no weights.
template <int ROWS>
__device__ __forceinline__ void join_rows(const WeighArgs& a, int token, int h, int first, int rows, f32x2* whole) {
    constexpr int AHEAD = 8;
    if ((int)threadIdx.x < ROWS) {
        const int row = first + (int)threadIdx.x;
        float top = -INFINITY, total = 0.f;
        if (row < rows) {
            const Quotient at = divide((unsigned)row, a.per_kv);
            const size_t all = (size_t)a.tokens * a.heads;
            const f32x2* const from = a.ml + (size_t)(token + (int)at.q) * a.heads + h * (int)a.per_kv.d + (int)at.r;
            for (unsigned s = 0; s < a.splits.d; s += AHEAD) {
                f32x2 part[AHEAD];
                float now = top;
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) part[u] = from[min(s + u, a.splits.d - 1) * all];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) now = fmaxf(now, part[u].x);
                total *= top == now ? 1.f : __builtin_amdgcn_exp2f(top - now);
#pragma unroll
                for (int u = 0; u < AHEAD; ++u)
                    if (s + u < a.splits.d) total += part[u].y * (part[u].x == now ? 1.f : __builtin_amdgcn_exp2f(part[u].x - now));
                top = now;
            }
        }
        whole[threadIdx.x] = total == 0.f ? f32x2{INFINITY, 0.f} : f32x2{top, 1.f / total};
    }
}

template <typename T, int D, int TILES>
__global__ __launch_bounds__(256, D > 128 ? 1 : 3) void key_weights_kernel(WeighArgs a) {
    hook_entry(a.notifier, a.job_id);
    using Walk = KeyWalk<T, D>;
    __shared__ u32x4 q[TILES * Walk::KC * 64];
    constexpr int SIDE = side_by_side<TILES>();
    __shared__ f32x2 whole[TILES * 16];  // of each row: maximum and one over the sum
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const Quotient by_head = divide(blockIdx.x, a.kv_heads), by_split = divide(by_head.q, a.own_splits);
    const int h = (int)by_head.r, split = (int)by_split.r, seq = (int)by_split.q;
    const NewTokens its = new_tokens(a.starts, a.past, seq, a.max_new, a.tokens);
    const int rows = its.count * (int)a.per_kv.d;
    if (rows > 0) {
        const int places = min(a.max_pages * a.page_size, 1 << 30), past = min(its.past, places), held = min(past + its.count, places);
        const int before = a.prefix_pages * a.page_size / Walk::STEP, steps = (a.prefix_pages * a.page_size + held + Walk::STEP - 1) / Walk::STEP - before;
        const int per = (int)divide((unsigned)steps + a.own_splits.d - 1, a.own_splits).q;
        const int begin = before + min(split * per, steps), end = min(begin + per, before + steps);
        const size_t head_at = ((size_t)seq * a.kv_heads.d + h) * ((size_t)a.max_pages * a.page_size);
        float *const weights = a.weights + head_at, *const sums = a.sums + head_at;
        Walk walk = key_walk<T, D>(a, seq, h);
        for (int first_row = 0; first_row < rows && begin < end; first_row += TILES * 16) {
            walk.start(begin + wave, lane);
            StagedQueries<T, D, TILES> staged;
            staged.request(a, its.first, h, first_row, rows);
            __syncthreads();
            join_rows<TILES * 16>(a, its.first, h, first_row, rows, whole);
            staged.put(q);
            __syncthreads();
            const bool whole_call = first_row + TILES * 16 >= rows;
            float* const to = whole_call ? weights : sums;
            float w[Walk::TPL];
#pragma unroll
            for (int e = 0; e < Walk::TPL; ++e) w[e] = 0.f;
            walk_keys<T, D, TILES, SIDE>(
                a, walk, q, first_row, rows, past, begin, end, wave, lane, [] {},
                [&](const f32x4 (&x)[SIDE][Walk::NT], int tile, int) {
                    f32x2 row[SIDE];
#pragma unroll
                    for (int i = 0; i < SIDE; ++i) row[i] = whole[(tile + i) * 16 + (lane & 15)];
#pragma unroll
                    for (int i = 0; i < SIDE; ++i)
#pragma unroll
                        for (int t = 0; t < Walk::NT; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[t * 4 + e] += row[i].y * __builtin_amdgcn_exp2f(__builtin_fmaf(x[i][t][e], a.scale_log2, -row[i].x));
                },
                [&](int first) {
                    float mine = 0.f;
#pragma unroll
                    for (int e = 0; e < Walk::TPL; ++e) {
                        const float sum = row_all(w[e], [](float x, float y) { return x + y; });
                        if ((lane & 15) == e) mine = sum;
                        w[e] = 0.f;
                    }
                    const int i = first + (lane >> 4) * Walk::TPL + (lane & 15) - a.prefix_pages * a.page_size;
                    // The call's sum by itself until it is whole: a heavy old weight would take a rounding of its own size from each part of it.  (A prompt of 2000 tokens, 8000 rows of 8 bf16 heads of 128,
                    // in 63 chunks: each added to the weight itself / so 542 / 546 us.)
                    if ((lane & 15) < Walk::TPL && i >= 0 && i < held) {
                        auto at = [](const float* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
                        const float before = first_row ? at(sums + i) : 0.f, old = whole_call && i < past ? at(weights + i) : 0.f;
                        store_out(to + i, old + (before + mine));
                    }
                });
        }
    }
    hook_exit(a.notifier, a.job_id);
}

using WeighKernel = void (*)(WeighArgs);

WeighKernel stored_weights();  // from stored scores, of every type

// few: at most 16 rows a sequence and key head
template <typename T, int D>
WeighKernel key_sums_kernel_of(bool few) { return few ? key_sums_kernel<T, D, 1> : key_sums_kernel<T, D, weigh_tiles<T, D>()>; }
template <typename T>
WeighKernel key_sums(int dim, bool few) {
    return dim == 64 ? key_sums_kernel_of<T, 64>(few) : dim == 128 ? key_sums_kernel_of<T, 128>(few) : key_sums_kernel_of<T, 256>(few);
}
template <typename T>
WeighKernel key_weights(int dim, bool few) {
    if (few) return stored_weights();
    return dim == 64 ? key_weights_kernel<T, 64, weigh_tiles<T, 64>()> : dim == 128 ? key_weights_kernel<T, 128, weigh_tiles<T, 128>()> : key_weights_kernel<T, 256, weigh_tiles<T, 256>()>;
}

// Defined once per type.
PageAttentionKernel page_attention_f32(int dim);
PageAttentionKernel page_attention_bf16(int dim);
PageAttentionKernel page_attention_f16(int dim);
WeighKernel key_sums_f32(int dim, bool few);
WeighKernel key_sums_bf16(int dim, bool few);
WeighKernel key_sums_f16(int dim, bool few);
WeighKernel key_weights_f32(int dim, bool few);
WeighKernel key_weights_bf16(int dim, bool few);
WeighKernel key_weights_f16(int dim, bool few);

}  // namespace paella
