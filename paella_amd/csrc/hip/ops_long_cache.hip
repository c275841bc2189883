// Operators that keep a long paged cache from being read and kept whole: bounds of the pages' keys, the selection of pages by them, and eviction.
// (Attention over the pages and the weights that tokens gather: long_attention.h.)

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "long_common.h"
#include "pick_largest.h"
#include "prefix_attention.h"

namespace {

using namespace paella;

// ------------------------------------------------------------------------------------------ bounds of a page's keys
// A wave per page and key head: 16 bytes of a key per lane, as many keys side by side as fit the wave, all of the page's requested eight at a time.  Bound by memory:
// each key of the pages is read once.
struct BoundsArgs {
    const char* k_cache;
    char* bounds;
    const int *starts, *past, *tables;
    int sequences, max_new, tokens, max_pages, num_pages, page_size, row_bytes, pieces, group_log2;  // pieces: 16 bytes of a key each; 2^group_log2 lanes side by side for a key
    Divisor kv_heads, touched;  // touched: most pages that a sequence's new tokens lie in
    unsigned items;
    uint32_t job_id;
    Notifier* notifier;
};

template <typename T>
__device__ __forceinline__ void widen(u32x4 w, float (&low)[16 / T::bytes], float (&high)[16 / T::bytes]) {
    if constexpr (T::bytes == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            low[e] = fminf(low[e], as_float(w[e]));
            high[e] = fmaxf(high[e], as_float(w[e]));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const f32x2 v = unpack2<T>(w[e]);
            low[2 * e] = fminf(low[2 * e], v.x);
            high[2 * e] = fmaxf(high[2 * e], v.x);
            low[2 * e + 1] = fminf(low[2 * e + 1], v.y);
            high[2 * e + 1] = fmaxf(high[2 * e + 1], v.y);
        }
    }
}

template <typename T>
__device__ __forceinline__ u32x4 packed(const float (&x)[16 / T::bytes]) {  // values of the type, so nothing is rounded
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (T::bytes == 4) w[e] = as_word(x[e]);
        else w[e] = pack2<T>(x[2 * e], x[2 * e + 1]);
    }
    return w;
}

template <typename T>
__global__ __launch_bounds__(256) void page_bounds_kernel(BoundsArgs a) {
    hook_entry(a.notifier, a.job_id);
    constexpr int V = 16 / T::bytes;
    const int lane = threadIdx.x & 63;
    const unsigned item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (item < a.items) {
        const Quotient by_head = divide(item, a.kv_heads), by_page = divide(by_head.q, a.touched);
        const int seq = (int)by_page.q;
        const NewTokens its = new_tokens(a.starts, a.past, seq, a.max_new, a.tokens);
        const unsigned page = (unsigned)its.past / (unsigned)a.page_size + by_page.r;  // along the sequence
        const int64_t first = (int64_t)page * a.page_size, end = (int64_t)its.past + its.count;
        int physical = -1;
        if (its.count > 0 && first < end && page < (unsigned)a.max_pages) physical = __builtin_amdgcn_readfirstlane(a.tables[(size_t)seq * a.max_pages + page]);
        if ((unsigned)physical < (unsigned)a.num_pages) {
            const int held = (int)min((int64_t)a.page_size, end - first);
            const size_t head_at = (size_t)physical * a.kv_heads.d + by_head.r;
            const char* const keys = a.k_cache + head_at * a.page_size * a.row_bytes;
            const __amdgpu_buffer_rsrc_t to = descriptor(a.bounds + head_at * 2 * a.row_bytes);
            const int group = 1 << a.group_log2, each = 64 >> a.group_log2;
            for (int piece = lane & (group - 1); piece < (a.pieces + group - 1) / group * group; piece += group) {  // (whole waves: lanes of all groups meet below)
                const bool in = piece < a.pieces;
                float low[V], high[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    low[e] = INFINITY;
                    high[e] = -INFINITY;
                }
                constexpr int AHEAD = 8;
                for (int key = lane >> a.group_log2; key < held; key += AHEAD * each) {
                    u32x4 w[AHEAD];
#pragma unroll
                    for (int u = 0; u < AHEAD; ++u)  // behind the last key: the last one again
                        w[u] = *reinterpret_cast<const u32x4*>(keys + (size_t)min(key + u * each, held - 1) * a.row_bytes + (in ? piece : 0) * 16);
#pragma unroll
                    for (int u = 0; u < AHEAD; ++u) widen<T>(w[u], low, high);
                }
                for (int off = group; off < 64; off <<= 1) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        low[e] = fminf(low[e], __shfl_xor(low[e], off, 64));
                        high[e] = fmaxf(high[e], __shfl_xor(high[e], off, 64));
                    }
                }
                if (lane < group && in) {
                    __builtin_amdgcn_raw_buffer_store_b128(packed<T>(low), to, piece * 16, 0, kThrough);
                    __builtin_amdgcn_raw_buffer_store_b128(packed<T>(high), to, a.row_bytes + piece * 16, 0, kThrough);
                }
            }
        }
    }
    hook_exit(a.notifier, a.job_id);
}

// ------------------------------------------------------------------------------------------ selection of pages
// worth(e) = max over the key head's query heads of sum_d max(q_d low_d, q_d high_d) = q+ . high + q- . low, q+ and q- the values above and below 0.  Which of two neighbours is taken is decided by their last
// digits, in 64 bits; but nearly all pages are far from the border.  So the matrix units take the worths in 32 bits, at the rate that memory delivers the bounds, together with how far each can
// be off: of a sum of 2 D products by 4 D * 2^-24 of the sum of their magnitudes, |q| . max(|low|, |high|).  Pages that are further from the border than
// that are decided; the few others, if they are not all taken or none of them, get their worths in 64 bits.  (All of them in 64 bits by the vector unit: 58 us for 32 rows of 1024 pages of 8 heads of 128 in bf16, 100 MB.)
struct SelectArgs {
    const char *q, *bounds;
    const int *starts, *past, *tables, *prefix_table;
    f32x2* entries;    // [tokens][kv_heads][pitch]
    int* pages;
    int64_t q_stride;  // bytes
    int sequences, tokens, max_pages, prefix_pages, num_pages, heads, first, last, count, dim, dtype;
    unsigned pitch;
    Divisor max_new, kv_heads, splits, page_size;
    uint32_t job_id;
    Notifier* notifier;
};

// What a page's entry holds beside its worth: how far that can be off, over 4 D * 2^-24, +inf where it is no number or may be infinite; or
constexpr float kNoPage = -1.f, kForced = -2.f;

__device__ __forceinline__ int page_along(const SelectArgs& a, int seq, unsigned e) {
    return e < (unsigned)a.prefix_pages ? a.prefix_table[e] : a.tables[(size_t)seq * a.max_pages + (e - a.prefix_pages)];
}

template <typename T> __device__ __forceinline__ u32x4 sign_mask(u32x4 q) {
    u32x4 m;
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = T::bytes == 4 ? (unsigned)((int)q[e] >> 31) : (q[e] >> 15 & 0x00010001u) * 0xFFFFu;
    return m;
}
template <typename T> __device__ __forceinline__ u32x4 magnitude(u32x4 v) { return v & (T::bytes == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu); }
template <typename T> __device__ __forceinline__ u32x4 larger_magnitude(u32x4 v, u32x4 w) {  // (magnitudes compare as whole numbers do, a NaN above all)
    v = magnitude<T>(v);
    w = magnitude<T>(w);
    u32x4 m;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (T::bytes == 4) {
            m[e] = max(v[e], w[e]);
        } else {
            typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
            m[e] = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, v[e]), __builtin_bit_cast(u16x2, w[e])));
        }
    }
    return m;
}

// x += v w^T of 16 rows each, 16 bytes of a row per lane
template <typename T>
__device__ __forceinline__ f32x4 multiply(u32x4 v, u32x4 w, f32x4 x) {
    if constexpr (T::bytes == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x = mfma_f32(as_float(v[e]), as_float(w[e]), x);
        return x;
    } else {
        return Mfma<T>::go(v, w, x);
    }
}

constexpr int kScreened = 32;  // pages of a wave's turn

// Turns first, first + step, ... of a row's pages: put(page, entry).
template <typename T, int D, typename Put>
__device__ __forceinline__ void screen_pages(const SelectArgs& a, int t, int seq, int h, unsigned pages, unsigned first, unsigned step, Put put) {
    constexpr int ROW = D * T::bytes, KC = ROW / 64, U = kScreened / 16;
    const int lane = threadIdx.x & 63, mm = lane & 15, group = lane >> 4;
    const int heads = a.heads / (int)a.kv_heads.d;
    for (unsigned turn = first; turn * kScreened < pages; turn += step) {
        int page[U];
        const char* from[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            page[u] = page_along(a, seq, min(turn * kScreened + u * 16 + mm, pages - 1));
            from[u] = a.bounds + ((size_t)((unsigned)page[u] < (unsigned)a.num_pages ? page[u] : 0) * a.kv_heads.d + h) * 2 * ROW + group * 16;
        }
        f32x4 worth[U], error[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            worth[u] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            error[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        for (int g = 0; g < heads; g += 16) {
            const char* const row = a.q + t * a.q_stride + (size_t)(h * heads + min(g + mm, heads - 1)) * ROW + group * 16;
            f32x4 x[U], y[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = y[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const u32x4 q = *reinterpret_cast<const u32x4*>(row + c * 64), below = sign_mask<T>(q);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const u32x4 low = *reinterpret_cast<const u32x4*>(from[u] + c * 64), high = *reinterpret_cast<const u32x4*>(from[u] + ROW + c * 64);
                    x[u] = multiply<T>(high, q & ~below, x[u]);
                    x[u] = multiply<T>(low, q & below, x[u]);
                    y[u] = multiply<T>(larger_magnitude<T>(low, high), magnitude<T>(q), y[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    worth[u][e] = fmaxf(worth[u][e], x[u][e]);
                    error[u][e] = fmaxf(error[u][e], y[u][e] < 1e38f ? y[u][e] : INFINITY);  // (below it no sum on the way was infinite either)
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            f32x2 mine = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // over the heads; lane mm = e has that of page 4 group + e
                const float w = row_all(worth[u][e], [](float p, float q) { return fmaxf(p, q); }), r = row_all(error[u][e], [](float p, float q) { return fmaxf(p, q); });
                if (mm == e) mine = f32x2{w, r};
            }
            const unsigned e = turn * kScreened + u * 16 + group * 4 + mm;
            const int at = __shfl(page[u], group * 4 + (mm & 3), 64);
            if (e < (unsigned)a.first || e + a.last >= pages) mine.y = kForced;
            if ((unsigned)at >= (unsigned)a.num_pages) mine.y = kNoPage;
            if (mm < 4 && e < pages) put(e, mine);
        }
    }
}

__device__ __forceinline__ double value_at(const char* p, int i, int dtype) {
    if (dtype == PAELLA_F32) return (double)reinterpret_cast<const float*>(p)[i];
    const unsigned w = reinterpret_cast<const unsigned short*>(p)[i];
    return (double)(dtype == PAELLA_BF16 ? unpack2<Bf16>(w).x : unpack2<F16>(w).x);
}

// A page's worth in 64 bits, by a whole wave.
__device__ __forceinline__ unsigned long long exact_worth(const SelectArgs& a, int t, int seq, int h, unsigned e) {
    const int lane = threadIdx.x & 63, heads = a.heads / (int)a.kv_heads.d, row = a.dim * (a.dtype == PAELLA_F32 ? 4 : 2);
    const int page = page_along(a, seq, e);  // (in the cache: others are not asked for)
    const char* const low = a.bounds + ((size_t)page * a.kv_heads.d + h) * 2 * row;
    const char* const q = a.q + t * a.q_stride + (size_t)h * heads * row;
    unsigned long long best = 0;
    for (int g = 0; g < heads; ++g) {
        double sum = 0.0;
        for (int d = lane; d < a.dim; d += 64) {
            const double x = value_at(q + (size_t)g * row, d, a.dtype), u = x * value_at(low, d, a.dtype), v = x * value_at(low + row, d, a.dtype);
            sum += u > v || u != u ? u : v;
        }
        for (int off = 32; off; off >>= 1) sum += __builtin_bit_cast(double, shuffle_xor64(__builtin_bit_cast(unsigned long long, sum), off));
        best = max(best, number_key(sum, number_key((double)INFINITY, 0ull)));  // a worth that is no number counts as the largest
    }
    return best;
}

__device__ __forceinline__ void put_int(int* p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

constexpr unsigned kOpen = 512;  // pages whose worths in 64 bits are taken at a time

template <int WAVES>
struct PageSpace {
    PickSpace<WAVES> pick;
    unsigned forced[WAVES], unknown[WAVES];
    float error[WAVES];
    unsigned inside[WAVES], open[WAVES];
    unsigned list[kOpen];
    unsigned long long worth[kOpen];
};

// The row's pages by their entries, load(i).  KEYS as in Span; where it is 0, keys take the entries' places, keep(i, key).
template <int WAVES, int KEYS, typename Load, typename Keep>
__device__ __forceinline__ void pick_pages(const SelectArgs& a, int t, int seq, int h, unsigned pages, int* to, PageSpace<WAVES>& s, Load load, Keep keep) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Span<WAVES, KEYS> span(pages);
    unsigned long long held[KEYS ? KEYS : 1];  // entries, and then keys
    span.hold(held, load);
    auto get = [&](int u, unsigned i) { return KEYS ? held[u] : load(i); };
    auto entry_of = [](bool is, unsigned long long v) { return is ? __builtin_bit_cast(f32x2, v) : f32x2{0.f, kNoPage}; };
    auto known = [](f32x2 e) { return e.y >= 0.f && e.y < INFINITY; };
    Range<unsigned> range;
    unsigned forced = 0, unknown = 0;
    float error = 0.f;
    span.visit(get, [&](int, unsigned, bool is, unsigned long long v) {
        const f32x2 e = entry_of(is, v);
        forced += __popcll(__ballot(e.y == kForced));
        unknown += __popcll(__ballot(e.y == INFINITY));
        range.add(known(e) ? number_key(e.x, 1u) : 0u);
        if (known(e)) error = fmaxf(error, e.y);
    });
    error = wave_max_f(error);
    if (lane == 0) {
        s.forced[wave] = forced;
        s.unknown[wave] = unknown;
        s.error[wave] = error;
    }
    range.join(s.pick);
    forced = unknown = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        forced += s.forced[w];
        unknown += s.unknown[w];
        error = fmaxf(error, s.error[w]);
    }
    const unsigned want = (unsigned)a.count - min(forced, (unsigned)a.count);
    // Pages worth more than `in` are taken, those worth less than `out` are not, those between are open.
    float in = -INFINITY, out = -INFINITY;
    const bool all = range.some + unknown <= want;
    if (!all && want) {
        const float off = 2.f * (error * (float)(4 * a.dim) * 0x1p-24f + 0x1p-110f);  // (products below the least number of 32 bits are lost, too)
        in = INFINITY;
        if (range.some >= want) {
            const float border = key_number(range.some == want ? range.least
                                                               : find_bound<WAVES, KEYS, unsigned>(span, range, want, s.pick, [&](int u, unsigned i) {
                                                                     const f32x2 e = entry_of(true, get(u, i));
                                                                     return known(e) ? number_key(e.x, 1u) : 0u;
                                                                 }).bound);
            out = border - off;
            if (!unknown) in = border + off;  // (a page that nothing is known of may be worth more)
        }
    }
    auto is_in = [&](f32x2 e) { return e.y == kForced || (all && e.y >= 0.f) || (known(e) && want && e.x > in); };
    auto is_open = [&](f32x2 e) { return !all && want && (e.y == INFINITY || (known(e) && e.x >= out && e.x <= in)); };
    unsigned inside = 0, open = 0;
    span.visit(get, [&](int, unsigned, bool is, unsigned long long v) {
        const f32x2 e = entry_of(is, v);
        inside += __popcll(__ballot(is_in(e)));
        open += __popcll(__ballot(is_open(e)));
    });
    if (lane == 0) {
        s.inside[wave] = inside;
        s.open[wave] = open;
    }
    __syncthreads();
    inside = open = 0;
    unsigned ahead = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) ahead += s.open[w];
        inside += s.inside[w];
        open += s.open[w];
    }
    const bool decided = inside + open <= (unsigned)a.count;  // all that are open are taken
    auto set = [&](int u, unsigned i, bool is, unsigned long long k) {
        if constexpr (KEYS > 0) held[u] = k;
        else if (is) keep(i, k);
    };
    // Keys: all ones for what is taken, 0 for what is not, and for what is open 1 until its worth in 64 bits is there (whose key is above that and below all ones).
    constexpr unsigned long long kIn = ~0ull, kWaiting = 1;
    span.visit(get, [&](int u, unsigned i, bool is, unsigned long long v) {
        const f32x2 e = entry_of(is, v);
        set(u, i, is, is_in(e) || (decided && is_open(e)) ? kIn : is_open(e) ? kWaiting : 0ull);
    });
    Bound<unsigned long long> bound = {1, ~0u};
    if (!decided) {
        for (unsigned first = 0; first < open; first += kOpen) {  // the waves share them
            const unsigned n = min(open - first, kOpen);
            auto each_open = [&](auto&& then) {
                unsigned slot = ahead - first;  // (those of other turns are far above n)
                span.visit(get, [&](int u, unsigned i, bool is, unsigned long long v) {
                    const bool mine = is && v && v != kIn;
                    const unsigned long long who = __ballot(mine);
                    const unsigned at = slot + (unsigned)__popcll(who & ((1ull << lane) - 1));
                    if (mine && at < n) then(u, i, at);
                    slot += (unsigned)__popcll(who);
                });
            };
            each_open([&](int, unsigned i, unsigned at) { s.list[at] = i; });
            __syncthreads();
            for (unsigned k = (unsigned)__builtin_amdgcn_readfirstlane(wave); k < n; k += WAVES) {
                const unsigned long long worth = exact_worth(a, t, seq, h, (unsigned)__builtin_amdgcn_readfirstlane((int)s.list[k]));
                if (lane == 0) s.worth[k] = worth;
            }
            __syncthreads();
            each_open([&](int u, unsigned i, unsigned at) { set(u, i, true, s.worth[at]); });
            __syncthreads();
        }
        Range<unsigned long long> keys;
        span.visit(get, [&](int, unsigned, bool is, unsigned long long v) { keys.add(is ? v : 0ull); });
        keys.join(s.pick);
        bound = find_bound<WAVES, KEYS, unsigned long long>(span, keys, (unsigned)a.count, s.pick, get);
    }
    const unsigned taken = emit_taken<WAVES, KEYS, unsigned long long>(span, bound, s.pick, get, [&](unsigned place, unsigned i) { put_int(to + place, (int)i); });
    for (unsigned i = taken + threadIdx.x; i < (unsigned)a.count; i += WAVES * 64) put_int(to + i, -1);
}

template <typename T, int D>
__global__ __launch_bounds__(256) void page_screen_kernel(SelectArgs a) {
    hook_entry(a.notifier, a.job_id);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const Quotient by_head = divide(blockIdx.x, a.kv_heads), by_split = divide(by_head.q, a.splits);
    const int t = (int)by_split.q, h = (int)by_head.r;
    int seq, j;
    if (row_owner(a.starts, a.sequences, a.max_new, t, lane, &seq, &j)) {
        const unsigned pages = (unsigned)a.prefix_pages + (unsigned)own_pages(__builtin_amdgcn_readfirstlane(a.past[seq]), j, a.page_size, a.max_pages);
        f32x2* const entries = a.entries + ((size_t)t * a.kv_heads.d + h) * a.pitch;
        screen_pages<T, D>(a, t, seq, h, pages, by_split.r * 4 + wave, a.splits.d * 4, [&](unsigned e, f32x2 x) { put_pair(entries + e, x.x, x.y); });
    }
    hook_exit(a.notifier, a.job_id);
}

template <int WAVES, int KEYS>
__global__ __launch_bounds__(WAVES * 64) void page_pick_kernel(SelectArgs a) {
    hook_entry(a.notifier, a.job_id);
    __shared__ PageSpace<WAVES> space;
    const int lane = threadIdx.x & 63;
    const Quotient by_head = divide(blockIdx.x, a.kv_heads);
    const int t = (int)by_head.q, h = (int)by_head.r;
    int seq, j;
    if (row_owner(a.starts, a.sequences, a.max_new, t, lane, &seq, &j)) {
        const unsigned pages = (unsigned)a.prefix_pages + (unsigned)own_pages(__builtin_amdgcn_readfirstlane(a.past[seq]), j, a.page_size, a.max_pages);
        unsigned long long* const entries = reinterpret_cast<unsigned long long*>(a.entries) + (size_t)blockIdx.x * a.pitch;
        pick_pages<WAVES, KEYS>(
            a, t, seq, h, pages, a.pages + (size_t)blockIdx.x * a.count, space, [&](unsigned i) { return entries[i]; }, [&](unsigned i, unsigned long long k) { entries[i] = k; });
    }
    hook_exit(a.notifier, a.job_id);
}

// ------------------------------------------------------------------------------------------ eviction
struct EvictArgs {
    char *k_cache, *v_cache;
    float* weights;
    const int *past, *tables;
    int *kept, *past_out;
    int sequences, max_pages, num_pages, page_size, row_bytes, keep, first, recent;
    unsigned places;  // of a sequence
    unsigned slice_log2;  // bytes of a row that a workgroup moves
    Divisor kv_heads, slices, pages;  // pages: divides by the page size
    uint32_t job_id;
    Notifier* notifier;
};

// The tokens that stay of a sequence, for one key head: those between the first and the recent ones by their weights.
template <int WAVES, int KEYS>
__global__ __launch_bounds__(WAVES * 64) void evict_pick_kernel(EvictArgs a) {
    hook_entry(a.notifier, a.job_id);
    __shared__ PickSpace<WAVES> space;
    const Quotient by_head = divide(blockIdx.x, a.kv_heads);
    const unsigned n = (unsigned)min(max((int64_t)__builtin_amdgcn_readfirstlane(a.past[by_head.q]), (int64_t)0), (int64_t)a.places);
    int* const to = a.kept + (size_t)blockIdx.x * a.keep;
    if (n <= (unsigned)a.keep) {
        for (unsigned i = threadIdx.x; i < (unsigned)a.keep; i += WAVES * 64) put_int(to + i, i < n ? (int)i : -1);
    } else {
        const unsigned first = (unsigned)a.first, middle = n - first - (unsigned)a.recent, want = (unsigned)(a.keep - a.first - a.recent);
        for (unsigned i = threadIdx.x; i < first; i += WAVES * 64) put_int(to + i, (int)i);
        for (unsigned i = threadIdx.x; i < (unsigned)a.recent; i += WAVES * 64) put_int(to + first + want + i, (int)(first + middle + i));
        if (want) {
            const float* const w = a.weights + (size_t)blockIdx.x * a.places + first;
            const Span<WAVES, KEYS> span(middle);
            unsigned held[KEYS ? KEYS : 1];
            auto load = [&](unsigned i) { return number_key(w[i], 1u); };
            span.hold(held, load);
            auto get = [&](int u, unsigned i) { return KEYS ? held[u] : load(i); };
            Range<unsigned> range;
            span.visit(get, [&](int, unsigned, bool is, unsigned k) { range.add(is ? k : 0u); });
            range.join(space);
            const Bound<unsigned> bound = find_bound<WAVES, KEYS, unsigned>(span, range, want, space, get);
            emit_taken<WAVES, KEYS, unsigned>(span, bound, space, get, [&](unsigned place, unsigned i) { put_int(to + first + place, (int)(first + i)); });
        }
    }
    hook_exit(a.notifier, a.job_id);
}

// Tokens move to lower places, in order: a workgroup takes some bytes of every key, or of every value, of a sequence's key head through, a run of tokens at a time, all of which it has read
// before it writes the first.  What later runs read lies behind everything that earlier ones wrote, and no two workgroups touch the same bytes, so nothing waits for another workgroup, and a
// run's reads go out ahead of the writes of the one before it.
constexpr int kMoveAhead = 4;   // tokens of a lane in a run

// 16 bytes that go through to memory.  (The wait states are those between a store and the next write of its registers.)
__device__ __forceinline__ void put16(char* p, u32x4 v) { asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" ::"v"(p), "v"(v) : "memory"); }

__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
    hook_entry(a.notifier, a.job_id);
    const Quotient by_slice = divide(blockIdx.x, a.slices), by_head = divide(by_slice.q, a.kv_heads);
    const unsigned slice = by_slice.r, h = by_head.r, seq = by_head.q, keep = (unsigned)a.keep;
    const int* const kept = a.kept + (size_t)by_slice.q * a.keep;
    const int* const table = a.tables + (size_t)seq * a.max_pages;
    const unsigned half = (a.slices.d - 1) / 2;  // slices of the keys, of the values, and one for the weights
    if (kept[keep - 1] >= 0) {                   // else all of the sequence stays
        if (slice == a.slices.d - 1) {
            float* const w = a.weights + (size_t)by_slice.q * a.places;
            for (unsigned first = 0; first < keep; first += 1024) {
                float x[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const unsigned i = first + u * 256 + threadIdx.x, from = i < keep ? (unsigned)kept[i] : 0u;
                    x[u] = from < a.places ? w[from] : 0.f;
                }
                __syncthreads();
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const unsigned i = first + u * 256 + threadIdx.x;
                    if (i < keep) store_out(w + i, x[u]);
                }
            }
            if (h == 0 && threadIdx.x == 0) put_int(a.past_out + seq, a.keep);
        } else {
            char* const cache = slice < half ? a.k_cache : a.v_cache;
            const unsigned lanes_log2 = a.slice_log2 - 4, tokens = 256u >> lanes_log2;  // side by side
            const unsigned piece = ((slice < half ? slice : slice - half) << a.slice_log2) + (threadIdx.x & ((1u << lanes_log2) - 1)) * 16;
            const unsigned mine = threadIdx.x >> lanes_log2;
            // a token's bytes, or nullptr where it is in no page
            auto at = [&](unsigned token) -> char* {
                const Quotient p = divide(token, a.pages);
                const int page = p.q < (unsigned)a.max_pages ? table[p.q] : -1;
                return (unsigned)page < (unsigned)a.num_pages ? cache + (((size_t)page * a.kv_heads.d + h) * a.page_size + p.r) * a.row_bytes + piece : nullptr;
            };
            u32x4 x[kMoveAhead];
            char* to[kMoveAhead];
            auto read = [&](unsigned first) {
#pragma unroll
                for (int u = 0; u < kMoveAhead; ++u) {
                    const unsigned i = first + u * tokens + mine;
                    const int from = i < keep && piece < (unsigned)a.row_bytes ? kept[i] : -1;
                    const char* whence = nullptr;
                    to[u] = nullptr;
                    if (from >= 0 && (unsigned)from != i) {
                        whence = at((unsigned)from);
                        to[u] = at(i);
                    }
                    if (!whence) to[u] = nullptr;
                    if (to[u]) x[u] = *reinterpret_cast<const u32x4*>(whence);
                }
            };
            read(0);
            for (unsigned first = 0; first < keep; first += tokens * kMoveAhead) {
                u32x4 y[kMoveAhead];
                char* p[kMoveAhead];
#pragma unroll
                for (int u = 0; u < kMoveAhead; ++u) {
                    y[u] = x[u];
                    p[u] = to[u];
                }
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                if (first + tokens * kMoveAhead < keep) read(first + tokens * kMoveAhead);
#pragma unroll
                for (int u = 0; u < kMoveAhead; ++u)
                    if (p[u]) put16(p[u], y[u]);
            }
        }
    } else if (slice == a.slices.d - 1 && h == 0 && threadIdx.x == 0) {
        put_int(a.past_out + seq, (int)min(max((int64_t)a.past[seq], (int64_t)0), (int64_t)min(keep, a.places)));
    }
    hook_exit(a.notifier, a.job_id);
}

// ------------------------------------------------------------------------------------------ host

using BoundsKernel = void (*)(BoundsArgs);
BoundsKernel bounds_kernel(int dtype) {
    return dtype == PAELLA_F32 ? page_bounds_kernel<F32> : dtype == PAELLA_BF16 ? page_bounds_kernel<Bf16> : page_bounds_kernel<F16>;
}

struct BoundsGrid {
    int64_t touched, items;
    unsigned grid() const { return (unsigned)((items + 3) / 4); }
};
BoundsGrid bounds_grid(const paella_kv_cache* c, const paella_kv_batch* b) {
    BoundsGrid g;
    g.touched = std::min<int64_t>(ceil_div(std::min(b->max_new, b->tokens) - 1, c->page_size) + 1, b->max_pages);
    g.items = (int64_t)b->sequences * g.touched * c->kv_heads;
    return g;
}

int bounds_check(const paella_kv_cache* c, const paella_kv_batch* b) {
    if (!cache_extents_ok(c) || !batch_extents_ok(b)) return PAELLA_EINVAL;
    return (double)b->sequences * bounds_grid(c, b).touched * c->kv_heads / 4 <= kMostWorkgroups - 1 ? 0 : PAELLA_ENOSUP;
}

using SelectKernel = void (*)(SelectArgs);
template <typename T>
SelectKernel screen_kernel_of(int dim) { return dim == 64 ? page_screen_kernel<T, 64> : dim == 128 ? page_screen_kernel<T, 128> : page_screen_kernel<T, 256>; }
SelectKernel screen_kernel(const paella_page_select_plan* p) {
    return p->dtype == PAELLA_F32 ? screen_kernel_of<F32>(p->head_dim) : p->dtype == PAELLA_BF16 ? screen_kernel_of<Bf16>(p->head_dim) : screen_kernel_of<F16>(p->head_dim);
}

// A kernel of one of these forms, by how many there are to pick from at most: with their keys in registers, or, beyond what the registers of 16 waves hold, read again for every pass.
template <typename Kernel>
struct PickForm {
    Kernel kernel;
    unsigned threads;
};
PickForm<SelectKernel> page_pick(int64_t n) {
    if (n <= 1024) return {page_pick_kernel<4, 4>, 256};
    if (n <= 4096) return {page_pick_kernel<16, 4>, 1024};
    if (n <= 16384) return {page_pick_kernel<16, 16>, 1024};
    return {page_pick_kernel<16, 0>, 1024};
}
using EvictKernel = void (*)(EvictArgs);
PickForm<EvictKernel> evict_pick(int64_t n) {
    if (n <= 1024) return {evict_pick_kernel<4, 4>, 256};
    if (n <= 4096) return {evict_pick_kernel<16, 4>, 1024};
    if (n <= 16384) return {evict_pick_kernel<16, 16>, 1024};
    return {evict_pick_kernel<16, 0>, 1024};
}

int64_t select_pages(const paella_page_select_plan* p) { return ceil_div(p->prefix_len, p->page_size) + p->max_pages; }

bool select_plan_ok(const paella_page_select_plan* p) {
    if (!p || !planned_extents_ok(p) || p->count <= 0 || p->first < 0 || p->last < 1 || (int64_t)p->first + p->last > p->count || p->splits <= 0) return false;
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return false;
    const double rows = (double)p->tokens * p->kv_heads;
    return rows * p->splits <= kMostWorkgroups && rows * p->count < 2147483648.0 && select_pages(p) < (1 << 30);
}

size_t select_pitch(const paella_page_select_plan* p) { return (size_t)(select_pages(p) + 15) / 16 * 16; }
size_t select_workspace(const paella_page_select_plan* p) { return (size_t)p->tokens * p->kv_heads * select_pitch(p) * 8; }

// Bytes of a row that a workgroup moves.
int evict_slice_log2(const paella_kv_cache* c) {
    (void)c;
    return 6;
}
int64_t evict_slices(const paella_kv_cache* c) { return 2 * ceil_div((int64_t)c->head_dim * element_bytes(c->dtype), 1 << evict_slice_log2(c)) + 1; }

int evict_check(const paella_kv_evict_desc* d, const paella_kv_cache* c) {
    if (!d || !cache_extents_ok(c) || d->sequences <= 0 || d->max_pages <= 0 || d->keep <= 0 || d->first < 0 || d->recent < 0 || (int64_t)d->first + d->recent > d->keep) return PAELLA_EINVAL;
    const double heads = (double)d->sequences * c->kv_heads;
    if ((double)d->max_pages * c->page_size >= 1073741824.0 || heads * evict_slices(c) > kMostWorkgroups || (double)d->sequences * d->max_pages >= 2147483648.0) return PAELLA_ENOSUP;
    return 0;
}

}  // namespace

extern "C" {

int paella_page_bounds_dims(const paella_kv_cache* c, const paella_kv_batch* b, paella_launch_dims* dims) {
    if (int rc = bounds_check(c, b)) return rc;
    if (!dims) return PAELLA_EINVAL;
    set_launch_dims(dims, bounds_grid(c, b).grid(), 256, 0, 64);
    loaded_dims((const void*)bounds_kernel(c->dtype), dims);
    return 0;
}

int paella_page_bounds_launch(const paella_kv_cache* c, const paella_kv_batch* b, void* bounds, void* stream, uint32_t job_id, void* notifier) {
    if (int rc = bounds_check(c, b)) return rc;
    if (!cache_ok(c) || !batch_ok(b) || !bounds || ((uintptr_t)bounds & 15)) return PAELLA_EINVAL;
    const double bytes = 2.0 * c->num_pages * c->kv_heads * c->head_dim * element_bytes(c->dtype);
    if (over_cache(c, bounds, bytes) || over_batch(b, c->page_size, bounds, bytes)) return PAELLA_EINVAL;
    const BoundsGrid g = bounds_grid(c, b);
    BoundsArgs a;
    a.k_cache = (const char*)c->k; a.bounds = (char*)bounds;
    a.starts = b->starts; a.past = b->past; a.tables = b->tables;
    a.sequences = b->sequences; a.max_new = b->max_new; a.tokens = b->tokens; a.max_pages = b->max_pages; a.num_pages = c->num_pages; a.page_size = c->page_size;
    a.row_bytes = c->head_dim * element_bytes(c->dtype); a.pieces = a.row_bytes / 16; a.group_log2 = 0;
    while ((1 << a.group_log2) < a.pieces && a.group_log2 < 6) ++a.group_log2;
    a.kv_heads = divisor((unsigned)c->kv_heads); a.touched = divisor((unsigned)g.touched); a.items = (unsigned)g.items;
    a.job_id = job_id; a.notifier = (Notifier*)notifier;
    launch(bounds_kernel(c->dtype), dim3(g.grid()), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

int paella_page_select_plan_make(const paella_kv_cache* c, const paella_kv_batch* b, int heads, int count, int first, int last, paella_page_select_plan* p) {
    if (!p || !cache_extents_ok(c) || !batch_extents_ok(b) || heads <= 0 || heads % c->kv_heads || count <= 0 || first < 0 || last < 1 || (int64_t)first + last > count) return PAELLA_EINVAL;
    *p = paella_page_select_plan{};
    plan_extents(p, c, b, heads);
    p->count = count; p->first = first; p->last = last;
    const int64_t pages = select_pages(p), rows = (int64_t)p->tokens * p->kv_heads;
    // enough workgroups to fill the device, none without a turn for each wave
    p->splits = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(2048, rows), ceil_div(pages, 4 * kScreened)));
    if (!select_plan_ok(p)) return PAELLA_ENOSUP;
    p->stages = 2;
    p->workspace_bytes = select_workspace(p);
    set_launch_dims(&p->dims, (unsigned)(rows * p->splits), 256, 0, 128);
    const double size = element_bytes(c->dtype);
    p->flops = 4.0 * p->tokens * p->heads * pages * p->head_dim;
    p->bytes = 2.0 * (pages - p->max_pages + (double)p->sequences * p->max_pages) * p->kv_heads * p->head_dim * size + (double)p->tokens * p->heads * p->head_dim * size + 4.0 * rows * count;
    return 0;
}

int paella_page_select_dims(const paella_page_select_plan* p, int stage, paella_launch_dims* dims) {
    if (!select_plan_ok(p) || !dims || stage < 0 || stage > 1) return PAELLA_EINVAL;
    const auto pick = page_pick(select_pages(p));
    if (stage) set_launch_dims(dims, (unsigned)(p->tokens * p->kv_heads), pick.threads, 0, 64);
    else set_launch_dims(dims, (unsigned)(p->tokens * p->kv_heads * p->splits), 256, 0, 128);
    loaded_dims(stage ? (const void*)pick.kernel : (const void*)screen_kernel(p), dims);
    return 0;
}

int paella_page_select_launch_stage(const paella_page_select_plan* p, int stage, const paella_kv_cache* c, const paella_kv_batch* b, const void* q, int64_t q_stride,
                                    const void* bounds, int32_t* pages, void* workspace, void* stream, uint32_t job_id, void* notifier) {
    if (!select_plan_ok(p) || stage < 0 || stage > 1 || !planned_for(p, c, b) || !q || !bounds || !pages || !workspace) return PAELLA_EINVAL;
    const int64_t size = element_bytes(c->dtype), row = (int64_t)p->heads * p->head_dim;
    if (q_stride < row || q_stride % 8 || (((uintptr_t)q | (uintptr_t)bounds | (uintptr_t)workspace) & 15) || ((uintptr_t)pages & 3)) return PAELLA_EINVAL;
    const double out_bytes = 4.0 * p->tokens * p->kv_heads * p->count, space = (double)select_workspace(p);
    const double bound_bytes = 2.0 * c->num_pages * c->kv_heads * c->head_dim * size;
    const struct { const void* at; double bytes; } outs[2] = {{pages, out_bytes}, {workspace, space}};
    for (const auto& o : outs)
        if (rows_overlap(q, p->tokens, q_stride * size, row * size, o.at, o.bytes) || overlap(bounds, bound_bytes, o.at, o.bytes) || over_batch(b, c->page_size, o.at, o.bytes)) return PAELLA_EINVAL;
    if (overlap(pages, out_bytes, workspace, space)) return PAELLA_EINVAL;
    SelectArgs a;
    a.q = (const char*)q; a.bounds = (const char*)bounds;
    a.starts = b->starts; a.past = b->past; a.tables = b->tables; a.prefix_table = b->prefix_table;
    a.entries = (f32x2*)workspace; a.pages = pages; a.q_stride = q_stride * size;
    a.sequences = b->sequences; a.tokens = b->tokens; a.max_pages = b->max_pages; a.prefix_pages = (int)ceil_div(b->prefix_len, c->page_size); a.num_pages = c->num_pages;
    a.heads = p->heads; a.first = p->first; a.last = p->last; a.count = p->count; a.dim = p->head_dim; a.dtype = p->dtype; a.pitch = (unsigned)select_pitch(p);
    a.max_new = divisor((unsigned)b->max_new); a.kv_heads = divisor((unsigned)p->kv_heads); a.splits = divisor((unsigned)p->splits); a.page_size = divisor((unsigned)c->page_size);
    a.job_id = job_id; a.notifier = (Notifier*)notifier;
    const unsigned rows = (unsigned)(p->tokens * p->kv_heads);
    if (stage == 0) {
        launch(screen_kernel(p), dim3(rows * (unsigned)p->splits), dim3(256), 0, (hipStream_t)stream, a);
    } else {
        const auto pick = page_pick(select_pages(p));
        launch(pick.kernel, dim3(rows), dim3(pick.threads), 0, (hipStream_t)stream, a);
    }
    return (int)hipGetLastError();
}

int paella_page_select_launch(const paella_page_select_plan* p, const paella_kv_cache* c, const paella_kv_batch* b, const void* q, int64_t q_stride, const void* bounds,
                              int32_t* pages, void* workspace, void* stream, uint32_t job_id, void* notifier) {
    if (!select_plan_ok(p)) return PAELLA_EINVAL;
    if (keeps_no_order(stream)) return PAELLA_ENOSUP;
    if (int rc = paella_page_select_launch_stage(p, 0, c, b, q, q_stride, bounds, pages, workspace, stream, job_id, nullptr)) return rc;
    return paella_page_select_launch_stage(p, 1, c, b, q, q_stride, bounds, pages, workspace, stream, job_id, notifier);
}

int paella_kv_evict_dims(const paella_kv_evict_desc* d, const paella_kv_cache* c, int stage, paella_launch_dims* dims) {
    if (int rc = evict_check(d, c)) return rc;
    if (!dims || stage < 0 || stage > 1) return PAELLA_EINVAL;
    if (stage) set_launch_dims(dims, (unsigned)(d->sequences * c->kv_heads * evict_slices(c)), 256, 0, 64);
    const auto pick = evict_pick((int64_t)d->max_pages * c->page_size);
    if (!stage) set_launch_dims(dims, (unsigned)(d->sequences * c->kv_heads), pick.threads, 0, 64);
    loaded_dims(stage ? (const void*)evict_move_kernel : (const void*)pick.kernel, dims);
    return 0;
}

int paella_kv_evict_launch_stage(const paella_kv_evict_desc* d, int stage, const paella_kv_cache* c, float* weights, const int32_t* past, const int32_t* tables, int32_t* kept,
                                 int32_t* past_out, void* stream, uint32_t job_id, void* notifier) {
    if (int rc = evict_check(d, c)) return rc;
    if (stage < 0 || stage > 1 || !cache_ok(c) || !weights || !past || !tables || !kept || !past_out) return PAELLA_EINVAL;
    const double heads = (double)d->sequences * c->kv_heads, kept_bytes = heads * d->keep * 4, weight_bytes = heads * d->max_pages * c->page_size * 4;
    const double table_bytes = (double)d->sequences * d->max_pages * 4, past_bytes = (double)d->sequences * 4;
    const struct { const void* at; double bytes; } outs[3] = {{kept, kept_bytes}, {past_out, past_bytes}, {weights, weight_bytes}};
    for (const auto& o : outs)
        if (overlap(tables, table_bytes, o.at, o.bytes) || over_cache(c, o.at, o.bytes) || (o.at != past_out && overlap(past, past_bytes, o.at, o.bytes))) return PAELLA_EINVAL;
    if (past_out != past && overlap(past, past_bytes, past_out, past_bytes)) return PAELLA_EINVAL;
    if (overlap(kept, kept_bytes, past_out, past_bytes) || overlap(kept, kept_bytes, weights, weight_bytes) || overlap(past_out, past_bytes, weights, weight_bytes) ||
        over_cache(c, past, past_bytes) || over_cache(c, tables, table_bytes))
        return PAELLA_EINVAL;
    EvictArgs a;
    a.k_cache = (char*)c->k; a.v_cache = (char*)c->v; a.weights = weights; a.past = past; a.tables = tables; a.kept = kept; a.past_out = past_out;
    a.sequences = d->sequences; a.max_pages = d->max_pages; a.num_pages = c->num_pages; a.page_size = c->page_size; a.row_bytes = c->head_dim * element_bytes(c->dtype);
    a.keep = d->keep; a.first = d->first; a.recent = d->recent; a.places = (unsigned)(d->max_pages * c->page_size);
    a.kv_heads = divisor((unsigned)c->kv_heads); a.slices = divisor((unsigned)evict_slices(c)); a.pages = divisor((unsigned)c->page_size);
    a.job_id = job_id; a.notifier = (Notifier*)notifier;
    a.slice_log2 = (unsigned)evict_slice_log2(c);
    const auto pick = evict_pick((int64_t)a.places);
    if (stage == 0) launch(pick.kernel, dim3((unsigned)(d->sequences * c->kv_heads)), dim3(pick.threads), 0, (hipStream_t)stream, a);
    else launch(evict_move_kernel, dim3((unsigned)(d->sequences * c->kv_heads * evict_slices(c))), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

int paella_kv_evict_launch(const paella_kv_evict_desc* d, const paella_kv_cache* c, float* weights, const int32_t* past, const int32_t* tables, int32_t* kept, int32_t* past_out,
                           void* stream, uint32_t job_id, void* notifier) {
    if (int rc = evict_check(d, c)) return rc;
    if (keeps_no_order(stream)) return PAELLA_ENOSUP;
    if (int rc = paella_kv_evict_launch_stage(d, 0, c, weights, past, tables, kept, past_out, stream, job_id, nullptr)) return rc;
    return paella_kv_evict_launch_stage(d, 1, c, weights, past, tables, kept, past_out, stream, job_id, notifier);
}

}  // extern "C"
