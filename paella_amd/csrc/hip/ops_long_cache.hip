// Operators that keep a long paged cache from being read and kept whole: bounds of the pages' keys, the selection of pages by them, and eviction.
// (Attention over the pages and the weights that tokens gather: long_attention.h.)

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "long_attention.h"
#include "long_common.h"
#include "pick_largest.h"
#include "prefix_attention.h"

namespace {

using namespace paella;

// ------------------------------------------------------------------------------------------ bounds of a page's keys
// A wave per page and key head, or some of its key heads: 16 bytes of a key per lane, as many keys side by side as fit the wave, four or eight requests at a time.  Bound by memory:
// each key of the pages is read once.
struct BoundsArgs {
    const char* k_cache;
    char* bounds;
    const int *starts, *past, *tables;
    int sequences, max_new, tokens, max_pages, num_pages, page_size, row_bytes, pieces, group_log2;  // pieces: 16 bytes of a key each; 2^group_log2 lanes side by side for a key
    int kv_heads;
    Divisor groups, touched;  // groups: of a page's key heads; touched: most pages that a sequence's new tokens lie in
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

// Of numbers: by comparison, since the library's minimum makes every operand canonical first.
__device__ __forceinline__ float lesser(float v, float w) { return v < w ? v : w; }
__device__ __forceinline__ float greater(float v, float w) { return v > w ? v : w; }

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

// Least and largest of the lanes that are multiples of 2^log2 apart, by the vector unit's own lane moves (some meet more than once).
template <int V>
__device__ __forceinline__ void lanes_apart(float (&low)[V], float (&high)[V], int log2) {
    auto meet = [&](auto other) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            low[e] = lesser(other(low[e]), low[e]);
            high[e] = greater(other(high[e]), high[e]);
        }
    };
    if (log2 <= 0) meet([](float v) { return lane_move<0xB1>(v); });   // lane ^ 1
    if (log2 <= 1) meet([](float v) { return lane_move<0x4E>(v); });   // lane ^ 2
    if (log2 <= 2) meet([](float v) { return lane_move<0x124>(v); });  // a quarter of a turn of sixteen, and half of one
    if (log2 <= 3) meet([](float v) { return lane_move<0x128>(v); });
    auto swapped = [&](auto swap) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const auto l = swap(as_word(low[e])), h = swap(as_word(high[e]));
            low[e] = lesser(as_float(l[0]), as_float(l[1]));
            high[e] = greater(as_float(h[0]), as_float(h[1]));
        }
    };
    if (log2 <= 4) swapped([](unsigned v) { return __builtin_amdgcn_permlane16_swap(v, v, false, false); });  // even and odd sixteens
    if (log2 <= 5) swapped([](unsigned v) { return __builtin_amdgcn_permlane32_swap(v, v, false, false); });  // both halves
}

// AHEAD: requests of a lane for a head that go out together; HEADS: key heads of a wave, which lie side by side in the page.
template <typename T, int AHEAD, int HEADS>
__global__ __launch_bounds__(256, AHEAD * HEADS == 4 && HEADS < 4 ? 8 : 1) void page_bounds_kernel(BoundsArgs a) {
    hook_entry(a.notifier, a.job_id);
    constexpr int V = 16 / T::bytes;
    const int lane = threadIdx.x & 63;
    const unsigned item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (item < a.items) {
        const Quotient by_head = divide(item, a.groups), by_page = divide(by_head.q, a.touched);
        const int seq = (int)by_page.q;
        const NewTokens its = new_tokens(a.starts, a.past, seq, a.max_new, a.tokens);
        const unsigned page = (unsigned)its.past / (unsigned)a.page_size + by_page.r;  // along the sequence
        const int64_t first = (int64_t)page * a.page_size, end = (int64_t)its.past + its.count;
        int physical = -1;
        if (its.count > 0 && first < end && page < (unsigned)a.max_pages) physical = __builtin_amdgcn_readfirstlane(a.tables[(size_t)seq * a.max_pages + page]);
        if ((unsigned)physical < (unsigned)a.num_pages) {
            const int held = (int)min((int64_t)a.page_size, end - first);
            const int heads = min(a.kv_heads - (int)by_head.r * HEADS, HEADS);
            const size_t head_at = (size_t)physical * a.kv_heads + by_head.r * HEADS;
            const char* const keys = a.k_cache + head_at * a.page_size * a.row_bytes;
            const __amdgpu_buffer_rsrc_t to = descriptor(a.bounds + head_at * 2 * a.row_bytes);
            const size_t head_bytes = (size_t)a.page_size * a.row_bytes;
            const int group = 1 << a.group_log2, each = 64 >> a.group_log2;
            for (int piece = lane & (group - 1); piece < (a.pieces + group - 1) / group * group; piece += group) {  // (whole waves: lanes of all groups meet below)
                const bool in = piece < a.pieces;
                float low[HEADS][V], high[HEADS][V];
#pragma unroll
                for (int h = 0; h < HEADS; ++h)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        low[h][e] = INFINITY;
                        high[h][e] = -INFINITY;
                    }
                for (int key = lane >> a.group_log2; key < held; key += AHEAD * each) {
                    u32x4 w[HEADS][AHEAD];
#pragma unroll
                    for (int h = 0; h < HEADS; ++h)
#pragma unroll
                        for (int u = 0; u < AHEAD; ++u)  // behind the last key, and the last head: the last one again
                            w[h][u] = *reinterpret_cast<const u32x4*>(keys + min(h, heads - 1) * head_bytes + (size_t)min(key + u * each, held - 1) * a.row_bytes + (in ? piece : 0) * 16);
#pragma unroll
                    for (int h = 0; h < HEADS; ++h)
#pragma unroll
                        for (int u = 0; u < AHEAD; ++u) widen<T>(w[h][u], low[h], high[h]);
                }
#pragma unroll
                for (int h = 0; h < HEADS; ++h) {
                    if (h >= heads) break;
                    lanes_apart<V>(low[h], high[h], a.group_log2);
                    if (lane < group && in) {
                        __builtin_amdgcn_raw_buffer_store_b128(packed<T>(low[h]), to, 2 * h * a.row_bytes + piece * 16, 0, kThrough);
                        __builtin_amdgcn_raw_buffer_store_b128(packed<T>(high[h]), to, (2 * h + 1) * a.row_bytes + piece * 16, 0, kThrough);
                    }
                }
            }
        }
    }
    hook_exit(a.notifier, a.job_id);
}

// ------------------------------------------------------------------------------------------ selection of pages
// worth(e) = max over the key head's query heads of sum_d max(q_d low_d, q_d high_d) = q+ . high + q- . low, q+ and q- the values above and below 0.  Which of two neighbours is taken is decided by their last
// digits, in 64 bits; but nearly all pages are far from the border.  So the matrix units take the worths in 32 bits, at the rate that memory delivers the bounds, together with how far each can
// be off: of a sum of 2 D products, half of them 0, by (2 D + 8) * 2^-24 of the sum of their magnitudes, q+ . |high| - q- . |low|.  Pages that are further from the border than
// that are decided; the few others, if they are not all taken or none of them, get their worths in 64 bits.  (All of them in 64 bits by the vector unit: 58 us for 32 rows of 1024 pages of 8 heads of 128 in bf16, 100 MB.)
constexpr int kCounterStride = 32;  // a cache line each

struct SelectArgs {
    const char *q, *bounds;
    const int *starts, *past, *tables, *prefix_table;
    unsigned* counters;          // [tokens][kv_heads][kCounterStride], zero between launches
    unsigned* entries;           // [tokens][kv_heads][pitch]
    float* errors;               // [tokens][kv_heads][4 * splits]: how far the worths can be off, over (2 D + 8) * 2^-24
    unsigned long long* worths;  // [tokens][kv_heads][pitch]
    int* pages;
    int64_t q_stride;  // bytes
    int sequences, tokens, max_pages, prefix_pages, num_pages, heads, first, last, count, dim, dtype;
    unsigned pitch;
    Divisor max_new, kv_heads, per_kv, splits, tiles, page_size;  // tiles: of a sequence's new tokens
    uint32_t job_id;
    Notifier* notifier;
};

// A page's entry: its worth as a number whose order is the worths', or
constexpr unsigned kNoPage = 0, kUnknown = 1, kForced = ~0u;  // (unknown: it is no number, or may be infinite)

__device__ __forceinline__ int page_along(const SelectArgs& a, int seq, unsigned e) {
    return *(e < (unsigned)a.prefix_pages ? a.prefix_table + e : a.tables + (size_t)seq * a.max_pages + (e - a.prefix_pages));  // (one load: two that meet are waited for)
}

// Values below 0, and magnitudes, of 16 bytes.
template <typename T> __device__ __forceinline__ u32x4 below_zero(u32x4 q) {
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] &= T::bytes == 4 ? (unsigned)((int)q[e] >> 31) : (q[e] >> 15 & 0x00010001u) * 0xFFFFu;
    return q;
}
template <typename T> __device__ __forceinline__ u32x4 magnitude(u32x4 v) { return v & (T::bytes == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu); }

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

constexpr int kScreened = 16;  // pages of a wave's turn

// New tokens of a sequence whose heads for one key head make up a tile of 16 rows: the bounds are read once for all of them.
__host__ __device__ constexpr int tokens_of_tile(int heads) { return heads >= 16 ? 1 : 16 / heads; }

// What a workgroup of the screen works on: the tile's tokens from j0 on, for one key head, and its part of their pages.
struct Screened {
    int h, seq, j0, n, split;
    NewTokens its;
    __device__ __forceinline__ explicit Screened(const SelectArgs& a) {
        const Quotient by_head = divide(blockIdx.x, a.kv_heads), by_split = divide(by_head.q, a.splits), by_tile = divide(by_split.q, a.tiles);
        const int each = tokens_of_tile((int)a.per_kv.d);
        h = (int)by_head.r;
        split = (int)by_split.r;
        seq = (int)by_tile.q;
        j0 = (int)by_tile.r * each;
        its = new_tokens(a.starts, a.past, seq, (int)a.max_new.d, a.tokens);
        n = min(its.count - j0, each);
    }
    __device__ __forceinline__ unsigned pages(const SelectArgs& a, int j) const {
        return (unsigned)a.prefix_pages + (unsigned)own_pages(its.past, j0 + j, a.page_size, a.max_pages);
    }
};

// A turn's bounds go to registers while the ones before are worked on, and the numbers of the pages behind them.  entry(j, e, key) and error(j, slot, worst) take what is left of page e for the tile's
// token j, and of all of a wave's.
template <typename T, int D, typename Entry, typename Error>
__device__ __forceinline__ void screen_pages(const SelectArgs& a, const Screened& w, Entry entry, Error error_of) {
    constexpr int ROW = D * T::bytes, KC = ROW / 64;
    const int lane = threadIdx.x & 63, mm = lane & 15, group = lane >> 4, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int h = w.h, seq = w.seq, heads = (int)a.per_kv.d, j0 = w.j0, n = w.n;
    const NewTokens& its = w.its;
    auto pages_of = [&](int j) { return w.pages(a, j); };
    const unsigned pages = n > 0 ? pages_of(n - 1) : 0u, step = a.splits.d * 4;
    unsigned turn = (unsigned)w.split * 4 + wave;
    float worst = 0.f;
    if (turn * kScreened < pages) {
        const Quotient row = divide((unsigned)min(mm, n * heads - 1), a.per_kv);  // the lane's token and head
        // Numbers of the pages of four turns, 16 each, and of the four behind.  (A request that follows others is answered after them: looked up turn by turn, pages would have each turn's bounds wait for
        // those of the one before.)
        auto look = [&](unsigned turn) { return page_along(a, seq, min((turn + group * step) * kScreened + mm, pages - 1)); };
        int numbers = look(turn), numbers_behind = look(turn + 4 * step), left = 4;
        auto next_page = [&](unsigned turn) {  // of the turns one after the other
            if (left == 0) {
                numbers = numbers_behind;
                numbers_behind = look(turn + 4 * step);
                left = 4;
            }
            return __shfl(numbers, (4 - left--) * 16 + mm, 64);
        };
        auto load = [&](int page, u32x4 (&low)[KC], u32x4 (&high)[KC]) {
            const char* const from = a.bounds + ((size_t)((unsigned)page < (unsigned)a.num_pages ? page : 0) * a.kv_heads.d + h) * 2 * ROW + group * 16;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                low[c] = *reinterpret_cast<const u32x4*>(from + c * 64);
                high[c] = *reinterpret_cast<const u32x4*>(from + ROW + c * 64);
            }
        };
        u32x4 low[KC], high[KC], above[KC], below[KC];  // of the queries: values above 0 and below it
        auto query = [&](int g) {
            const int head = heads > 16 ? min(g + mm, heads - 1) : (int)row.r;
            const char* const from = a.q + (size_t)(its.first + j0 + (heads > 16 ? 0 : (int)row.q)) * a.q_stride + (size_t)(h * heads + head) * ROW + group * 16;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const u32x4 q = *reinterpret_cast<const u32x4*>(from + c * 64);
                below[c] = below_zero<T>(q);
                above[c] = q ^ below[c];
            }
        };
        int page = next_page(turn);
        load(page, low, high);
        query(0);
        const bool one_group = n * heads <= 4;  // the first lane group has all rows
        auto work = [&]() {
            // Lane mm has page mm, register e of lane group g row 4 g + e.
            f32x4 worth = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, error = {0.f, 0.f, 0.f, 0.f};
            for (int g = 0; g < heads; g += 16) {  // more than once where a token has more heads than a tile rows
                if (heads > 16) query(g);
                f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x, z = x;
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    x = multiply<T>(above[c], high[c], x);
                    x = multiply<T>(below[c], low[c], x);
                    y = multiply<T>(above[c], magnitude<T>(high[c]), y);
                    z = multiply<T>(below[c], magnitude<T>(low[c]), z);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float off = y[e] - z[e];
                    worth[e] = fmaxf(worth[e], x[e]);
                    error[e] = fmaxf(error[e], off < 1e38f ? off : INFINITY);  // (below it no sum on the way was infinite either)
                    if (off < 1e38f) worst = fmaxf(worst, off);
                }
            }
            const unsigned e = turn * kScreened + mm;
            for (int j = 0; j < n; ++j) {
                f32x2 mine = {-INFINITY, 0.f};  // worth, and how far it can be off
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // the token's rows
                    const int r = group * 4 + i;
                    const bool ours = heads > 16 || (r >= j * heads && r < (j + 1) * heads);
                    mine.x = fmaxf(mine.x, ours ? worth[i] : -INFINITY);
                    mine.y = fmaxf(mine.y, ours ? error[i] : 0.f);
                }
                if (!one_group) {
#pragma unroll
                    for (int off = 16; off < 64; off <<= 1) {
                        mine.x = fmaxf(mine.x, __shfl_xor(mine.x, off, 64));
                        mine.y = fmaxf(mine.y, __shfl_xor(mine.y, off, 64));
                    }
                }
                const unsigned seen = pages_of(j);
                unsigned key = mine.y < INFINITY ? number_key(mine.x, kUnknown) : kUnknown;
                if (e < (unsigned)a.first || e + a.last >= seen) key = kForced;
                if ((unsigned)page >= (unsigned)a.num_pages) key = kNoPage;
                if (group == 0 && e < seen) entry(j, e, key);
            }
        };
        // (The next turn's bounds are requested whatever comes, or not at all: a request that may not have been made turns every wait for older ones into one for all.)
        for (; (turn + step) * kScreened < pages; turn += step) {
            const int page_next = next_page(turn + step);
            if constexpr (KC <= 8) {
                u32x4 next_low[KC], next_high[KC];
                load(page_next, next_low, next_high);
                work();
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    low[c] = next_low[c];
                    high[c] = next_high[c];
                }
            } else {
                work();
                load(page_next, low, high);
            }
            page = page_next;
        }
        work();
    }
    worst = wave_max_f(worst);  // of all rows of the tile
    if (lane < n) error_of(lane, (unsigned)w.split * 4 + wave, worst);
}

// A page's worth in 64 bits, by a whole wave: 16 bytes of a row per lane, the bounds and G heads' queries requested together.
template <typename T, int G>
__device__ __forceinline__ unsigned long long exact_worth_of(const SelectArgs& a, int t, int seq, int h, unsigned e) {
    constexpr int V = 16 / T::bytes;
    const int lane = threadIdx.x & 63, heads = (int)a.per_kv.d, row = a.dim * T::bytes;
    const int at = min(lane * 16, row - 16);
    const char* const q = a.q + t * a.q_stride + (size_t)h * heads * row + at;
    const unsigned page = (unsigned)page_along(a, seq, e);  // (outside the cache only if entries are another call's)
    const char* const from = a.bounds + ((size_t)(page < (unsigned)a.num_pages ? page : 0u) * a.kv_heads.d + h) * 2 * row + at;
    const u32x4 low = *reinterpret_cast<const u32x4*>(from), high = *reinterpret_cast<const u32x4*>(from + row);
    unsigned long long best = 0;
    for (int g = 0; g < heads; g += G) {
        u32x4 x[G];
        double sum[G];
#pragma unroll
        for (int i = 0; i < G; ++i) x[i] = *reinterpret_cast<const u32x4*>(q + (size_t)min(g + i, heads - 1) * row);
#pragma unroll
        for (int i = 0; i < G; ++i) {
            sum[i] = 0.0;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                auto value = [&](u32x4 w) {
                    if constexpr (T::bytes == 4) return (double)as_float(w[v]);
                    else return (double)(v & 1 ? unpack2<T>(w[v / 2]).y : unpack2<T>(w[v / 2]).x);
                };
                const double l = value(x[i]) * value(low), r = value(x[i]) * value(high);
                sum[i] += l > r || l != l ? l : r;
            }
            sum[i] = lane * 16 < row ? sum[i] : 0.0;
            sum[i] = row_all(sum[i], Sum());
#pragma unroll
            for (int off = 16; off < 64; off <<= 1) {
                const unsigned long long b = __builtin_bit_cast(unsigned long long, sum[i]);
                sum[i] += __builtin_bit_cast(double, (unsigned long long)(unsigned)__shfl_xor((int)(unsigned)(b >> 32), off, 64) << 32 | (unsigned)__shfl_xor((int)(unsigned)b, off, 64));
            }
            best = max(best, number_key(sum[i], number_key((double)INFINITY, 0ull)));  // a worth that is no number counts as the largest
        }
    }
    return best;
}
template <int G>
__device__ __forceinline__ unsigned long long exact_worth(const SelectArgs& a, int t, int seq, int h, unsigned e) {
    return a.dtype == PAELLA_F32 ? exact_worth_of<F32, G>(a, t, seq, h, e) : a.dtype == PAELLA_BF16 ? exact_worth_of<Bf16, G>(a, t, seq, h, e) : exact_worth_of<F16, G>(a, t, seq, h, e);
}

__device__ __forceinline__ void put_int(int* p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

constexpr unsigned kOpen = 256;  // pages whose worths in 64 bits are ranked against each other

template <int WAVES>
struct PageSpace {
    PickSpace<WAVES> pick;
    unsigned forced[WAVES], unknown[WAVES], inside[WAVES], open[WAVES];
    float error[WAVES];
    unsigned list[kOpen];
    unsigned long long worth[kOpen];
};

// The row's pages by their entries, load(i).  error: this thread's share of the screen's.  KEYS as in Span.
template <int WAVES, int KEYS, typename Load>
__device__ __forceinline__ void pick_pages(const SelectArgs& a, int t, int seq, int h, unsigned pages, float error, PageSpace<WAVES>& s, Load load) {
    const size_t row = (size_t)t * a.kv_heads.d + h;
    unsigned long long* const worths = a.worths + row * a.pitch;
    int* const to = a.pages + row * a.count;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const Span<WAVES, KEYS> span(pages);
    unsigned held[KEYS ? KEYS : 1];
    span.hold(held, load, [](unsigned k) { return k; });
    auto get = [&](int u, unsigned i) { return KEYS ? held[u] : load(i); };
    auto known = [](unsigned k) { return k - (kUnknown + 1) < kForced - (kUnknown + 1) ? k : 0u; };
    Range<unsigned> range;
    unsigned forced = 0, unknown = 0;
    span.visit(get, [&](int, unsigned, unsigned k) {
        forced += wave_count(k == kForced);
        unknown += wave_count(k == kUnknown);
        range.add(known(k));
    });
    error = wave_max_f(error);
    if (lane == 0) {
        s.forced[wave] = forced;
        s.unknown[wave] = unknown;
        s.error[wave] = error;
    }
    range.join(s.pick);
    error = waves_all(s.error, Most());
    forced = uniform(waves_all(s.forced, Sum()));
    unknown = uniform(waves_all(s.unknown, Sum()));
    const unsigned want = (unsigned)a.count - min(forced, (unsigned)a.count);
    // Pages whose entries are above `in` are taken, those below `out` are not, those between are open, and those that nothing is known of as well.
    unsigned in = kForced - 1, out = kForced;
    bool any_unknown = false;
    if (range.some + unknown <= want) {
        in = kNoPage;
    } else if (want) {
        any_unknown = unknown > 0;
        out = 0;
        if (range.some >= want) {
            const float border = key_number(range.some == want ? range.least : find_bound<WAVES, KEYS, unsigned>(span, range, want, s.pick, get).bound);
            const float off = 2.f * (error * (float)(2 * a.dim + 8) * 0x1p-24f + 0x1p-110f);  // (products below the least number of 32 bits are lost, too)
            out = number_key(border - off, 1u);
            if (!unknown) in = number_key(border + off, 1u);  // (a page that nothing is known of may be worth more)
        }
        out = max(out, kUnknown + 1);
    }
    const unsigned width = in >= out ? in - out + 1 : 0;
    auto is_in = [&](unsigned k) { return k > in; };
    auto is_open = [&](unsigned k) { return k - out < width || (any_unknown && k == kUnknown); };
    unsigned inside = 0, open = 0;
    span.visit(get, [&](int, unsigned, unsigned k) {
        inside += wave_count(is_in(k));
        open += wave_count(is_open(k));
    });
    if (lane == 0) {
        s.inside[wave] = inside;
        s.open[wave] = open;
    }
    __syncthreads();
    const unsigned open_ahead = ahead_of(s.open, wave, &open);
    const unsigned inside_ahead = ahead_of(s.inside, wave, &inside);
    auto take = [&](unsigned place, unsigned i) {
        if (place < (unsigned)a.count) put_int(to + place, (int)i);  // (more only if entries are another call's)
    };
    auto none = [](auto) { return false; };
    unsigned taken;
    if (inside + open <= (unsigned)a.count) {
        emit_from(span, inside_ahead + open_ahead, get, [&](unsigned k) { return is_in(k) || is_open(k); }, take);
        taken = inside + open;
    } else {
        // The open pages, in order, a list at a time, whose worths the waves share out.
        for (unsigned first = 0; first < open; first += kOpen) {
            const unsigned n = min(open - first, kOpen);
            auto each_open = [&](auto then) {
                unsigned slot = open_ahead - first;  // (those of other lists are far above n)
                span.visit(get, [&](int u, unsigned i, unsigned k) {
                    const bool mine = is_open(k);
                    const unsigned long long who = __ballot(mine);
                    const unsigned at = slot + (unsigned)__popcll(who & ((1ull << lane) - 1));
                    if (mine && at < n) then(u, i, at);
                    slot += (unsigned)__popcll(who);
                });
            };
            each_open([&](int, unsigned i, unsigned at) { s.list[at] = i; });
            __syncthreads();
            for (unsigned k = wave; k < n; k += WAVES) {
                const unsigned long long worth = exact_worth<WAVES == 16 ? 2 : 4>(a, t, seq, h, uniform(s.list[k]));  // (sixteen waves have 128 registers each)
                if (lane == 0) s.worth[k] = worth;
            }
            __syncthreads();
            if (open <= kOpen && KEYS > 0) {  // all of them: each is ranked against the others
                for (unsigned k = threadIdx.x; k < n; k += WAVES * 64) {
                    const unsigned long long mine = s.worth[k];
                    unsigned before = 0;
                    for (unsigned o = 0; o < n; ++o) before += s.worth[o] > mine || (s.worth[o] == mine && o < k);
                    s.list[k] = before < (unsigned)a.count - inside ? kForced : kNoPage;
                }
                __syncthreads();
                each_open([&](int u, unsigned, unsigned at) { held[u] = s.list[at]; });
            } else {
                // (through to memory, as all that a kernel here writes: on a direct queue nothing writes a cache back behind it, and the workspace may be another tensor's by the time a line leaves the cache)
                for (unsigned k = threadIdx.x; k < n; k += WAVES * 64) __hip_atomic_store(worths + s.list[k], s.worth[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __syncthreads();
            }
        }
        if (open <= kOpen && KEYS > 0) {
            taken = emit(span, s.pick, get, is_in, none, 0u, take);
        } else {  // the worths are in memory, in the pages' places
            const Span<WAVES, 0> all(pages);
            auto key = [&](int, unsigned i) {
                const unsigned k = load(i);
                return is_in(k) ? ~0ull : is_open(k) ? worths[i] : 0ull;
            };
            Range<unsigned long long> keys;
            all.visit(key, [&](int, unsigned, unsigned long long k) { keys.add(k); });
            keys.join(s.pick);
            taken = emit_taken<WAVES, 0, unsigned long long>(all, find_bound<WAVES, 0, unsigned long long>(all, keys, (unsigned)a.count, s.pick, key), s.pick, key, take);
        }
    }
    for (unsigned i = taken + threadIdx.x; i < (unsigned)a.count; i += WAVES * 64) put_int(to + i, -1);
}

template <typename T, int D>
__global__ __launch_bounds__(256) void page_screen_kernel(SelectArgs a) {
    hook_entry(a.notifier, a.job_id);
    const Screened w(a);
    auto row = [&](int j) { return (size_t)(w.its.first + w.j0 + j) * a.kv_heads.d + w.h; };
    screen_pages<T, D>(
        a, w, [&](int j, unsigned e, unsigned key) { __hip_atomic_store(a.entries + row(j) * a.pitch + e, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); },
        [&](int j, unsigned slot, float worst) { store_out(a.errors + row(j) * 4 * a.splits.d + slot, worst); });
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
        const size_t row = (size_t)t * a.kv_heads.d + h;
        const unsigned* const entries = a.entries + row * a.pitch;
        const float* const errors = a.errors + row * 4 * a.splits.d;
        float error = errors[min(threadIdx.x, 4 * a.splits.d - 1)];  // (the last one again behind it)
        for (unsigned i = threadIdx.x + WAVES * 64; i < 4 * a.splits.d; i += WAVES * 64) error = fmaxf(error, errors[i]);
        pick_pages<WAVES, KEYS>(a, t, seq, h, pages, error, space, [&](unsigned i) { return entries[i]; });
    }
    hook_exit(a.notifier, a.job_id);
}

// One launch for both: the workgroup that arrives last at a row picks its pages, while others are still screening.  (Entries are written through ahead of the count, and read past this XCD's
// caches.)  Where a row has one workgroup, its entries stay in LDS.
constexpr int kSelectKeys = 8;  // of a thread: up to 2048 pages

template <typename T, int D>
__global__ __launch_bounds__(256) void page_select_kernel(SelectArgs a) {
    hook_entry(a.notifier, a.job_id);
    __shared__ PageSpace<4> space;
    __shared__ unsigned entries[256 * kSelectKeys];
    __shared__ float errors[4];
    __shared__ unsigned arrived;
    const Screened w(a);
    if (w.n > 0) {  // (a tile is one token's)
        const bool alone = a.splits.d == 1;
        const size_t row = (size_t)(w.its.first + w.j0) * a.kv_heads.d + w.h;
        unsigned* const entries_of = a.entries + row * a.pitch;
        float* const errors_of = a.errors + row * 4 * a.splits.d;
        screen_pages<T, D>(
            a, w,
            [&](int, unsigned e, unsigned key) {
                if (alone) entries[e] = key;
                else __hip_atomic_store(entries_of + e, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            },
            [&](int, unsigned slot, float worst) {
                if (alone) errors[slot] = worst;
                else store_out(errors_of + slot, worst);
            });
        if (!alone) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (threadIdx.x == 0) {
                unsigned* const counter = a.counters + row * kCounterStride;
                arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (arrived == a.splits.d - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        __syncthreads();
        if (alone || arrived == a.splits.d - 1) {
            const unsigned pages = w.pages(a, 0);
            float error = 0.f;
            if (alone) {
                error = errors[threadIdx.x & 3];
            } else {
                unsigned held[kSelectKeys];
                auto read = [](auto* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
#pragma unroll
                for (int u = 0; u < kSelectKeys; ++u) held[u] = read(entries_of + min(threadIdx.x + u * 256, pages - 1));
                for (unsigned i = threadIdx.x; i < 4 * a.splits.d; i += 256) error = fmaxf(error, read(errors_of + i));
#pragma unroll
                for (int u = 0; u < kSelectKeys; ++u) entries[threadIdx.x + u * 256] = held[u];
                __syncthreads();
            }
            pick_pages<4, kSelectKeys>(a, w.its.first + w.j0, w.seq, w.h, pages, error, space, [&](unsigned i) { return entries[i]; });
        }
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
            auto load = [&](unsigned i) { return as_word(w[i]); };
            auto key = [](unsigned bits) { return number_key(as_float(bits), 1u); };
            span.hold(held, load, key);
            auto get = [&](int u, unsigned i) { return KEYS ? held[u] : key(load(i)); };
            Range<unsigned> range;
            span.visit(get, [&](int, unsigned, unsigned k) { range.add(k); });
            range.join(space);
            const Bound<unsigned> bound = find_bound<WAVES, KEYS, unsigned>(span, range, want, space, get);
            emit_taken<WAVES, KEYS, unsigned>(span, bound, space, get, [&](unsigned place, unsigned i) { put_int(to + first + place, (int)(first + i)); });
        }
    }
    hook_exit(a.notifier, a.job_id);
}

// Tokens move to lower places, in order: a workgroup takes some bytes of every key, or of every value, of a sequence's key head through, a run of tokens at a time, all of which it has read
// before it writes the first.  What later runs read lies behind everything that earlier ones wrote, and no two workgroups touch the same bytes, so nothing waits for another workgroup.

// 16 bytes that go through to memory.  (The wait states are those between a store and the next write of its registers.)
__device__ __forceinline__ void put16(char* p, u32x4 v) { asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" ::"v"(p), "v"(v) : "memory"); }

__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
    hook_entry(a.notifier, a.job_id);
    constexpr int AHEAD = 8;  // tokens of a lane in a run
    const Quotient by_slice = divide(blockIdx.x, a.slices), by_head = divide(by_slice.q, a.kv_heads);
    const unsigned slice = by_slice.r, h = by_head.r, seq = by_head.q, keep = (unsigned)a.keep;
    const int* const kept = a.kept + (size_t)by_slice.q * a.keep;
    const int* const table = a.tables + (size_t)seq * a.max_pages;
    const unsigned half = (a.slices.d - 1) / 2;  // slices of the keys, of the values, and one for the weights
    // What leads the list with its own places stays where it is: a place's distance from its token's does not shrink along the list, so 256 samples tell where to begin, but for a sample's distance.
    __shared__ unsigned alike[4];
    const unsigned apart = (keep + 255) / 256, sample = threadIdx.x * apart;
    const bool stays = sample < keep && (unsigned)kept[sample] == sample;
    const int last = kept[keep - 1];
    const unsigned long long who = __ballot(stays);
    if ((threadIdx.x & 63) == 0) alike[threadIdx.x >> 6] = (unsigned)__popcll(who);
    __syncthreads();
    const unsigned lead = alike[0] + alike[1] + alike[2] + alike[3], begin = lead ? (lead - 1) * apart : 0u;
    if (last >= 0) {  // else all of the sequence stays
        if (slice == a.slices.d - 1) {
            float* const w = a.weights + (size_t)by_slice.q * a.places;
            for (unsigned first = begin; first < keep; first += 1024) {
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
                    if (i < min(keep, a.places)) store_out(w + i, x[u]);
                }
            }
            if (h == 0 && threadIdx.x == 0) put_int(a.past_out + seq, a.keep);
        } else {
            char* const cache = slice < half ? a.k_cache : a.v_cache;
            const unsigned lanes_log2 = a.slice_log2 - 4, tokens = 256u >> lanes_log2;  // side by side
            const unsigned piece = ((slice < half ? slice : slice - half) << a.slice_log2) + (threadIdx.x & ((1u << lanes_log2) - 1)) * 16;
            const unsigned mine = threadIdx.x >> lanes_log2;
            const bool in = piece < (unsigned)a.row_bytes;
            const unsigned run = tokens * AHEAD;
            // A run's pages are looked up while the one ahead of it is read, and its tokens a run earlier still: then only keys and values, and the stores behind them, are waited for.
            int from[AHEAD], page[AHEAD], page_to[AHEAD];
            unsigned slot[AHEAD], slot_to[AHEAD];
            auto look = [&](unsigned first) {
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const unsigned i = first + u * tokens + mine;
                    from[u] = kept[min(i, keep - 1)];
                    if (!in || i >= keep || (unsigned)from[u] == i) from[u] = -1;
                }
            };
            auto resolve = [&](unsigned first) {
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {  // (a token that does not move: the first one's page, which is there)
                    const Quotient p = divide(from[u] < 0 ? 0u : (unsigned)from[u], a.pages), q = divide(from[u] < 0 ? 0u : first + u * tokens + mine, a.pages);
                    page[u] = table[min(p.q, (unsigned)a.max_pages - 1)];
                    page_to[u] = table[min(q.q, (unsigned)a.max_pages - 1)];
                    slot[u] = from[u] < 0 || p.q >= (unsigned)a.max_pages || q.q >= (unsigned)a.max_pages ? ~0u : p.r;
                    slot_to[u] = q.r;
                }
            };
            look(begin);
            resolve(begin);
            look(begin + run);
            for (unsigned first = begin; first < keep; first += run) {
                u32x4 x[AHEAD];
                char* to[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    to[u] = nullptr;
                    if (slot[u] != ~0u && (unsigned)page[u] < (unsigned)a.num_pages && (unsigned)page_to[u] < (unsigned)a.num_pages) {
                        to[u] = cache + (((size_t)page_to[u] * a.kv_heads.d + h) * a.page_size + slot_to[u]) * a.row_bytes + piece;
                        x[u] = *reinterpret_cast<const u32x4*>(cache + (((size_t)page[u] * a.kv_heads.d + h) * a.page_size + slot[u]) * a.row_bytes + piece);
                    }
                }
                resolve(first + run);
                look(first + 2 * run);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
#pragma unroll
                for (int u = 0; u < AHEAD; ++u)
                    if (to[u]) put16(to[u], x[u]);
            }
        }
    } else if (slice == a.slices.d - 1 && h == 0 && threadIdx.x == 0) {
        put_int(a.past_out + seq, (int)min(max((int64_t)a.past[seq], (int64_t)0), (int64_t)min(keep, a.places)));
    }
    hook_exit(a.notifier, a.job_id);
}

// ------------------------------------------------------------------------------------------ host

using BoundsKernel = void (*)(BoundsArgs);
template <int AHEAD, int HEADS>
BoundsKernel bounds_kernel_of(int dtype) {
    return dtype == PAELLA_F32 ? page_bounds_kernel<F32, AHEAD, HEADS> : dtype == PAELLA_BF16 ? page_bounds_kernel<Bf16, AHEAD, HEADS> : page_bounds_kernel<F16, AHEAD, HEADS>;
}
// 2^n lanes side by side have a key's 16-byte pieces.
int bounds_group_log2(const paella_kv_cache* c) {
    int n = 0;
    while ((16 << n) < c->head_dim * element_bytes(c->dtype) && n < 6) ++n;
    return n;
}
// Requests that a lane needs for a head's keys: four together where they fit that (with half the registers of eight twice as many waves are there), and where two or one do, two or four heads of a page by one
// wave (fp16 heads of 64: 32 MB in pages of 16 tokens of 4 heads by one / two heads a wave
// 15.0 / 12.9 us, 42 MB in pages of 8 of 8 heads by one / four 33 / 26).
int bounds_requests(const paella_kv_cache* c) { return (int)ceil_div(c->page_size, 64 >> bounds_group_log2(c)); }

struct BoundsGrid {
    int64_t touched, groups, items;
    unsigned grid() const { return (unsigned)((items + 3) / 4); }
};
BoundsGrid bounds_grid(const paella_kv_cache* c, const paella_kv_batch* b) {
    const int requests = bounds_requests(c);
    BoundsGrid g;
    g.touched = std::min<int64_t>(ceil_div(std::min(b->max_new, b->tokens) - 1, c->page_size) + 1, b->max_pages);
    g.groups = ceil_div(c->kv_heads, requests > 2 ? 1 : 4 / requests);
    g.items = (int64_t)b->sequences * g.touched * g.groups;
    return g;
}
BoundsKernel bounds_kernel(const paella_kv_cache* c) {
    const int requests = bounds_requests(c);
    return requests == 1 ? bounds_kernel_of<1, 4>(c->dtype) : requests == 2 ? bounds_kernel_of<2, 2>(c->dtype) : requests <= 4 ? bounds_kernel_of<4, 1>(c->dtype) : bounds_kernel_of<8, 1>(c->dtype);
}

int bounds_check(const paella_kv_cache* c, const paella_kv_batch* b) {
    if (!cache_extents_ok(c) || !batch_extents_ok(b)) return PAELLA_EINVAL;
    if ((double)b->max_pages * c->page_size >= 1073741824.0) return PAELLA_ENOSUP;
    return (double)b->sequences * bounds_grid(c, b).touched * c->kv_heads / 4 <= kMostWorkgroups - 1 ? 0 : PAELLA_ENOSUP;
}

using SelectKernel = void (*)(SelectArgs);
template <typename T>
SelectKernel screen_kernel_of(int dim, bool whole) {
    if (whole) return dim == 64 ? page_select_kernel<T, 64> : dim == 128 ? page_select_kernel<T, 128> : page_select_kernel<T, 256>;
    return dim == 64 ? page_screen_kernel<T, 64> : dim == 128 ? page_screen_kernel<T, 128> : page_screen_kernel<T, 256>;
}
// whole: the kernel that does both stages in one launch
SelectKernel screen_kernel(const paella_page_select_plan* p, bool whole) {
    return p->dtype == PAELLA_F32    ? screen_kernel_of<F32>(p->head_dim, whole)
           : p->dtype == PAELLA_BF16 ? screen_kernel_of<Bf16>(p->head_dim, whole)
                                     : screen_kernel_of<F16>(p->head_dim, whole);
}

// A kernel of one of these forms, by how many there are to pick from at most: with their keys in registers, or, beyond what the registers of 16 waves hold, read again for every pass.
// (Pages of 96 rows: 1001 by 4 / 16 waves 9.2 / 9.4 us, 4001 by 4 / 16 14.3 / 11.1; 1001 of 1536 rows 18.4 / 41.2; 15626 of 32 rows from registers / read again 19.4 / 42. Tokens of 8 to 192 heads: 4000 by
// 4 / 16 waves 11.1 / 8.2, 4000 from registers / read again 8.3 / 10.9, 16384 15.4 / 20.7, 49285 in 64 registers a thread, more than there are, / read again 90 / 46.)
template <typename Kernel>
struct PickForm {
    Kernel kernel;
    unsigned threads;
};
PickForm<SelectKernel> page_pick(int64_t n) {
    if (n <= 1024) return {page_pick_kernel<4, 4>, 256};
    if (n <= 2048) return {page_pick_kernel<4, 8>, 256};
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

int64_t select_tiles(const paella_page_select_plan* p) { return ceil_div(std::min(p->max_new, p->tokens), tokens_of_tile(p->heads / p->kv_heads)); }
int64_t screen_grid(const paella_page_select_plan* p) { return p->sequences * select_tiles(p) * p->kv_heads * p->splits; }
int64_t select_pages(const paella_page_select_plan* p) { return ceil_div(p->prefix_len, p->page_size) + p->max_pages; }

bool select_plan_ok(const paella_page_select_plan* p) {
    if (!p || !planned_extents_ok(p) || p->count <= 0 || p->first < 0 || p->last < 1 || (int64_t)p->first + p->last > p->count || p->splits <= 0) return false;
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return false;
    const double rows = (double)p->tokens * p->kv_heads;
    return rows <= kMostWorkgroups / 4 && (double)p->sequences * select_tiles(p) * p->kv_heads * p->splits <= kMostWorkgroups && rows * p->count < 2147483648.0 && select_pages(p) < (1 << 30);
}

size_t select_pitch(const paella_page_select_plan* p) { return (size_t)(select_pages(p) + 15) / 16 * 16; }
// One launch where four waves hold a row's pages in registers, a tile is one token's (a workgroup that picked for several would take as much longer), and the workgroups are at most two to a
// compute unit; of more, those that pick are in the way of those that still screen.  (3 fp32 rows of 57 pages of 2 heads of 64 in one launch / two 9.4 / 10.5 us, 32 bf16 rows of 1025 pages of 8 heads
// of 128, 512 workgroups, 30.9 / 33.6; by 1024 45.2 / 41.3.)
int select_stages(const paella_page_select_plan* p) {
    const bool one = std::min(p->max_new, p->tokens) == 1 || tokens_of_tile(p->heads / p->kv_heads) == 1;
    return one && screen_grid(p) <= 512 && select_pages(p) <= 256 * kSelectKeys ? 1 : 2;
}
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
size_t select_counters(const paella_page_select_plan* p) { return select_stages(p) == 1 ? (size_t)p->tokens * p->kv_heads * kCounterStride * 4 : 0; }
size_t select_errors(const paella_page_select_plan* p) { return up256((size_t)p->tokens * p->kv_heads * p->splits * 16); }
size_t select_entries(const paella_page_select_plan* p) { return up256((size_t)p->tokens * p->kv_heads * select_pitch(p) * 4); }
size_t select_workspace(const paella_page_select_plan* p) { return select_counters(p) + select_errors(p) + 3 * select_entries(p); }  // (worths of 64 bits: twice the entries)

// Bytes of a row that a workgroup moves: 128, which memory likes best, where that still makes a workgroup for each compute unit, else 64, or 32 where even those leave half of the device idle, or 16 where
// three quarters.  (bf16 heads of 128, 4096 tokens kept of 8 heads: 24 sequences by 128 / 64 bytes 193 / 247 us, 8 91 / 94, 4 57 / 48; one by 64 / 32 / 16 40 / 26 / 44; 20000 tokens of 2 heads by 32 / 16
// 111 / 85.)
int evict_slice_log2(int sequences, const paella_kv_cache* c) {
    const int64_t heads = (int64_t)sequences * c->kv_heads, row = (int64_t)c->head_dim * element_bytes(c->dtype);
    return 2 * heads * ceil_div(row, 128) >= 256 ? 7 : 2 * heads * ceil_div(row, 64) >= 128 ? 6 : 2 * heads * ceil_div(row, 32) >= 64 ? 5 : 4;
}
int64_t evict_slices(int sequences, const paella_kv_cache* c) {
    return 2 * ceil_div((int64_t)c->head_dim * element_bytes(c->dtype), 1 << evict_slice_log2(sequences, c)) + 1;
}
int evict_check(const paella_kv_evict_desc* d, const paella_kv_cache* c) {
    if (!d || !cache_extents_ok(c) || d->sequences <= 0 || d->max_pages <= 0 || d->keep <= 0 || d->first < 0 || d->recent < 0 || (int64_t)d->first + d->recent > d->keep) return PAELLA_EINVAL;
    const double heads = (double)d->sequences * c->kv_heads;
    if ((double)d->max_pages * c->page_size >= 1073741824.0 || (double)d->sequences * d->max_pages >= 2147483648.0) return PAELLA_ENOSUP;
    const double picking = heads * evict_pick((int64_t)d->max_pages * c->page_size).threads / 256, moving = heads * evict_slices(d->sequences, c);
    return picking <= kMostWorkgroups && moving <= kMostWorkgroups ? 0 : PAELLA_ENOSUP;
}

// ------------------------------------------------------------------------------------------ the weights of stored scores (long_attention.h)
// Four tokens a thread.
__global__ __launch_bounds__(256) void stored_weights_kernel(WeighArgs a) {
    hook_entry(a.notifier, a.job_id);
    __shared__ f32x2 whole[16];
    const Quotient by_head = divide(blockIdx.x, a.kv_heads), by_split = divide(by_head.q, a.own_splits);
    const int h = (int)by_head.r, split = (int)by_split.r, seq = (int)by_split.q;
    const NewTokens its = new_tokens(a.starts, a.past, seq, a.max_new, a.tokens);
    const int rows = its.count * (int)a.per_kv.d, places = a.max_pages * a.page_size, past = min(its.past, places), held = min(past + its.count, places);
    const int per = (int)divide((unsigned)held + a.own_splits.d - 1, a.own_splits).q, begin = min(split * ((per + 3) / 4 * 4), held), end = min(begin + (per + 3) / 4 * 4, held);
    if (rows > 0 && begin < end) {
        join_rows<16>(a, its.first, h, 0, rows, whole);
        __syncthreads();
        const size_t head = (size_t)seq * a.kv_heads.d + h;
        const float* const scores = a.scores + head * a.score_rows * (size_t)places;
        float* const weights = a.weights + head * (size_t)places;
        const __amdgpu_buffer_rsrc_t to = descriptor(weights);
        for (int i = begin + (int)threadIdx.x * 4; i < end; i += 1024) {  // (places are a multiple of eight: four of them are there)
            const f32x4 old = *reinterpret_cast<const f32x4*>(weights + i);
            f32x4 w = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int r = 0; r < rows; ++r) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(scores + (size_t)r * places + i);
                const f32x2 row = whole[r];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] += row.y * __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], a.scale_log2, -row.x));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = i + e >= held ? old[e] : i + e >= past ? w[e] : old[e] + w[e];
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, w), to, (int)((unsigned)i * 4), 0, kThrough);
        }
    }
    hook_exit(a.notifier, a.job_id);
}

}  // namespace

namespace paella {
WeighKernel stored_weights() { return stored_weights_kernel; }
}  // namespace paella

extern "C" {

int paella_page_bounds_dims(const paella_kv_cache* c, const paella_kv_batch* b, paella_launch_dims* dims) {
    if (int rc = bounds_check(c, b)) return rc;
    if (!dims) return PAELLA_EINVAL;
    const BoundsGrid g = bounds_grid(c, b);
    set_launch_dims(dims, g.grid(), 256, 0, 64);
    loaded_dims((const void*)bounds_kernel(c), dims);
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
    a.row_bytes = c->head_dim * element_bytes(c->dtype); a.pieces = a.row_bytes / 16; a.group_log2 = bounds_group_log2(c);
    a.kv_heads = c->kv_heads; a.groups = divisor((unsigned)g.groups); a.touched = divisor((unsigned)g.touched); a.items = (unsigned)g.items;
    a.job_id = job_id; a.notifier = (Notifier*)notifier;
    launch(bounds_kernel(c), dim3(g.grid()), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

int paella_page_select_plan_make(const paella_kv_cache* c, const paella_kv_batch* b, int heads, int count, int first, int last, paella_page_select_plan* p) {
    if (!p || !cache_extents_ok(c) || !batch_extents_ok(b) || heads <= 0 || heads % c->kv_heads || count <= 0 || first < 0 || last < 1 || (int64_t)first + last > count) return PAELLA_EINVAL;
    *p = paella_page_select_plan{};
    plan_extents(p, c, b, heads);
    p->count = count; p->first = first; p->last = last;
    const int64_t pages = select_pages(p), rows = (int64_t)p->tokens * p->kv_heads;
    // as many workgroups as the device holds at once, two to a compute unit, or none without a turn for each wave (32 rows of 1025 pages of 8 heads of 128 in bf16 by 512 / 1024 / 2048 workgroups 21.9 /
    // 22.8 / 26.1 us, 4 of 15626 of 8 heads of 64 13.2 / 12.0 / 12.7)
    p->splits = 1;
    if (!select_plan_ok(p)) return PAELLA_ENOSUP;
    p->splits = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(512, screen_grid(p)), ceil_div(pages, 4 * kScreened)));
    if (!select_plan_ok(p)) return PAELLA_ENOSUP;
    p->stages = select_stages(p);
    p->workspace_bytes = select_workspace(p);
    p->zero_bytes = select_counters(p);
    set_launch_dims(&p->dims, (unsigned)screen_grid(p), 256, 0, 128);
    const double size = element_bytes(c->dtype);
    p->flops = 4.0 * p->tokens * p->heads * pages * p->head_dim;
    p->bytes = 2.0 * (pages - p->max_pages + (double)p->sequences * p->max_pages) * p->kv_heads * p->head_dim * size + (double)p->tokens * p->heads * p->head_dim * size + 4.0 * rows * count;
    return 0;
}

int paella_page_select_dims(const paella_page_select_plan* p, int stage, paella_launch_dims* dims) {
    if (!select_plan_ok(p) || !dims || stage < 0 || stage >= select_stages(p)) return PAELLA_EINVAL;
    const auto pick = page_pick(select_pages(p));
    if (stage) set_launch_dims(dims, (unsigned)(p->tokens * p->kv_heads), pick.threads, 0, 64);
    else set_launch_dims(dims, (unsigned)screen_grid(p), 256, 0, 128);
    loaded_dims(stage ? (const void*)pick.kernel : (const void*)screen_kernel(p, select_stages(p) == 1), dims);
    return 0;
}

int paella_page_select_launch_stage(const paella_page_select_plan* p, int stage, const paella_kv_cache* c, const paella_kv_batch* b, const void* q, int64_t q_stride,
                                    const void* bounds, int32_t* pages, void* workspace, void* stream, uint32_t job_id, void* notifier) {
    if (!select_plan_ok(p) || stage < 0 || stage >= select_stages(p) || !planned_for(p, c, b) || !q || !bounds || !pages || !workspace) return PAELLA_EINVAL;
    const int64_t size = element_bytes(c->dtype), row = (int64_t)p->heads * p->head_dim;
    if (q_stride < row || q_stride % 8 || (((uintptr_t)q | (uintptr_t)bounds | (uintptr_t)workspace) & 15) || ((uintptr_t)pages & 3)) return PAELLA_EINVAL;
    const double out_bytes = 4.0 * p->tokens * p->kv_heads * p->count, space = (double)select_workspace(p);
    const double bound_bytes = 2.0 * c->num_pages * c->kv_heads * c->head_dim * size;
    const struct { const void* at; double bytes; } outs[2] = {{pages, out_bytes}, {workspace, space}};
    for (const auto& o : outs)
        if (rows_overlap(q, p->tokens, q_stride * size, row * size, o.at, o.bytes) || overlap(bounds, bound_bytes, o.at, o.bytes) || over_cache(c, o.at, o.bytes) ||
            over_batch(b, c->page_size, o.at, o.bytes))
            return PAELLA_EINVAL;
    if (overlap(pages, out_bytes, workspace, space)) return PAELLA_EINVAL;
    SelectArgs a;
    a.q = (const char*)q; a.bounds = (const char*)bounds;
    a.starts = b->starts; a.past = b->past; a.tables = b->tables; a.prefix_table = b->prefix_table;
    a.counters = (unsigned*)workspace; a.errors = (float*)((char*)workspace + select_counters(p)); a.entries = (unsigned*)((char*)a.errors + select_errors(p)); a.worths = (unsigned long long*)((char*)a.entries + select_entries(p)); a.pages = pages; a.q_stride = q_stride * size;
    a.sequences = b->sequences; a.tokens = b->tokens; a.max_pages = b->max_pages; a.prefix_pages = (int)ceil_div(b->prefix_len, c->page_size); a.num_pages = c->num_pages;
    a.heads = p->heads; a.first = p->first; a.last = p->last; a.count = p->count; a.dim = p->head_dim; a.dtype = p->dtype; a.pitch = (unsigned)select_pitch(p);
    a.max_new = divisor((unsigned)b->max_new); a.kv_heads = divisor((unsigned)p->kv_heads); a.per_kv = divisor((unsigned)(p->heads / p->kv_heads)); a.splits = divisor((unsigned)p->splits);
    a.tiles = divisor((unsigned)select_tiles(p)); a.page_size = divisor((unsigned)c->page_size);
    a.job_id = job_id; a.notifier = (Notifier*)notifier;
    const unsigned rows = (unsigned)(p->tokens * p->kv_heads);
    if (stage == 0) {
        launch(screen_kernel(p, select_stages(p) == 1), dim3((unsigned)screen_grid(p)), dim3(256), 0, (hipStream_t)stream, a);
    } else {
        const auto pick = page_pick(select_pages(p));
        launch(pick.kernel, dim3(rows), dim3(pick.threads), 0, (hipStream_t)stream, a);
    }
    return (int)hipGetLastError();
}

int paella_page_select_launch(const paella_page_select_plan* p, const paella_kv_cache* c, const paella_kv_batch* b, const void* q, int64_t q_stride, const void* bounds,
                              int32_t* pages, void* workspace, void* stream, uint32_t job_id, void* notifier) {
    if (!select_plan_ok(p)) return PAELLA_EINVAL;
    const int stages = select_stages(p);
    if (stages > 1) {
        if (keeps_no_order(stream)) return PAELLA_ENOSUP;
        if (int rc = paella_page_select_launch_stage(p, 0, c, b, q, q_stride, bounds, pages, workspace, stream, job_id, nullptr)) return rc;
    }
    return paella_page_select_launch_stage(p, stages - 1, c, b, q, q_stride, bounds, pages, workspace, stream, job_id, notifier);
}

int paella_kv_evict_dims(const paella_kv_evict_desc* d, const paella_kv_cache* c, int stage, paella_launch_dims* dims) {
    if (int rc = evict_check(d, c)) return rc;
    if (!dims || stage < 0 || stage > 1) return PAELLA_EINVAL;
    if (stage) set_launch_dims(dims, (unsigned)(d->sequences * c->kv_heads * evict_slices(d->sequences, c)), 256, 0, 64);
    const auto pick = evict_pick((int64_t)d->max_pages * c->page_size);
    if (!stage) set_launch_dims(dims, (unsigned)(d->sequences * c->kv_heads), pick.threads, 0, 64);
    loaded_dims(stage ? (const void*)evict_move_kernel : (const void*)pick.kernel, dims);
    return 0;
}

int paella_kv_evict_launch_stage(const paella_kv_evict_desc* d, int stage, const paella_kv_cache* c, float* weights, const int32_t* past, const int32_t* tables, int32_t* kept,
                                 int32_t* past_out, void* stream, uint32_t job_id, void* notifier) {
    if (int rc = evict_check(d, c)) return rc;
    if (stage < 0 || stage > 1 || !cache_ok(c) || !weights || !past || !tables || !kept || !past_out) return PAELLA_EINVAL;
    if (((uintptr_t)weights | (uintptr_t)past | (uintptr_t)tables | (uintptr_t)kept | (uintptr_t)past_out) & 3) return PAELLA_EINVAL;
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
    a.kv_heads = divisor((unsigned)c->kv_heads); a.slices = divisor((unsigned)evict_slices(d->sequences, c)); a.pages = divisor((unsigned)c->page_size);
    a.job_id = job_id; a.notifier = (Notifier*)notifier;
    a.slice_log2 = (unsigned)evict_slice_log2(d->sequences, c);
    const auto pick = evict_pick((int64_t)a.places);
    if (stage == 0) launch(pick.kernel, dim3((unsigned)(d->sequences * c->kv_heads)), dim3(pick.threads), 0, (hipStream_t)stream, a);
    else launch(evict_move_kernel, dim3((unsigned)(d->sequences * c->kv_heads * evict_slices(d->sequences, c))), dim3(256), 0, (hipStream_t)stream, a);
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
