// Operators that keep a long paged cache from being read and kept whole: bounds of the pages' keys, the selection of pages by them, and eviction.
// (Attention over the pages and the weights that tokens gather: long_attention.h.)

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "long_common.h"

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
// worth(e) = max over the key head's query heads of sum_d max(q_d low_d, q_d high_d) = (q . (low + high) + |q| . (high - low)) / 2.  Which of two neighbours is taken is decided
// by their last digits, so everything is in 64 bits, where the products are exact; a 64-bit fma takes the vector unit no longer than two 32-bit ones, and the bounds are
// what takes the time.  A first launch leaves the worths as numbers whose order is theirs, a second one takes the largest.
struct ScoreArgs {
    const char *q, *bounds;
    const int *starts, *past, *tables, *prefix_table;
    unsigned long long* keys;  // [tokens][kv_heads][pitch]
    int64_t q_stride;          // bytes
    int sequences, tokens, max_pages, prefix_pages, num_pages, heads, first, last;
    unsigned pitch;
    Divisor max_new, kv_heads, splits, page_size;
    uint32_t job_id;
    Notifier* notifier;
};

constexpr unsigned long long kTaken = ~0ull;  // whatever it is worth

__device__ __forceinline__ unsigned long long worth_key(double v) {
    if (v != v) v = INFINITY;
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v + 0.0);
    const unsigned long long k = b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
    return k;  // (above 0, which is no page, and below kTaken)
}

template <typename T>
__device__ __forceinline__ void to_double(u32x4 w, double (&x)[16 / T::bytes]) {
    if constexpr (T::bytes == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (double)as_float(w[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const f32x2 v = unpack2<T>(w[e]);
            x[2 * e] = (double)v.x;
            x[2 * e + 1] = (double)v.y;
        }
    }
}

__device__ __forceinline__ double shuffle_xor(double v, int mask) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = (unsigned)__shfl_xor((int)(unsigned)b, mask, 64), hi = (unsigned)__shfl_xor((int)(unsigned)(b >> 32), mask, 64);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

template <int LANES>
__device__ __forceinline__ double lanes_sum64(double v) {
    v += lane_move<0xB1>(v);
    v += lane_move<0x4E>(v);
    v += lane_move<0x141>(v);
    if constexpr (LANES > 8) v += lane_move<0x140>(v);
    if constexpr (LANES > 16) v += shuffle_xor(v, 16);
    if constexpr (LANES > 32) v += shuffle_xor(v, 32);
    return v;
}

constexpr int kScoreAhead = 4;  // pages of a lane that are requested together

template <typename T, int D>
constexpr int score_batch() { return 64 / (D * T::bytes / 16) * kScoreAhead; }  // pages of a wave's turn

// GC: query heads at a time.
template <typename T, int D, int GC>
__global__ __launch_bounds__(256) void page_score_kernel(ScoreArgs a) {
    hook_entry(a.notifier, a.job_id);
    constexpr int V = 16 / T::bytes, LANES = D / V, EACH = 64 / LANES, U = kScoreAhead, BATCH = score_batch<T, D>(), ROW = D * T::bytes;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const Quotient by_head = divide(blockIdx.x, a.kv_heads), by_split = divide(by_head.q, a.splits);
    const int t = (int)by_split.q, h = (int)by_head.r;
    int seq, j;
    if (row_owner(a.starts, a.sequences, a.max_new, t, lane, &seq, &j)) {
        const int own = own_pages(__builtin_amdgcn_readfirstlane(a.past[seq]), j, a.page_size, a.max_pages);
        const unsigned pages = (unsigned)a.prefix_pages + (unsigned)own;
        const unsigned batches = (pages + BATCH - 1) / BATCH;
        unsigned long long* const keys = a.keys + ((size_t)t * a.kv_heads.d + h) * a.pitch;
        const int* const table = a.tables + (size_t)seq * a.max_pages;
        const int piece = lane % LANES, group = a.heads / (int)a.kv_heads.d;
        const char* const q_head = a.q + t * a.q_stride + (size_t)h * group * ROW + piece * 16;
        double q[GC][V];
        auto load_q = [&](int first) {
#pragma unroll
            for (int g = 0; g < GC; ++g) to_double<T>(*reinterpret_cast<const u32x4*>(q_head + min(first + g, group - 1) * ROW), q[g]);
        };
        load_q(0);
        for (unsigned b = by_split.r * 4 + wave; b < batches; b += a.splits.d * 4) {
            unsigned e[U];
            int page[U];
            u32x4 low[U], high[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                e[u] = b * BATCH + u * EACH + lane / LANES;
                const unsigned at = min(e[u], pages - 1);
                page[u] = at < (unsigned)a.prefix_pages ? a.prefix_table[at] : table[at - a.prefix_pages];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const char* const from = a.bounds + ((size_t)((unsigned)page[u] < (unsigned)a.num_pages ? page[u] : 0) * a.kv_heads.d + h) * 2 * ROW + piece * 16;
                low[u] = *reinterpret_cast<const u32x4*>(from);
                high[u] = *reinterpret_cast<const u32x4*>(from + ROW);
            }
            unsigned long long best[U];
#pragma unroll
            for (int u = 0; u < U; ++u) best[u] = 0;
            for (int g0 = 0; g0 < group; g0 += GC) {
                if (group > GC) load_q(g0);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    double lo[V], hi[V], sum[GC];
                    to_double<T>(low[u], lo);
                    to_double<T>(high[u], hi);
#pragma unroll
                    for (int g = 0; g < GC; ++g) sum[g] = 0.0;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const double both = lo[v] + hi[v], wide = hi[v] - lo[v];
#pragma unroll
                        for (int g = 0; g < GC; ++g) sum[g] = __builtin_fma(__builtin_fabs(q[g][v]), wide, __builtin_fma(q[g][v], both, sum[g]));
                    }
#pragma unroll
                    for (int g = 0; g < GC; ++g) best[u] = max(best[u], worth_key(lanes_sum64<LANES>(sum[g])));
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (piece == 0 && e[u] < pages) {
                    if (e[u] < (unsigned)a.first || e[u] + a.last >= pages) best[u] = kTaken;
                    if ((unsigned)page[u] >= (unsigned)a.num_pages) best[u] = 0;
                    __hip_atomic_store(keys + e[u], best[u], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
        }
    }
    hook_exit(a.notifier, a.job_id);
}

// ------------------------------------------------------------------------------------------ the largest of many
// The `want` largest of n keys (0 is none; of equals the lower index), in the order of their indices.  Digit by digit from the highest one in which the keys
// differ: a histogram of the keys that agree with the bound so far says which digit the last one taken has, until the keys of that digit are just as many as are wanted.  Waves
// have keys that lie side by side, so that they come out in order.  Called by all threads of a workgroup of WAVES waves; get(i): key i, called several times; take(place, i)
// for each taken.  Returns how many.
template <int WAVES>
struct PickSpace {
    unsigned bins[256];
    unsigned long long low[WAVES], high[WAVES];
    unsigned above[WAVES], equal[WAVES];
    unsigned digit, taken, left, done;
};

template <int WAVES, typename Key, typename Get, typename Take>
__device__ __forceinline__ unsigned pick_largest(unsigned n, unsigned want, PickSpace<WAVES>& s, Get get, Take take) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const unsigned per = (n + WAVES * 64 - 1) / (WAVES * 64) * 64;
    const unsigned begin = min((unsigned)wave * per, n), end = min(begin + per, n);
    // the least and largest key, and how many there are
    Key least = ~(Key)0, most = 0;
    unsigned some = 0;
    for (unsigned i = begin + lane; i < end; i += 64) {
        const Key k = get(i);
        if (k) {
            least = min(least, k);
            ++some;
        }
        most = max(most, k);
    }
    for (int off = 32; off; off >>= 1) {
        least = min(least, (Key)__shfl_xor((unsigned long long)least, off, 64));
        most = max(most, (Key)__shfl_xor((unsigned long long)most, off, 64));
        some += __shfl_xor(some, off, 64);
    }
    if (lane == 0) {
        s.low[wave] = least;
        s.high[wave] = most;
        s.equal[wave] = some;
    }
    __syncthreads();
    some = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        least = min(least, (Key)s.low[w]);
        most = max(most, (Key)s.high[w]);
        some += s.equal[w];
    }
    // keys >= bound are taken, but of those equal to it (where `left` says so) the first `left` alone
    Key bound = 1;
    unsigned left = ~0u;
    if (some > want) {
        const int differ = least == most ? 0 : 64 - __clzll((unsigned long long)(least ^ most));  // bits; those above are the same in all keys
        int shift = max(differ - 8, 0);
        Key known = shift + 8 < (int)sizeof(Key) * 8 ? (Key)(~(Key)0 << (shift + 8)) : (Key)0;  // the bits that the bound has so far
        bound = differ ? most & known : most;
        left = want;
        while (differ) {
            __syncthreads();
            for (int b = threadIdx.x; b < 256; b += WAVES * 64) s.bins[b] = 0;
            __syncthreads();
            for (unsigned i = begin + lane; i < end; i += 64) {
                const Key k = get(i);
                if (k && (k & known) == (bound & known)) atomicAdd(&s.bins[(unsigned)(k >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (threadIdx.x < 64) {  // four digits a lane, the highest first
                unsigned c[4], sum = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    c[e] = s.bins[255 - (lane * 4 + e)];
                    sum += c[e];
                }
                unsigned upto = sum;
                for (int off = 1; off < 64; off <<= 1) {
                    const unsigned other = __shfl_up(upto, off, 64);
                    if (lane >= off) upto += other;
                }
                unsigned before = upto - sum;
                if (before < left && left <= upto) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (before < left && left <= before + c[e]) {
                            s.digit = 255 - (lane * 4 + e);
                            s.left = left - before;
                            s.done = c[e] == left - before;
                        }
                        before += c[e];
                    }
                }
            }
            __syncthreads();
            bound |= (Key)s.digit << shift;
            left = s.left;
            known |= (Key)255 << shift;
            if (s.done) {  // all that begin so are taken
                left = ~0u;
                break;
            }
            if (shift == 0) break;
            shift = max(shift - 8, 0);
        }
    }
    // in the order of their places: how many each wave has above the bound and at it, then where they go
    unsigned above = 0, equal = 0;
    for (unsigned i = begin + lane; i < (end + 63) / 64 * 64; i += 64) {
        const Key k = i < end ? get(i) : 0;
        above += __popcll(__ballot(left == ~0u ? k >= bound : k > bound));
        equal += __popcll(__ballot(left != ~0u && k == bound));
    }
    __syncthreads();
    if (lane == 0) {
        s.above[wave] = above;
        s.equal[wave] = equal;
    }
    __syncthreads();
    unsigned place = 0, ties = 0, all = 0, ties_all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const unsigned here = left == ~0u ? 0u : min(s.equal[w], left - min(left, ties_all));
        if (w < wave) {
            place += s.above[w] + here;
            ties += s.equal[w];
        }
        all += s.above[w] + here;
        ties_all += s.equal[w];
    }
    for (unsigned i = begin + lane; i < (end + 63) / 64 * 64; i += 64) {
        const Key k = i < end ? get(i) : 0;
        const unsigned long long tied = __ballot(left != ~0u && k == bound), before = (1ull << lane) - 1;
        const bool mine = left == ~0u ? k >= bound : k > bound || (k == bound && ties + __popcll(tied & before) < left);
        const unsigned long long who = __ballot(mine);
        if (mine) take(place + __popcll(who & before), i);
        place += __popcll(who);
        ties += __popcll(tied);
    }
    return all;
}

struct PickArgs {
    const unsigned long long* keys;
    int* pages;
    const int *starts, *past;
    int sequences, max_pages, prefix_pages, count;
    unsigned pitch;
    Divisor max_new, kv_heads, page_size;
    uint32_t job_id;
    Notifier* notifier;
};

__device__ __forceinline__ void put_int(int* p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

constexpr int kPickWaves = 4;

__global__ __launch_bounds__(kPickWaves * 64) void page_pick_kernel(PickArgs a) {
    hook_entry(a.notifier, a.job_id);
    __shared__ PickSpace<kPickWaves> space;
    const int lane = threadIdx.x & 63;
    const Quotient by_head = divide(blockIdx.x, a.kv_heads);
    int seq, j;
    if (row_owner(a.starts, a.sequences, a.max_new, (int)by_head.q, lane, &seq, &j)) {
        const unsigned pages = (unsigned)a.prefix_pages + (unsigned)own_pages(__builtin_amdgcn_readfirstlane(a.past[seq]), j, a.page_size, a.max_pages);
        const unsigned long long* const keys = a.keys + (size_t)blockIdx.x * a.pitch;
        int* const to = a.pages + (size_t)blockIdx.x * a.count;
        const unsigned taken = pick_largest<kPickWaves, unsigned long long>(
            pages, (unsigned)a.count, space, [&](unsigned i) { return keys[i]; }, [&](unsigned place, unsigned i) { put_int(to + place, (int)i); });
        for (unsigned i = taken + threadIdx.x; i < (unsigned)a.count; i += kPickWaves * 64) put_int(to + i, -1);
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
    Divisor kv_heads, slices, pages;  // pages: divides by the page size
    uint32_t job_id;
    Notifier* notifier;
};

// A weight as a number whose order is the weights', above 0; NaN as the least.
__device__ __forceinline__ unsigned weight_key(float w) {
    if (w != w) return 1u;
    const unsigned b = as_word(w + 0.f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

__global__ __launch_bounds__(kPickWaves * 64) void evict_pick_kernel(EvictArgs a) {
    hook_entry(a.notifier, a.job_id);
    __shared__ PickSpace<kPickWaves> space;
    const Quotient by_head = divide(blockIdx.x, a.kv_heads);
    const unsigned n = (unsigned)min(max((int64_t)__builtin_amdgcn_readfirstlane(a.past[by_head.q]), (int64_t)0), (int64_t)a.places);
    int* const to = a.kept + (size_t)blockIdx.x * a.keep;
    unsigned taken = n;
    if (n <= (unsigned)a.keep) {
        for (unsigned i = threadIdx.x; i < n; i += kPickWaves * 64) put_int(to + i, (int)i);
    } else {
        const float* const w = a.weights + (size_t)blockIdx.x * a.places;
        const unsigned first = (unsigned)a.first, behind = n - (unsigned)a.recent;
        taken = pick_largest<kPickWaves, unsigned>(
            n, (unsigned)a.keep, space, [&](unsigned i) { return i < first || i >= behind ? ~0u : weight_key(w[i]); },
            [&](unsigned place, unsigned i) { put_int(to + place, (int)i); });
    }
    for (unsigned i = taken + threadIdx.x; i < (unsigned)a.keep; i += kPickWaves * 64) put_int(to + i, -1);
    hook_exit(a.notifier, a.job_id);
}

// Tokens move to lower places, in order: a workgroup takes 64 bytes of every key, or of every value, of a sequence's key head through, a run of tokens at a time, all of which it has read
// before it writes the first.  What later runs read lies behind everything that earlier ones wrote, and no two workgroups touch the same bytes, so nothing waits for another workgroup.
constexpr int kSlice = 64;      // bytes of a row
constexpr int kMoveAhead = 4;   // tokens of a lane in a run
constexpr int kMoveRun = 256 / (kSlice / 16) * kMoveAhead;

__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
    hook_entry(a.notifier, a.job_id);
    const Quotient by_slice = divide(blockIdx.x, a.slices), by_head = divide(by_slice.q, a.kv_heads);
    const unsigned slice = by_slice.r, h = by_head.r, seq = by_head.q;
    const int* const kept = a.kept + (size_t)by_slice.q * a.keep;
    const int* const table = a.tables + (size_t)seq * a.max_pages;
    const unsigned half = (a.slices.d - 1) / 2;  // slices of the keys, of the values, and one for the weights
    if (kept[a.keep - 1] >= 0) {                 // else all of the sequence stays
        if (slice == a.slices.d - 1) {
            float* const w = a.weights + (size_t)by_slice.q * a.places;
            for (int first = 0; first < a.keep; first += 1024) {
                float x[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int i = first + u * 256 + (int)threadIdx.x;
                    const unsigned from = i < a.keep ? (unsigned)kept[i] : 0u;
                    x[u] = from < a.places ? w[from] : 0.f;
                }
                __syncthreads();
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int i = first + u * 256 + (int)threadIdx.x;
                    if (i < a.keep) store_out(w + i, x[u]);
                }
            }
            if (h == 0 && threadIdx.x == 0) put_int(a.past_out + seq, a.keep);
        } else {
            char* const cache = slice < half ? a.k_cache : a.v_cache;
            const unsigned piece = (slice < half ? slice : slice - half) * kSlice + (threadIdx.x & (kSlice / 16 - 1)) * 16;
            const bool in = piece < (unsigned)a.row_bytes;
            const unsigned mine = threadIdx.x / (kSlice / 16);
            auto at = [&](unsigned token, bool* there) {
                const Quotient p = divide(token, a.pages);
                const int page = p.q < (unsigned)a.max_pages ? table[p.q] : -1;
                *there = (unsigned)page < (unsigned)a.num_pages;
                return (((size_t)(*there ? page : 0) * a.kv_heads.d + h) * a.page_size + p.r) * a.row_bytes + piece;
            };
            for (unsigned first = 0; first < (unsigned)a.keep; first += kMoveRun) {
                u32x4 x[kMoveAhead];
                size_t to[kMoveAhead];
                bool go[kMoveAhead];
#pragma unroll
                for (int u = 0; u < kMoveAhead; ++u) {
                    const unsigned i = first + u * (256 / (kSlice / 16)) + mine;
                    const int from = i < (unsigned)a.keep ? kept[i] : -1;
                    bool there = false, here = false;
                    size_t whence = 0;
                    to[u] = 0;
                    if (in && from >= 0 && (unsigned)from != i) {
                        whence = at((unsigned)from, &there);
                        to[u] = at(i, &here);
                    }
                    go[u] = there && here;
                    if (go[u]) x[u] = *reinterpret_cast<const u32x4*>(cache + whence);
                }
                __syncthreads();
#pragma unroll
                for (int u = 0; u < kMoveAhead; ++u)
                    if (go[u]) {
                        unsigned* const p = reinterpret_cast<unsigned*>(cache + to[u]);
                        __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), (unsigned long long)x[u].y << 32 | x[u].x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                        __hip_atomic_store(reinterpret_cast<unsigned long long*>(p + 2), (unsigned long long)x[u].w << 32 | x[u].z, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    }
            }
        }
    } else if (slice == a.slices.d - 1 && h == 0 && threadIdx.x == 0) {
        put_int(a.past_out + seq, (int)min(max((int64_t)a.past[seq], (int64_t)0), (int64_t)min((unsigned)a.keep, a.places)));
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

using ScoreKernel = void (*)(ScoreArgs);
template <typename T, int D>
ScoreKernel score_kernel_of(int group) {
    return group == 1 ? page_score_kernel<T, D, 1> : group == 2 ? page_score_kernel<T, D, 2> : page_score_kernel<T, D, 4>;
}
template <typename T>
ScoreKernel score_kernel_for(int dim, int group) {
    return dim == 64 ? score_kernel_of<T, 64>(group) : dim == 128 ? score_kernel_of<T, 128>(group) : score_kernel_of<T, 256>(group);
}
ScoreKernel score_kernel(const paella_page_select_plan* p) {
    const int group = p->heads / p->kv_heads;
    return p->dtype == PAELLA_F32 ? score_kernel_for<F32>(p->head_dim, group) : p->dtype == PAELLA_BF16 ? score_kernel_for<Bf16>(p->head_dim, group) : score_kernel_for<F16>(p->head_dim, group);
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

int64_t evict_slices(const paella_kv_cache* c) { return 2 * ceil_div((int64_t)c->head_dim * element_bytes(c->dtype), kSlice) + 1; }

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
    // a wave's turn is `batch` pages: enough workgroups to fill the device, none without a turn for each wave
    const int batch = 64 * kScoreAhead / std::max<int>(1, c->head_dim * element_bytes(c->dtype) / 16);
    p->splits = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(2048, rows), ceil_div(pages, 4 * std::max(1, batch))));
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
    if (stage) set_launch_dims(dims, (unsigned)(p->tokens * p->kv_heads), kPickWaves * 64, 0, 64);
    else set_launch_dims(dims, (unsigned)(p->tokens * p->kv_heads * p->splits), 256, 0, 128);
    loaded_dims(stage ? (const void*)page_pick_kernel : (const void*)score_kernel(p), dims);
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
    if (stage == 0) {
        ScoreArgs a;
        a.q = (const char*)q; a.bounds = (const char*)bounds;
        a.starts = b->starts; a.past = b->past; a.tables = b->tables; a.prefix_table = b->prefix_table;
        a.keys = (unsigned long long*)workspace; a.q_stride = q_stride * size;
        a.sequences = b->sequences; a.tokens = b->tokens; a.max_pages = b->max_pages; a.prefix_pages = (int)ceil_div(b->prefix_len, c->page_size); a.num_pages = c->num_pages;
        a.heads = p->heads; a.first = p->first; a.last = p->last; a.pitch = (unsigned)select_pitch(p);
        a.max_new = divisor((unsigned)b->max_new); a.kv_heads = divisor((unsigned)p->kv_heads); a.splits = divisor((unsigned)p->splits); a.page_size = divisor((unsigned)c->page_size);
        a.job_id = job_id; a.notifier = (Notifier*)notifier;
        launch(score_kernel(p), dim3((unsigned)(p->tokens * p->kv_heads * p->splits)), dim3(256), 0, (hipStream_t)stream, a);
    } else {
        PickArgs a;
        a.keys = (const unsigned long long*)workspace; a.pages = pages; a.starts = b->starts; a.past = b->past;
        a.sequences = b->sequences; a.max_pages = b->max_pages; a.prefix_pages = (int)ceil_div(b->prefix_len, c->page_size); a.count = p->count; a.pitch = (unsigned)select_pitch(p);
        a.max_new = divisor((unsigned)b->max_new); a.kv_heads = divisor((unsigned)p->kv_heads); a.page_size = divisor((unsigned)c->page_size);
        a.job_id = job_id; a.notifier = (Notifier*)notifier;
        launch(page_pick_kernel, dim3((unsigned)(p->tokens * p->kv_heads)), dim3(kPickWaves * 64), 0, (hipStream_t)stream, a);
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
    else set_launch_dims(dims, (unsigned)(d->sequences * c->kv_heads), kPickWaves * 64, 0, 64);
    loaded_dims(stage ? (const void*)evict_move_kernel : (const void*)evict_pick_kernel, dims);
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
    if (stage == 0) launch(evict_pick_kernel, dim3((unsigned)(d->sequences * c->kv_heads)), dim3(kPickWaves * 64), 0, (hipStream_t)stream, a);
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
