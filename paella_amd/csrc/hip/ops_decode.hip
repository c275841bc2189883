// Operators of a decoding step over a paged cache, all bounded by memory traffic or latency: appending keys and values
// (with norms and rotation), beam search's selection, and the reordering of the beams' caches.

#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>

#include "decode_common.h"

namespace {

using namespace paella;

// ------------------------------------------------------------------------------------------ append
// Per new token: x' = x / sqrt(mean(x^2) + eps) * w for each query and key head, pairs (a, b) turned by the angle p * f_i:
// (a cos - b sin, b cos + a sin); keys and values to the slot that the page table names.  One pass over the data: a workgroup per token,
// 16 bytes (8 values of 16 bits; two loads in 32 bits) per lane, a head per group of lanes that lane moves norm and pair up.
// Bounds: a few tokens the trips to memory in a row (length -> page -> stores), 3.8 us for 4 tokens of 12 heads of 64; a batch's step
// those and a token's 48 heads by one workgroup, on 64 of the 256 compute units, 6.8 us for 64 tokens of heads of 128 in bf16; prompts memory,
// 9 k such tokens 39 us, 207 MB at 5.3 TB/s, as fast as a copy.
struct AppendArgs {
    const char *q, *k, *v;
    char *q_out, *k_cache, *v_cache;
    const float *q_weight, *k_weight, *inv_freq;
    const int *starts, *past, *tables;
    int64_t q_stride, k_stride, v_stride;  // bytes
    int sequences, max_pages, prefix_len;
    Divisor max_new, page_size;
    int heads, kv_heads, dim, num_pages, rotary, interleaved, group_log2;  // a head's group of lanes: 2^group_log2 of 8 values each
    float eps, inv_dim;
    uint32_t job_id;
    Notifier* notifier;
};

template <typename T>
struct Eight {  // eight values of a head as they lie in memory
    u32x4 raw[T::bytes / 2];
    __device__ __forceinline__ void load(const char* p) {
#pragma unroll
        for (int i = 0; i < T::bytes / 2; ++i) raw[i] = *reinterpret_cast<const u32x4*>(p + 16 * i);
    }
    __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t to, unsigned at) const {
#pragma unroll
        for (int i = 0; i < T::bytes / 2; ++i) __builtin_amdgcn_raw_buffer_store_b128(raw[i], to, (int)(at + 16 * i), 0, kThrough);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        if constexpr (T::bytes == 4) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = as_float(raw[e / 4][e % 4]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const f32x2 v = unpack2<T>(raw[0][e]);
                x[2 * e] = v.x;
                x[2 * e + 1] = v.y;
            }
        }
    }
    __device__ __forceinline__ void set(const float (&x)[8]) {
        if constexpr (T::bytes == 4) {
#pragma unroll
            for (int e = 0; e < 8; ++e) raw[e / 4][e % 4] = as_word(x[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) raw[0][e] = pack2<T>(x[2 * e], x[2 * e + 1]);
        }
    }
};

// 16 bytes from an address on a value's boundary (rows of an odd number of logits begin anywhere, weights may be views).
__device__ __forceinline__ u32x4 load_unaligned(const char* p) {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

template <typename T>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
    hook_entry(a.notifier, a.job_id);
    // (cos, sin) of each pair's angle and the norms' weights, the same for every head.  In LDS rather than in registers: with them there five
    // workgroups fit a compute unit instead of eight, and the prompts' rate goes by the loads in flight.
    __shared__ __attribute__((aligned(16))) f32x2 turn[256];
    __shared__ __attribute__((aligned(16))) float norm[2][512];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.x;
    int seq, j;
    if (row_owner(a.starts, a.sequences, a.max_new, t, lane, &seq, &j)) {
        const int group = 1 << a.group_log2, li = lane & (group - 1);
        const int per_wave = 64 >> a.group_log2;
        const int total = a.heads + 2 * a.kv_heads;
        const int head_bytes = a.dim * T::bytes;
        const bool in_head = li * 8 < a.dim;
        constexpr int AHEAD = 4;  // heads of a lane that are requested together: all of them up to 4 * 4 * (64 / group), 64 at 128 values
        Eight<T> x[AHEAD];
        auto fetch = [&](int first) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int h = first + (u * 4 + wave) * per_wave + (lane >> a.group_log2);
                if (!in_head || h >= total) continue;
                const char* row = h < a.heads                ? a.q + t * a.q_stride + h * head_bytes
                                  : h < a.heads + a.kv_heads ? a.k + t * a.k_stride + (h - a.heads) * head_bytes
                                                             : a.v + t * a.v_stride + (h - a.heads - a.kv_heads) * head_bytes;
                x[u].load(row + li * 8 * T::bytes);
            }
        };
        fetch(0);
        // Trips to memory that do not wait for one another go out together: heads, length, weights and frequencies, then the page.
        const int past = a.past[seq];
        float wq[2], wk[2], freq = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = u * 256 + (int)threadIdx.x;
            wq[u] = a.q_weight && i < a.dim ? a.q_weight[i] : 0.f;
            wk[u] = a.k_weight && i < a.dim ? a.k_weight[i] : 0.f;
        }
        if ((int)threadIdx.x < a.rotary / 2) freq = a.inv_freq[threadIdx.x];
        // where the token goes; a place outside the table or the cache is none
        const unsigned own = (unsigned)max(past, 0) + (unsigned)j;
        const Quotient place = divide(own, a.page_size);
        const unsigned column = place.q, slot = place.r;
        int page = -1;
        if (column < (unsigned)a.max_pages) page = a.tables[(size_t)seq * a.max_pages + column];
        // The angle in revolutions, reduced to half a turn in 64 bits: in 32 bits a position of 100000 would be off by 0.006 radians.  Each pair once per
        // token, by one lane.
        if ((int)threadIdx.x < a.rotary / 2) {
            const double turns = ((double)a.prefix_len + (double)own) * (double)freq * 0.15915494309189533577;
            float s, c;
            sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
            turn[threadIdx.x] = f32x2{c, s};
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = u * 256 + (int)threadIdx.x;
            if (i < a.dim) {
                norm[0][i] = wq[u];
                norm[1][i] = wk[u];
            }
        }
        __syncthreads();
        page = __builtin_amdgcn_readfirstlane(page);  // (descriptors are built from it)
        const bool placed = (unsigned)page < (unsigned)a.num_pages;
        const size_t page_bytes = (size_t)a.kv_heads * a.page_size.d * head_bytes;
        const __amdgpu_buffer_rsrc_t to_q = descriptor(a.q_out + (size_t)t * a.heads * head_bytes);
        const __amdgpu_buffer_rsrc_t to_k = descriptor(a.k_cache + (placed ? page : 0) * page_bytes);
        const __amdgpu_buffer_rsrc_t to_v = descriptor(a.v_cache + (placed ? page : 0) * page_bytes);
        const int half = a.rotary >> 1, d0 = li * 8;  // rotary_dim is a multiple of 16: a lane's values are all in one half, or none is rotated
        const bool turned = d0 < a.rotary, lower = d0 < half;
        const int other = ((lane & ~(group - 1)) + (lower ? li + (half >> 3) : li - (half >> 3))) & 63;
        const f32x4* const turns = reinterpret_cast<const f32x4*>(turn + (!turned ? 0 : a.interleaved ? d0 >> 1 : lower ? d0 : d0 - half));
        for (int first = 0; first < total; first += AHEAD * 4 * per_wave) {
            if (first) fetch(first);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int at = first + (u * 4 + wave) * per_wave;
                if (at >= total) break;  // whole waves
                const int h = at + (lane >> a.group_log2);
                const bool live = in_head && h < total;
                const bool is_q = h < a.heads, is_v = h >= a.heads + a.kv_heads;
                float f[8];
                x[u].get(f);
                if (!live) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = 0.f;
                }
                if (a.q_weight || a.k_weight) {
                    float sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum += f[e] * f[e];
                    sum = lanes_sum(sum, a.group_log2);
                    if (is_q ? a.q_weight != nullptr : !is_v && a.k_weight != nullptr) {
                        const float r = rsqrtf(sum * a.inv_dim + a.eps);  // (the bare instruction takes subnormal numbers for 0, and eps may be 0)
                        const f32x4* const w = reinterpret_cast<const f32x4*>(norm[is_q ? 0 : 1] + (in_head ? d0 : 0));
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] = f[e] * r * w[e / 4][e % 4];
                    }
                }
                if (a.rotary) {
                    if (a.interleaved) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float c = turns[e / 2][e % 2 * 2], s = turns[e / 2][e % 2 * 2 + 1], p = f[2 * e], q = f[2 * e + 1];
                            f[2 * e] = turned ? p * c - q * s : p;
                            f[2 * e + 1] = turned ? q * c + p * s : q;
                        }
                    } else {
                        float partner[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) partner[e] = __shfl(f[e], other, 64);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float c = turns[e / 2][e % 2 * 2], s = turns[e / 2][e % 2 * 2 + 1];
                            if (turned) f[e] = f[e] * c + (lower ? -partner[e] : partner[e]) * s;
                        }
                    }
                }
                if (!live) continue;
                if (is_q) {
                    x[u].set(f);
                    x[u].store(to_q, (unsigned)(h * head_bytes + li * 8 * T::bytes));
                } else if (placed) {
                    const int hk = is_v ? h - a.heads - a.kv_heads : h - a.heads;
                    const unsigned to = ((unsigned)hk * a.page_size.d + slot) * head_bytes + li * 8 * T::bytes;
                    if (is_v) {
                        x[u].store(to_v, to);  // as it came
                    } else {
                        x[u].set(f);
                        x[u].store(to_k, to);
                    }
                }
            }
        }
    }
    hook_exit(a.notifier, a.job_id);
}

// ------------------------------------------------------------------------------------------ beam selection
// value(w, t) = scores[w] + x - lse_w: within a beam the order of the logits is the order of the values, so one pass over the logits takes each
// workgroup's running maximum, its sum of exponentials and its `count` largest logits; the workgroup that arrives last in a group puts the beams'
// logarithms together and merges the lists.  Few launches and few trips: 4 beams over 32000 fp32 logits take 7.6 us, of which the pass 3 and the merge 5
// (four trips to memory in a row); 128 rows of 131072 bf16 logits 15.4 us, of which reading 33.5 MB is 5.4, the pass's arithmetic keeps the vector
// units for about as long, and the merge is the rest.  (Registers for seven workgroups per compute unit, without the bound six: 16.9; eight, or seven with 32 fp32
// logits, do not do without scratch memory.)  64 logits per thread instead of 32: 19.9 (its registers leave three workgroups per compute unit).
//
// A logit as a number whose order is the logits' (-0 and 0 alike, NaN as -inf), with its index behind it such that the larger of two is the one to
// take; 0 is no candidate.
__device__ __forceinline__ unsigned order_key(float v) {
    const unsigned b = as_word(v + 0.f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) { return as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }
constexpr unsigned kLowestKey = 0x00800000u;  // order_key(-FLT_MAX); -inf lies right below
__device__ __forceinline__ unsigned long long entry(unsigned key, unsigned index) { return (unsigned long long)key << 32 | (0xFFFFFFFFu - index); }

constexpr int kMostLists = 1024;     // beams * splits
constexpr int kMostSplits = 64;      // parts of a beam that the merge adds up
constexpr int kMostStaged = 1024;    // entries that the merge fetches at once
constexpr int kCounterStride = 32;   // a cache line each: counts on one line go one after the other, 2048 of 32 groups for 7 us
constexpr int kWaveCandidates = 128;  // of one wave's logits that go on to the workgroup's ranking

struct SelectArgs {
    const char* logits;
    int64_t row_stride;  // bytes
    const float* scores;
    const unsigned char* finished;
    int pad_token, groups, beams, vocab, count, splits;
    unsigned long long* sums;     // [groups * beams * splits]: maximum and sum of exponentials
    unsigned long long* entries;  // [groups * beams * splits][count], best first
    unsigned* counters;           // [groups][kCounterStride], zero between launches
    float* out_scores;
    int *out_parents, *out_tokens;
    uint32_t job_id;
    Notifier* notifier;
};

__device__ __forceinline__ void put64(unsigned long long* p, unsigned long long v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ unsigned long long get64(const unsigned long long* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <typename T, int VALUES>
__device__ __forceinline__ void load_logits(const char* row, int first, int vocab, float (&x)[VALUES]) {
    constexpr int VEC = 16 / T::bytes;
    if (first + 256 * VALUES <= vocab) {  // all requested ahead of the first use
        u32x4 w[VALUES / VEC];
#pragma unroll
        for (int i = 0; i < VALUES / VEC; ++i) w[i] = load_unaligned(row + (unsigned)(first + (i * 256 + (int)threadIdx.x) * VEC) * T::bytes);
#pragma unroll
        for (int i = 0; i < VALUES / VEC; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (T::bytes == 4) {
                    x[i * VEC + e] = as_float(w[i][e]);
                } else {
                    const f32x2 two = unpack2<T>(w[i][e]);
                    x[i * VEC + 2 * e] = two.x;
                    x[i * VEC + 2 * e + 1] = two.y;
                }
            }
    } else {  // the row's end: one by one, the last logit in place of what is behind it
        unsigned w[VALUES];
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            const unsigned at = (unsigned)min(first + (i / VEC * 256 + (int)threadIdx.x) * VEC + i % VEC, vocab - 1);
            if constexpr (T::bytes == 4) w[i] = *reinterpret_cast<const unsigned*>(row + at * 4);
            else w[i] = *reinterpret_cast<const unsigned short*>(row + at * 2);
        }
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            const float v = T::bytes == 4 ? as_float(w[i]) : unpack2<T>(w[i]).x;
            x[i] = first + (i / VEC * 256 + (int)threadIdx.x) * VEC + i % VEC < vocab ? v : -INFINITY;
        }
    }
}

// How many lanes of `who` come before this one.
__device__ __forceinline__ int lanes_before(unsigned long long who) {
    return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(who >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)who, 0));
}

// What at least K of the lanes' keys reach (0 where fewer lanes have one): their K-th largest, bit by bit, to the upper 16 bits -- a few more logits
// pass than would behind all 32, and it takes half the time.
__device__ __forceinline__ unsigned kth_of_lanes(unsigned key, int K) {
    unsigned bound = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const unsigned trial = bound | (1u << bit);
        if (__popcll(__ballot(key >= trial)) >= K) bound = trial;
    }
    return bound;
}

// c / d for c < 2048 by d's reciprocal: the quotient's distance from a whole number is half of 1 / d at least.
__device__ __forceinline__ int small_div(int c, float inv) { return (int)(((float)c + 0.5f) * inv); }

constexpr float kLog2e = 1.44269504088896340736f;

// Calls emit(rank, i) for the K best of n (value, where) pairs in LDS, larger values and then smaller places first; no two places are alike.  Few: each
// counts those ahead of it.  Many (equal logits by the hundred): one after the other.
template <typename Emit>
__device__ __forceinline__ void best_of(const double* value, const unsigned* where, int n, int K, Emit emit) {
    constexpr int kCounted = 512;
    __shared__ double step_value[4];
    __shared__ unsigned step_where[4];
    __shared__ int step_at[4];
    auto ahead = [](double v, unsigned f, double w, unsigned g) { return (bool)((int)(v > w) | ((int)(v == w) & (int)(f < g))); };
    if (n <= kCounted) {
        for (int c = threadIdx.x; c < n; c += 256) {
            const double v = value[c];
            const unsigned f = where[c];
            int rank = 0;
#pragma unroll 8
            for (int o = 0; o < n; ++o) rank += ahead(value[o], where[o], v, f);
            if (rank < K) emit(rank, c);
        }
        return;
    }
    double taken = INFINITY;  // the pair taken last
    unsigned taken_where = 0;
    for (int rank = 0; rank < K; ++rank) {
        double v = -INFINITY;
        unsigned f = 0xFFFFFFFFu;
        int at = -1;
        for (int c = threadIdx.x; c < n; c += 256)
            if (ahead(taken, taken_where, value[c], where[c]) && (at < 0 || ahead(value[c], where[c], v, f))) {
                v = value[c];
                f = where[c];
                at = c;
            }
        for (int off = 32; off > 0; off >>= 1) {
            const double w = __shfl_xor(v, off, 64);
            const unsigned g = __shfl_xor(f, off, 64);
            const int other = __shfl_xor(at, off, 64);
            if (other >= 0 && (at < 0 || ahead(w, g, v, f))) {
                v = w;
                f = g;
                at = other;
            }
        }
        if ((threadIdx.x & 63) == 0) {
            step_value[threadIdx.x >> 6] = v;
            step_where[threadIdx.x >> 6] = f;
            step_at[threadIdx.x >> 6] = at;
        }
        __syncthreads();
        at = -1;
        for (int w = 0; w < 4; ++w)
            if (step_at[w] >= 0 && (at < 0 || ahead(step_value[w], step_where[w], v, f))) {
                v = step_value[w];
                f = step_where[w];
                at = step_at[w];
            }
        taken = v;
        taken_where = f;
        if (threadIdx.x == 0) emit(rank, at);
        __syncthreads();
    }
}

template <typename T, int VALUES>
__global__ __launch_bounds__(256, T::bytes == 4 && VALUES == 32 ? 5 : 7) void beam_select_kernel(SelectArgs a) {
    hook_entry(a.notifier, a.job_id);
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float wave_top[4], wave_total[4];
    __shared__ unsigned wave_bound[4], found, arrived;
    __shared__ double row_lse[33], row_score[32];
    constexpr int VEC = 16 / T::bytes;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.x / a.splits, split = blockIdx.x - row * a.splits;
    const int group = row / a.beams;
    const int K = a.count;

    if (!a.finished || !a.finished[row]) {
        unsigned long long* const cand = reinterpret_cast<unsigned long long*>(lds);
        const int first = split * 256 * VALUES;
        float x[VALUES];
        load_logits<T, VALUES>(a.logits + (size_t)row * a.row_stride, first, a.vocab, x);
        if (threadIdx.x == 0) found = 0;
        float mine = -INFINITY;  // (a NaN loses against any number)
#pragma unroll
        for (int i = 0; i < VALUES; ++i) mine = fmaxf(mine, x[i]);
        const float top = wave_max_f(mine);
        // 2^(x log2e - base): what the base lost by its rounding is the same in every term and comes back as one factor
        const float base = top == -INFINITY ? 0.f : top * kLog2e;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < VALUES; ++i) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], kLog2e, -base));
        sum = wave_sum_f(sum);
        if (sum > 0.f && sum < INFINITY) {
            sum *= __builtin_amdgcn_exp2f(-__builtin_fmaf(top, kLog2e, -base));
        } else {  // NaN among the logits, a maximum so far from 0 that the base overflows (the type's lowest, where everything is masked), or an infinity; NaN where there is no
                  // number among them, which the sums further on leave out
            sum = 0.f;
#pragma unroll
            for (int i = 0; i < VALUES; ++i) sum += x[i] == x[i] ? __builtin_amdgcn_exp2f((x[i] - top) * kLog2e) : 0.f;
            sum = wave_sum_f(sum);
        }
        if (lane == 0) {
            wave_top[wave] = top;
            wave_total[wave] = sum;
        }
        // A bound that at least K of the workgroup's logits reach, and few others: what a quarter of K of each wave's lanes reach with their best.
        unsigned bound = kth_of_lanes(order_key(mine), (K + 3) / 4);
        if (lane == 0) wave_bound[wave] = bound;
        __syncthreads();
        bound = max(min(min(wave_bound[0], wave_bound[1]), min(wave_bound[2], wave_bound[3])), kLowestKey);
        const float least = key_value(bound);
        unsigned long long* const own = cand + wave * kWaveCandidates;
        const int lane_base = first + (int)threadIdx.x * VEC;
        auto behind = [](int i) { return i / VEC * 256 * VEC + i % VEC; };  // of value i, how far behind the lane's first index
        int taken = 0;
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            const unsigned long long who = __ballot(x[i] >= least);
            if (who) {
                const int at = taken + lanes_before(who);
                if (x[i] >= least && at < kWaveCandidates) own[at] = entry(order_key(x[i]), (unsigned)(lane_base + behind(i)));
                taken += __popcll(who);
            }
        }
        if (taken > kWaveCandidates) {  // equal logits, or the best ones in few lanes: the K-th of all of the wave's logits, ties by index
            unsigned key[VALUES];
#pragma unroll
            for (int i = 0; i < VALUES; ++i) key[i] = order_key(x[i] == x[i] ? x[i] : -INFINITY);
            auto count = [&](auto wanted) {
                int n = 0;
#pragma unroll
                for (int i = 0; i < VALUES; ++i) n += __popcll(__ballot(wanted(i)));
                return n;
            };
            bound = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const unsigned trial = bound | (1u << bit);
                if (count([&](int i) { return key[i] >= trial; }) >= K) bound = trial;
            }
            bound = max(bound, kLowestKey);
            const int larger = count([&](int i) { return key[i] > bound; });
            int last = 0;  // the largest index with fewer than the wanted number of equals below it
            for (int bit = 19; bit >= 0; --bit) {
                const int trial = last | (1 << bit);
                if (count([&](int i) { return key[i] == bound && lane_base < trial - behind(i); }) < K - larger) last = trial;
            }
            taken = 0;
#pragma unroll
            for (int i = 0; i < VALUES; ++i) {
                const bool take = key[i] > bound || (key[i] == bound && lane_base <= last - behind(i));
                const unsigned long long who = __ballot(take);
                if (take) own[taken + lanes_before(who)] = entry(key[i], (unsigned)(lane_base + behind(i)));
                taken += __popcll(who);
            }
        }
        // one list of the four waves' (their order does not matter: the entries are ranked)
        unsigned at = 0;
        if (lane == 0) at = atomicAdd(&found, (unsigned)taken);
        at = __builtin_amdgcn_readfirstlane(at);
        unsigned long long* const all = cand + 4 * kWaveCandidates;
        for (int c = lane; c < taken; c += 64) all[at + c] = own[c];
        __syncthreads();
        const int n = (int)found;
        unsigned long long* const to = a.entries + (size_t)blockIdx.x * K;
        for (int c = threadIdx.x; c < n; c += 256) {
            const unsigned long long e = all[c];
            int rank = 0;
#pragma unroll 8
            for (int o = 0; o < n; ++o) rank += all[o] > e;
            if (rank < K) put64(to + rank, e);
        }
        for (int c = n + threadIdx.x; c < K; c += 256) put64(to + c, 0);
        if (threadIdx.x == 255) {
            const float m = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3]));
            float s = 0.f;
            if (fabsf(m) < INFINITY) {
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    if (wave_total[w] > 0.f) s += wave_total[w] * __builtin_amdgcn_exp2f((wave_top[w] - m) * kLog2e);
            }
            put64(a.sums + blockIdx.x, (unsigned long long)as_word(m) << 32 | as_word(s));
        }
    }

    // The last workgroup of the group merges.  As in the convs' split reductions: the stores above go through to memory ahead of the count.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const int lists = a.beams * a.splits;
    if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(a.counters + group * kCounterStride, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(arrived) == (unsigned)lists - 1) {
        const bool whole = lists * K <= kMostStaged;  // every list's entries are fetched at once, else the best ones and then those of the lists that matter
        const int staged = whole ? lists * K : lists, per = whole ? K : 1;
        // LDS: (maximum, sum) per list, or what has been found; values and flat indices w * vocab + t of the staged entries
        double* const value = reinterpret_cast<double*>(lds);
        unsigned* const where = reinterpret_cast<unsigned*>(value + max(staged, min(lists, K) * K));
        f32x2* const ms = reinterpret_cast<f32x2*>(lds);
        const int first_list = group * lists, first_row = group * a.beams;
        const unsigned long long* const from = a.entries + (size_t)first_list * K;
        auto ended = [&](int w) { return a.finished && a.finished[first_row + w]; };
        // All trips to memory that do not wait for one another go out together.
        constexpr int AHEAD = kMostStaged / 256;
        const float inv_per = 1.f / (float)per, inv_splits = 1.f / (float)a.splits;
        auto beam_of = [&](int l) { return small_div(l, inv_splits); };
        unsigned long long e[AHEAD];
        const double score = (int)threadIdx.x < a.beams ? (double)a.scores[first_row + threadIdx.x] : 0.;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int c = u * 256 + (int)threadIdx.x;
            e[u] = 0;
            if (c < staged) {
                const int l = small_div(c, inv_per);
                if (!ended(beam_of(l))) e[u] = get64(from + (size_t)l * K + (c - l * per));
            }
        }
        for (int l = threadIdx.x; l < lists; l += 256) {
            const unsigned long long s = ended(beam_of(l)) ? 0 : get64(a.sums + first_list + l);
            ms[l] = f32x2{as_float((unsigned)(s >> 32)), as_float((unsigned)s)};
        }
        if (threadIdx.x == 0) found = 0;
        __syncthreads();
        for (int w = threadIdx.x >> 4; w < (a.beams + 15) / 16 * 16; w += 16) {  // a beam's parts by 16 lanes
            f32x2 p[kMostSplits / 16];
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < kMostSplits / 16; ++i) {
                const int s = i * 16 + (lane & 15);
                p[i] = f32x2{-INFINITY, 0.f};
                if (w < a.beams && s < a.splits) p[i] = ms[w * a.splits + s];
                m = fmaxf(m, p[i].x);
            }
            m = row_all(m, [](float x, float y) { return fmaxf(x, y); });
            double total = 0.;
#pragma unroll
            for (int i = 0; i < kMostSplits / 16; ++i)
                if (p[i].y > 0.f) total += (double)p[i].y * (double)__builtin_amdgcn_exp2f((p[i].x - m) * kLog2e);
            total = row_all(total, [](double x, double y) { return x + y; });
            if ((lane & 15) == 0 && w < a.beams) {
                row_lse[w] = total;
                row_score[w] = (double)m;
            }
        }
        __syncthreads();
        if ((int)threadIdx.x < a.beams) {
            const double m = row_score[threadIdx.x];
            row_lse[threadIdx.x] = m == INFINITY ? INFINITY : m + log(row_lse[threadIdx.x]);
            row_score[threadIdx.x] = score;
        }
        __syncthreads();
        // in 64 bits: 32 would make equals of neighbours, and the lower index would win
        auto finite = [](double v) { return v > -INFINITY && v < INFINITY ? v : -INFINITY; };
        auto worth = [&](unsigned long long e, int w) {
            return e ? finite(row_score[w] + ((double)key_value((unsigned)(e >> 32)) - row_lse[w])) : -INFINITY;
        };
        auto flat = [&](unsigned long long e, int w) { return (unsigned)w * a.vocab + (0xFFFFFFFFu - (unsigned)e); };
        // Of n entries (up to AHEAD * 256 looked at first, by all threads) those that can be among the K best go to LDS: a bound that K of them reach is the
        // K-th largest of a wave's lanes' best, rounded down to 32 bits.
        double least = -INFINITY;
        auto put = [&](double v, unsigned f) {
            if (v > -INFINITY && v >= least) {
                const unsigned at = atomicAdd(&found, 1u);
                value[at] = v;
                where[at] = f;
            }
        };
        double v[AHEAD];
        unsigned f[AHEAD];
        auto filter = [&]() {
            double best = v[0];
#pragma unroll
            for (int u = 1; u < AHEAD; ++u) best = fmax(best, v[u]);
            float down = (float)best;
            if ((double)down > best) down = as_float(as_word(down) + (down > 0.f ? -1 : 1));  // (to nearest went up; 0 is exact)
            const unsigned reached = kth_of_lanes(order_key(down), K);
            if (lane == 0) wave_top[wave] = reached > kLowestKey ? key_value(reached) : -INFINITY;
            __syncthreads();
            least = fmax(least, (double)fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3])));
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) put(v[u], f[u]);
        };
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            v[u] = -INFINITY;
            f[u] = 0;
            const int c = u * 256 + (int)threadIdx.x;
            if (c < staged) {
                const int w = beam_of(small_div(c, inv_per));
                if (!ended(w)) {
                    v[u] = worth(e[u], w);
                    f[u] = flat(e[u], w);
                } else if (c == w * a.splits * per) {
                    v[u] = finite(row_score[w]);
                    f[u] = (unsigned)w * a.vocab + (unsigned)a.pad_token;
                }
            }
        }
        filter();
        __syncthreads();
        int n = (int)found;
        if (!whole) {  // these were the lists' best: the K best lists hold the K best entries
            __shared__ unsigned taken_list[64];
            const int most = min(n, K);
            best_of(value, where, n, K, [&](int rank, int i) {
                const unsigned w = where[i] / (unsigned)a.vocab, t = where[i] - w * (unsigned)a.vocab;
                taken_list[rank] = w * (unsigned)a.splits + (ended(w) ? 0 : t / (256 * VALUES));
                if (rank == K - 1) row_lse[32] = value[i];
            });
            __syncthreads();
            if (n >= K) least = row_lse[32];  // what the last of them begins with
            if (threadIdx.x == 0) found = 0;
            auto fetch = [&](int c, double& v, unsigned& f) {  // the lists' first entries first: they give the better bound
                v = -INFINITY;
                f = 0;
                if (c >= most * K) return;
                const int i = c / most, l = (int)taken_list[c - i * most], w = beam_of(l);
                if (!ended(w)) {
                    const unsigned long long e = get64(from + (size_t)l * K + i);
                    v = worth(e, w);
                    f = flat(e, w);
                } else if (i == 0) {
                    v = row_score[w];
                    f = (unsigned)w * a.vocab + (unsigned)a.pad_token;
                }
            };
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) fetch(u * 256 + (int)threadIdx.x, v[u], f[u]);
            filter();
            for (int c = AHEAD * 256 + (int)threadIdx.x; c < most * K; c += 256) {
                double v;
                unsigned f;
                fetch(c, v, f);
                put(v, f);
            }
            __syncthreads();
            n = (int)found;
        }
        const size_t out = (size_t)group * K;
        best_of(value, where, n, K, [&](int rank, int i) {
            if (i < 0) return;
            const unsigned w = where[i] / (unsigned)a.vocab;
            store_out(a.out_scores + out + rank, (float)value[i]);
            __hip_atomic_store(a.out_parents + out + rank, (int)w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(a.out_tokens + out + rank, (int)(where[i] - w * (unsigned)a.vocab), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        });
        for (int c = n + threadIdx.x; c < K; c += 256) {
            store_out(a.out_scores + out + c, -INFINITY);
            __hip_atomic_store(a.out_parents + out + c, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(a.out_tokens + out + c, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (threadIdx.x == 0) __hip_atomic_store(a.counters + group * kCounterStride, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    hook_exit(a.notifier, a.job_id);
}

// ------------------------------------------------------------------------------------------ reordering of the beams' caches
// A workgroup per child and key head: the tokens that the parent's last page holds lie side by side for a head, keys and values each one run of
// bytes.  Nothing is copied for a parent's first child; the first head's workgroup writes the child's row of the table.  4 beams 3.0 us (launch and three trips
// to memory); 256 children, 160 half pages of 64 tokens of 8 heads of 128 in bf16, 42 MB, 8.5 us: 4.9 TB/s, as fast as a copy.
struct ReorderArgs {
    char *k_cache, *v_cache;
    const int *parents, *past, *tables, *spare;
    int *tables_out, *past_out;
    int groups, beams, count, max_pages, num_pages, kv_heads, page_size, head_bytes;
    uint32_t job_id;
    Notifier* notifier;
};

__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderArgs a) {
    hook_entry(a.notifier, a.job_id);
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x / a.kv_heads, head = blockIdx.x - row * a.kv_heads;
    const int group = row / a.count, child = row - group * a.count;
    const int parent = a.parents[row];
    const int spare = __builtin_amdgcn_readfirstlane(a.spare[row]);
    bool first = true;
    for (int c = 0; c < child && first; c += 64) first = !__any(c + lane < child && a.parents[group * a.count + c + lane] == parent);
    if ((unsigned)parent < (unsigned)a.beams) {
        const int source = group * a.beams + parent;
        const unsigned past = (unsigned)max(a.past[source], 0);
        const unsigned full = past / (unsigned)a.page_size, rest = past - full * (unsigned)a.page_size;
        const int* const from = a.tables + (size_t)source * a.max_pages;
        const bool inside = full < (unsigned)a.max_pages;
        int last = -1;
        if (inside && rest) last = __builtin_amdgcn_readfirstlane(from[full]);
        if (head == 0) {
            int* const to = a.tables_out + (size_t)row * a.max_pages;
            const int whole = (int)min(full, (unsigned)a.max_pages);
            for (int i = threadIdx.x; i < whole; i += 256) __hip_atomic_store(to + i, from[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (threadIdx.x == 0) {
                if (inside) __hip_atomic_store(to + full, first && rest ? last : spare, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(a.past_out + row, (int)past, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        if (!first && (unsigned)last < (unsigned)a.num_pages && (unsigned)spare < (unsigned)a.num_pages) {
            const size_t run = (size_t)a.page_size * a.head_bytes, page_bytes = run * a.kv_heads;
            const unsigned bytes = rest * (unsigned)a.head_bytes;
            const size_t src = last * page_bytes + head * run, dst = spare * page_bytes + head * run;
            const __amdgpu_buffer_rsrc_t to_k = descriptor(a.k_cache + dst), to_v = descriptor(a.v_cache + dst);
            for (unsigned at = threadIdx.x * 16; at < bytes; at += 4096) {
                const u32x4 x = *reinterpret_cast<const u32x4*>(a.k_cache + src + at);
                const u32x4 y = *reinterpret_cast<const u32x4*>(a.v_cache + src + at);
                __builtin_amdgcn_raw_buffer_store_b128(x, to_k, (int)at, 0, kThrough);
                __builtin_amdgcn_raw_buffer_store_b128(y, to_v, (int)at, 0, kThrough);
            }
        }
    } else if (head == 0 && threadIdx.x == 0) {
        __hip_atomic_store(a.past_out + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    hook_exit(a.notifier, a.job_id);
}

using AppendKernel = void (*)(AppendArgs);
AppendKernel append_kernel(int dtype) {
    return dtype == PAELLA_F32 ? kv_append_kernel<F32> : dtype == PAELLA_BF16 ? kv_append_kernel<Bf16> : kv_append_kernel<F16>;
}

using SelectKernel = void (*)(SelectArgs);
SelectKernel select_kernel(int dtype, int values) {
    if (values == 8) return dtype == PAELLA_F32 ? beam_select_kernel<F32, 8> : dtype == PAELLA_BF16 ? beam_select_kernel<Bf16, 8> : beam_select_kernel<F16, 8>;
    return dtype == PAELLA_F32 ? beam_select_kernel<F32, 32> : dtype == PAELLA_BF16 ? beam_select_kernel<Bf16, 32> : beam_select_kernel<F16, 32>;
}

int append_check(const paella_kv_append_desc* d, const paella_kv_cache* c, const paella_kv_batch* b) {
    if (!d || !cache_extents_ok(c) || !batch_extents_ok(b)) return PAELLA_EINVAL;
    if (b->tokens > kMostWorkgroups || d->heads < 0 || d->heads > 65536 || d->rotary_dim < 0 || d->rotary_dim % 16 || d->rotary_dim > c->head_dim || !(d->eps >= 0.f)) return PAELLA_EINVAL;
    return 0;
}

// LDS of a selection: the waves' candidates of the pass over the logits and their common list, and the merge's entries, in the same place.  At most 48 KiB (64 lists of 64
// entries), which any launch may have.
unsigned select_lds(const paella_beam_select_plan* p) {
    const unsigned lists = p->beams * p->splits, taken = ((unsigned)p->count < lists ? p->count : lists) * p->count;
    const unsigned staged = lists * p->count <= kMostStaged ? lists * p->count : lists;
    const unsigned merge = (staged > taken ? staged : taken) * 12, pass = 8 * kWaveCandidates * 8;
    return ((merge > pass ? merge : pass) + 15) / 16 * 16;
}

bool select_plan_ok(const paella_beam_select_plan* p) {
    if (!p || p->dtype < PAELLA_F32 || p->dtype > PAELLA_F16 || p->groups <= 0 || p->beams <= 0 || p->beams > 32 || p->vocab <= 0 || p->vocab > 524288) return false;
    if (p->count <= 0 || p->count > 64 || (p->values != 8 && p->values != 32)) return false;
    const int splits = (p->vocab + 256 * p->values - 1) / (256 * p->values);
    return p->splits == splits && splits <= kMostSplits && p->beams * splits <= kMostLists && (double)p->groups * p->beams * splits <= kMostWorkgroups;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

size_t select_workspace(const paella_beam_select_plan* p) {
    const size_t lists = (size_t)p->groups * p->beams * p->splits;
    return up256((size_t)p->groups * 4 * kCounterStride) + up256(lists * 8) + lists * p->count * 8;
}

}  // namespace

extern "C" {

int paella_kv_append_dims(const paella_kv_append_desc* desc, const paella_kv_cache* cache, const paella_kv_batch* batch, paella_launch_dims* dims) {
    if (int rc = append_check(desc, cache, batch)) return rc;
    if (!dims) return PAELLA_EINVAL;
    set_launch_dims(dims, (unsigned)batch->tokens, 256, 0, 64);
    loaded_dims((const void*)append_kernel(cache->dtype), dims);
    return 0;
}

int paella_kv_append_launch(const paella_kv_append_desc* d, const paella_kv_cache* c, const paella_kv_batch* b, const void* q, const void* k, const void* v,
                            const float* q_weight, const float* k_weight, const float* inv_freq, void* q_out, void* stream, uint32_t job_id,
                            void* notifier) {
    if (int rc = append_check(d, c, b)) return rc;
    if (!cache_ok(c) || !batch_ok(b) || !k || !v || (d->heads > 0) != (q != nullptr) || (d->heads > 0) != (q_out != nullptr)) return PAELLA_EINVAL;
    if (d->rotary_dim && !inv_freq) return PAELLA_EINVAL;
    const int64_t size = element_bytes(c->dtype), kv_row = (int64_t)c->kv_heads * c->head_dim, q_row = (int64_t)d->heads * c->head_dim;
    if (d->k_stride < kv_row || d->v_stride < kv_row || d->k_stride % 8 || d->v_stride % 8) return PAELLA_EINVAL;
    if (d->heads && (d->q_stride < q_row || d->q_stride % 8 || q_row * size >= (int64_t)1 << 31)) return PAELLA_EINVAL;
    if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out) & 15) != 0) return PAELLA_EINVAL;
    if (d->heads && overlap(q, (double)(b->tokens - 1) * d->q_stride * size + q_row * size, q_out, (double)b->tokens * q_row * size) &&
        !(q == q_out && d->q_stride == q_row))
        return PAELLA_EINVAL;
    // other tokens' workgroups may still read keys and values
    const double out_bytes = (double)b->tokens * q_row * size;
    if (d->heads && (rows_overlap(k, b->tokens, d->k_stride * size, kv_row * size, q_out, out_bytes) || over_cache(c, q_out, out_bytes) ||
                     rows_overlap(v, b->tokens, d->v_stride * size, kv_row * size, q_out, out_bytes)))
        return PAELLA_EINVAL;
    AppendArgs a;
    a.q = (const char*)q; a.k = (const char*)k; a.v = (const char*)v;
    a.q_out = (char*)q_out; a.k_cache = (char*)c->k; a.v_cache = (char*)c->v;
    a.q_weight = q_weight; a.k_weight = k_weight; a.inv_freq = inv_freq;
    a.starts = b->starts; a.past = b->past; a.tables = b->tables;
    a.q_stride = d->q_stride * size; a.k_stride = d->k_stride * size; a.v_stride = d->v_stride * size;
    a.sequences = b->sequences; a.max_pages = b->max_pages; a.prefix_len = b->prefix_len;
    a.max_new = divisor((unsigned)b->max_new); a.page_size = divisor((unsigned)c->page_size);
    a.heads = d->heads; a.kv_heads = c->kv_heads; a.dim = c->head_dim; a.num_pages = c->num_pages;
    a.rotary = d->rotary_dim; a.interleaved = d->interleaved; a.eps = d->eps; a.inv_dim = 1.f / (float)c->head_dim;
    a.group_log2 = 0;
    while ((8 << a.group_log2) < c->head_dim) ++a.group_log2;
    a.job_id = job_id; a.notifier = (Notifier*)notifier;
    launch(append_kernel(c->dtype), dim3(b->tokens), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

int paella_beam_select_plan_make(int dtype, int groups, int beams, int vocab, int count, paella_beam_select_plan* p) {
    if (!p || dtype < PAELLA_F32 || dtype > PAELLA_F16 || groups <= 0 || beams <= 0 || vocab <= 0 || count <= 0) return PAELLA_EINVAL;
    if (beams > 32 || vocab > 524288 || count > 64) return PAELLA_ENOSUP;
    *p = paella_beam_select_plan{};
    p->dtype = dtype; p->groups = groups; p->beams = beams; p->vocab = vocab; p->count = count;
    // 32 logits per thread where that still gives every compute unit a workgroup, else 8 (up to the lists per beam that the merge takes)
    const int long_splits = (vocab + 8191) / 8192, short_splits = (vocab + 2047) / 2048;
    p->values = (double)groups * beams * long_splits >= 256 || short_splits > kMostSplits || beams * short_splits > kMostLists ? 32 : 8;
    p->splits = p->values == 32 ? long_splits : short_splits;
    if (!select_plan_ok(p)) return PAELLA_ENOSUP;
    const size_t lists = (size_t)groups * beams * p->splits;
    p->workspace_bytes = select_workspace(p);
    set_launch_dims(&p->dims, (unsigned)lists, 256, select_lds(p), 64);
    p->flops = 4.0 * groups * beams * vocab;
    p->bytes = (double)groups * beams * vocab * element_bytes(dtype) + groups * (beams * 4.0 + count * 12.0);
    return 0;
}

int paella_beam_select_dims(const paella_beam_select_plan* p, paella_launch_dims* dims) {
    if (!select_plan_ok(p) || !dims) return PAELLA_EINVAL;
    set_launch_dims(dims, (unsigned)(p->groups * p->beams * p->splits), 256, select_lds(p), 64);
    loaded_dims((const void*)select_kernel(p->dtype, p->values), dims);
    return 0;
}

int paella_beam_select_launch(const paella_beam_select_plan* p, const void* logits, int64_t row_stride, const float* scores, const uint8_t* finished,
                              int pad_token, float* out_scores, int32_t* out_parents, int32_t* out_tokens, void* workspace, void* stream,
                              uint32_t job_id, void* notifier) {
    if (!select_plan_ok(p) || !logits || !scores || !out_scores || !out_parents || !out_tokens || !workspace) return PAELLA_EINVAL;
    if (row_stride < p->vocab || (finished && (pad_token < 0 || pad_token >= p->vocab))) return PAELLA_EINVAL;
    const int size = element_bytes(p->dtype);
    if (((uintptr_t)logits & (size - 1)) || ((uintptr_t)workspace & 15)) return PAELLA_EINVAL;
    const size_t lists = (size_t)p->groups * p->beams * p->splits;
    // A group is merged while others are still read.  Its own scores have been by then: they may become the next step's.
    const int64_t beams = (int64_t)p->groups * p->beams;
    const double in_bytes = (double)beams * 4, bytes = (double)p->groups * p->count * 4, space = (double)select_workspace(p);
    const bool in_place = p->groups == 1 || (out_scores == scores && p->count == p->beams);
    const void* const outs[3] = {out_scores, out_parents, out_tokens};
    for (int i = 0; i < 3; ++i) {
        if (rows_overlap(logits, beams, row_stride * size, (int64_t)p->vocab * size, outs[i], bytes) || (finished && overlap(finished, (double)beams, outs[i], bytes)) ||
            (!(i == 0 && in_place) && overlap(scores, in_bytes, outs[i], bytes)) || overlap(outs[i], bytes, outs[(i + 1) % 3], bytes) || overlap(workspace, space, outs[i], bytes))
            return PAELLA_EINVAL;
    }
    if (rows_overlap(logits, beams, row_stride * size, (int64_t)p->vocab * size, workspace, space) || overlap(scores, in_bytes, workspace, space)) return PAELLA_EINVAL;
    SelectArgs a;
    a.logits = (const char*)logits; a.row_stride = row_stride * size; a.scores = scores; a.finished = finished;
    a.pad_token = pad_token; a.groups = p->groups; a.beams = p->beams; a.vocab = p->vocab; a.count = p->count; a.splits = p->splits;
    a.counters = (unsigned*)workspace;
    a.sums = (unsigned long long*)((char*)workspace + up256((size_t)p->groups * 4 * kCounterStride));
    a.entries = (unsigned long long*)((char*)a.sums + up256(lists * 8));
    a.out_scores = out_scores; a.out_parents = out_parents; a.out_tokens = out_tokens;
    a.job_id = job_id; a.notifier = (Notifier*)notifier;
    const unsigned lds = select_lds(p);
    const SelectKernel kernel = select_kernel(p->dtype, p->values);
    launch(kernel, dim3((unsigned)lists), dim3(256), lds, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

static int reorder_check(const paella_beam_reorder_desc* d, const paella_kv_cache* c) {
    if (!d || !cache_extents_ok(c) || d->groups <= 0 || d->beams <= 0 || d->count <= 0 || d->max_pages <= 0) return PAELLA_EINVAL;
    const double rows = (double)d->groups * (d->count > d->beams ? d->count : d->beams);
    return rows * c->kv_heads <= kMostWorkgroups ? 0 : PAELLA_EINVAL;
}

int paella_beam_reorder_dims(const paella_beam_reorder_desc* d, const paella_kv_cache* c, paella_launch_dims* dims) {
    if (int rc = reorder_check(d, c)) return rc;
    if (!dims) return PAELLA_EINVAL;
    set_launch_dims(dims, (unsigned)(d->groups * d->count * c->kv_heads), 256, 0, 32);
    loaded_dims((const void*)beam_reorder_kernel, dims);
    return 0;
}

int paella_beam_reorder_launch(const paella_beam_reorder_desc* d, const paella_kv_cache* c, const int32_t* parents, const int32_t* past, const int32_t* tables,
                               const int32_t* spare, int32_t* tables_out, int32_t* past_out, void* stream, uint32_t job_id, void* notifier) {
    if (int rc = reorder_check(d, c)) return rc;
    if (!cache_ok(c) || !parents || !past || !tables || !spare || !tables_out || !past_out) return PAELLA_EINVAL;
    // every output: written by one workgroup while others may still read the inputs
    const double in = (double)d->groups * d->beams * 4, out = (double)d->groups * d->count * 4;
    const struct { const void* at; double bytes; } outs[2] = {{tables_out, out * d->max_pages}, {past_out, out}};
    for (const auto& o : outs)
        if (overlap(tables, in * d->max_pages, o.at, o.bytes) || overlap(past, in, o.at, o.bytes) || overlap(parents, out, o.at, o.bytes) ||
            overlap(spare, out, o.at, o.bytes) || over_cache(c, o.at, o.bytes))
            return PAELLA_EINVAL;
    if (overlap(tables_out, out * d->max_pages, past_out, out)) return PAELLA_EINVAL;
    ReorderArgs a;
    a.k_cache = (char*)c->k; a.v_cache = (char*)c->v;
    a.parents = parents; a.past = past; a.tables = tables; a.spare = spare; a.tables_out = tables_out; a.past_out = past_out;
    a.groups = d->groups; a.beams = d->beams; a.count = d->count; a.max_pages = d->max_pages;
    a.num_pages = c->num_pages; a.kv_heads = c->kv_heads; a.page_size = c->page_size; a.head_bytes = c->head_dim * element_bytes(c->dtype);
    a.job_id = job_id; a.notifier = (Notifier*)notifier;
    launch(beam_reorder_kernel, dim3((unsigned)(d->groups * d->count * c->kv_heads)), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

}  // extern "C"
