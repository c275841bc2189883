#pragma once
// Attention of a decoding step: every new token over a prefix that all sequences share and over its own sequence's tokens, both in a paged
// cache.  Included by one translation unit per element type (PAELLA_ATTENTION_TYPE), so that they compile side by side.
//
// out = sum_i p_i v_i / sum_i p_i with p_i = exp(scale * q . k_i - m): one pass over the keys with the running maximum m and sum, in 32 bits.
//
// Work.  A workgroup takes either a tile of up to 64 query rows (a row: a head of a new token; all heads that share a key head, of all
// sequences, side by side) over a part of the prefix, or the rows of one sequence over a part of its own tokens; its four waves take every
// fourth step of 32 (fp32: 16) keys each and put their sums together in LDS.  What the workgroups of a row leave is put together by the one
// that arrives last at the row (a counter per row), in the order of the parts, so results do not depend on who that is.
//
// Registers instead of LDS.  With v_mfma_*_16x16 and the products turned round (scores^T = K q^T, out^T = V^T p^T), every operand comes
// straight from memory or from the other product's result: lane l of a wave holds query row l % 16 throughout; lane group l / 16 gets the scores
// of exactly the keys whose probabilities it has to supply to the second product (the key that row m of score tile t stands for is
// m / 4 * TPL + 4 t + m % 4, TPL = 4 * tiles), and of V a lane loads TPL whole keys by 16 bytes, its group's keys by 16 lanes' dimensions: the 16-bit
// types need one byte permutation per operand register to put a dimension's keys side by side, fp32 none.  The output's dimensions are
// permuted by the same rule.  K and V are therefore read once per wave, in runs of 64 bytes and of whole keys, and both wait in registers for
// one step while the other product runs.

#include <hip/hip_runtime.h>

#include "decode_common.h"

namespace paella {

struct AttentionArgs {
    const char *q, *k_cache, *v_cache;
    char* out;
    const int *starts, *past, *tables, *prefix_table;
    int64_t q_stride;  // bytes
    int sequences, max_new, tokens, max_pages, prefix_len;
    int heads, kv_heads, per_kv, page_size, num_pages;
    unsigned page_blocks, page_blocks_inv;  // blocks of 8 tokens in a page, and 2^32 over that, rounded down
    float scale_log2;                       // scale * log2(e): probabilities are powers of two
    int prefix_tiles, prefix_splits, own_tiles, own_splits;
    unsigned prefix_items;
    unsigned* counters;  // [tokens * heads], zero between launches
    f32x2* ml;           // [splits][tokens * heads]: running maximum and sum of each part
    float* acc;          // [splits][tokens * heads][head_dim]
    uint32_t job_id;
    Notifier* notifier;
};

template <typename T> struct Mfma;
template <> struct Mfma<Bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 go(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
};
template <> struct Mfma<F16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 go(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
};
__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// What a walk over keys reads them through: the pages of a table, for one key head.
struct Keys {
    const int* table;
    int table_len;
    const char *k, *v;   // the cache, moved to the key head
    size_t page_bytes;
    unsigned page_blocks, page_blocks_inv, num_pages;
};

template <typename T, int D, int R>
struct AttentionTile {
    static constexpr bool F = T::bytes == 4;
    static constexpr int NT = F ? 1 : 2;              // score tiles of 16 keys per step
    static constexpr int TPL = 4 * NT;                // keys of a step that a lane group supplies to the second product
    static constexpr int STEP = 16 * NT;
    static constexpr int KC = D * T::bytes / 64;      // 16-byte pieces of a key row per lane
    static constexpr int PER = D / 16 * T::bytes < 16 ? D / 16 : 16 / T::bytes;  // neighbouring dimensions that a lane loads of V
    static constexpr int GRP = D / 16 / PER;
    static constexpr int VW = PER * T::bytes / 4;     // words of such a piece
    static constexpr int ROW = D * T::bytes;

    f32x4 acc[R][GRP * PER];
    float m[R], l[R];
    u32x4 q[R][KC];
    u32x4 k[NT][KC];
    unsigned v[TPL][GRP * VW];

    // page numbers of a lane's blocks of 8 keys in the step whose keys are loaded next, and the blocks' places in them
    int page_k, page_v;
    unsigned in_k, in_v;

    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
#pragma unroll
            for (int d = 0; d < GRP * PER; ++d) acc[r][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }

    __device__ __forceinline__ void load_q(int r, const char* row, int lane) {
#pragma unroll
        for (int c = 0; c < KC; ++c) q[r][c] = *reinterpret_cast<const u32x4*>(row + c * 64 + (lane >> 4) * 16);
    }

    // The pages of the step that begins at block b8 (of 8 keys); beyond the table a lane reads the last entry and is masked by the caller's limit.
    __device__ __forceinline__ void look_up(const Keys& s, unsigned b8, int lane) {
        constexpr int BLOCK_LANES_K = F ? 8 : 4;  // rows of the score tile that lie in one block
        const unsigned bk = b8 + (unsigned)(lane & 15) / BLOCK_LANES_K, bv = b8 + (unsigned)(lane >> 4) * TPL / 8;
        auto split = [&](unsigned b, unsigned& in) {
            unsigned page = __umulhi(b, s.page_blocks_inv);
            in = b - page * s.page_blocks;
            if (in >= s.page_blocks) {
                ++page;
                in -= s.page_blocks;
            }
            return min(page, (unsigned)s.table_len - 1);
        };
        const unsigned ik = split(bk, in_k), iv = split(bv, in_v);
        page_k = s.table[ik];
        page_v = s.table[iv];
    }

    __device__ __forceinline__ void load_k(const Keys& s, int lane) {
        const unsigned page = (unsigned)page_k < s.num_pages ? page_k : 0;
        const int mm = lane & 15;
        const unsigned slot = F ? in_k * 8 + (mm & 7) : in_k * 8 + (mm & 3);
        const char* p = s.k + page * s.page_bytes + (size_t)slot * ROW + (lane >> 4) * 16;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < KC; ++c) k[t][c] = *reinterpret_cast<const u32x4*>(p + t * 4 * ROW + c * 64);
    }

    __device__ __forceinline__ void load_v(const Keys& s, int lane) {
        const unsigned page = (unsigned)page_v < s.num_pages ? page_v : 0;
        const unsigned slot = in_v * 8 + (F ? (lane >> 4 & 1) * 4 : 0);
        const char* p = s.v + page * s.page_bytes + (size_t)slot * ROW + (lane & 15) * PER * T::bytes;
#pragma unroll
        for (int u = 0; u < TPL; ++u)
#pragma unroll
            for (int g = 0; g < GRP; ++g) {
                const char* at = p + u * ROW + g * 16 * PER * T::bytes;
                if constexpr (VW == 4) {
                    const u32x4 w = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[u][g * 4 + e] = w[e];
                } else {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(at);
                    v[u][g * 2] = w.x;
                    v[u][g * 2 + 1] = w.y;
                }
            }
    }

    // One step over the keys from `first` on, of which row r sees those below limit[r]; `least` and `most` bound the limits of all rows, `absent`: this
    // lane group's keys are in no page.  next(true) is called once K is no longer needed, next(false) once V is.
    template <typename Next>
    __device__ __forceinline__ void step(int first, const bool absent, const int (&limit)[R], int least, int most, float scale, int lane, Next next) {
        f32x4 x[R][NT];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < NT; ++t) x[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if constexpr (F) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int r = 0; r < R; ++r) x[r][t] = mfma_f32(as_float(k[t][c][e]), as_float(q[r][c][e]), x[r][t]);
                } else {
#pragma unroll
                    for (int r = 0; r < R; ++r) x[r][t] = Mfma<T>::go(k[t][c], q[r][c], x[r][t]);
                }
            }
        next(true);
        if (first + STEP > least || __any(absent)) {
            const int mine = first + (lane >> 4) * TPL;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (absent || mine + t * 4 + e >= limit[r]) x[r][t][e] = -INFINITY;
            // what lies in places that no row may see can be anything, and 0 * NaN is NaN
#pragma unroll
            for (int u = 0; u < TPL; ++u)
                if (absent || mine + u >= most) {
#pragma unroll
                    for (int w = 0; w < GRP * VW; ++w) v[u][w] = 0;
                }
        }
        // The running maximum moves only when a score is above it by a factor of 2^8: until then probabilities are at most 256 (their sums stay in
        // 32 bits, and 16-bit ones keep their relative precision), and neither the lanes' exchange nor the rescaling is needed.
        bool grown = false;
        float top[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            top[r] = x[r][0][0];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) top[r] = fmaxf(top[r], x[r][t][e]);
            top[r] *= scale;
            grown |= top[r] > m[r] + 8.f;
        }
        if (__any(grown)) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float now = fmaxf(top[r], m[r]);
                now = fmaxf(now, __shfl_xor(now, 16, 64));
                now = fmaxf(now, __shfl_xor(now, 32, 64));
                const float shrink = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - now);
                m[r] = now;
                l[r] *= shrink;
#pragma unroll
                for (int d = 0; d < GRP * PER; ++d) acc[r][d] *= shrink;
            }
        }
        unsigned p[R][4];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float base = m[r] == -INFINITY ? 0.f : m[r];
            float y[TPL];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) y[t * 4 + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r][t][e], scale, -base));
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < TPL; ++e) sum += y[e];
            l[r] += sum;
            if constexpr (F) {
#pragma unroll
                for (int e = 0; e < 4; ++e) p[r][e] = as_word(y[e]);
            } else {  // probabilities to the products' type: half a step of relative error each, as much as the values they weigh have
#pragma unroll
                for (int e = 0; e < 4; ++e) p[r][e] = pack2<T>(y[2 * e], y[2 * e + 1]);
            }
        }
#pragma unroll
        for (int d = 0; d < GRP * PER; ++d) {
            if constexpr (F) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int r = 0; r < R; ++r) acc[r][d] = mfma_f32(as_float(v[e][d]), as_float(p[r][e]), acc[r][d]);
            } else {
                u32x4 a;
                const int w = d / 2;
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] = __builtin_amdgcn_perm(v[2 * e + 1][w], v[2 * e][w], d & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int r = 0; r < R; ++r) acc[r][d] = Mfma<T>::go(a, u32x4{p[r][0], p[r][1], p[r][2], p[r][3]}, acc[r][d]);
            }
        }
        next(false);
    }

    // Steps `at`, at + 4, ... below `end` (in steps of the table's keys).  Page numbers are asked for a step ahead of the keys.
    __device__ __forceinline__ void walk(const Keys& s, int at, int end, const int (&limit)[R], int least, int most, float scale, int lane) {
        if (at >= end) return;
        look_up(s, (unsigned)at * (STEP / 8), lane);
        load_k(s, lane);
        load_v(s, lane);
        bool absent = (unsigned)page_v >= s.num_pages;
        look_up(s, (unsigned)(at + 4) * (STEP / 8), lane);
        for (; at + 4 < end; at += 4) {
            step(at * STEP, absent, limit, least, most, scale, lane, [&](bool k_is_free) {
                if (k_is_free) {
                    load_k(s, lane);
                } else {
                    load_v(s, lane);
                    absent = (unsigned)page_v >= s.num_pages;
                    look_up(s, (unsigned)(at + 8) * (STEP / 8), lane);
                }
            });
        }
        step(at * STEP, absent, limit, least, most, scale, lane, [](bool) {});
    }
};

// One 16-byte (8-byte) piece of four outputs.
template <typename T>
__device__ __forceinline__ void put_out(__amdgpu_buffer_rsrc_t to, unsigned value_at, f32x4 v) {
    if constexpr (T::bytes == 4) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), to, (int)(value_at * 4), 0, kThrough);
    } else {
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{pack2<T>(v.x, v.y), pack2<T>(v.z, v.w)}, to, (int)(value_at * 2), 0, kThrough);
    }
}

// A workgroup's part: rows `row_id` (LDS; -1: none) of its tile over steps [begin, end) of `s`, left in slot `part` (or, where there is one, as the output).
template <typename T, int D, int R>
__device__ __forceinline__ void attend(const AttentionArgs& a, const Keys& s, const char* const (&q_row)[R], const int (&limit)[R], int least, int most, int begin,
                                       int end, int part, const int* row_id, char* lds) {
    using Tile = AttentionTile<T, D, R>;
    constexpr int PITCH = D + 4;  // floats of a row in LDS: lanes of different rows on different banks
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    f32x2* const ml = reinterpret_cast<f32x2*>(lds);                   // [4][16 R]
    float* const sums = reinterpret_cast<float*>(lds + 4 * 16 * R * 8);  // [4][16 R][PITCH]
    {
        Tile tile;
        tile.begin();
#pragma unroll
        for (int r = 0; r < R; ++r) tile.load_q(r, q_row[r], lane);
        tile.walk(s, begin + wave, end, limit, least, most, a.scale_log2, lane);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float l = tile.l[r];
            l += __shfl_xor(l, 16, 64);
            l += __shfl_xor(l, 32, 64);
            if (lane < 16) ml[wave * 16 * R + r * 16 + lane] = f32x2{tile.m[r], l};
            float* const to = sums + (wave * 16 * R + r * 16 + (lane & 15)) * PITCH;
#pragma unroll
            for (int g = 0; g < Tile::GRP; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < Tile::PER; e += 4) {
                        const int d = g * Tile::PER + e;
                        *reinterpret_cast<f32x4*>(to + g * 16 * Tile::PER + ((lane >> 4) * 4 + i) * Tile::PER + e) =
                            f32x4{tile.acc[r][d][i], tile.acc[r][d + 1][i], tile.acc[r][d + 2][i], tile.acc[r][d + 3][i]};
                    }
        }
    }
    __syncthreads();
    const size_t rows = (size_t)a.tokens * a.heads;
    const bool whole = a.counters == nullptr;
    const __amdgpu_buffer_rsrc_t to = whole ? descriptor(a.out) : descriptor(a.acc + (size_t)part * rows * D);
    const __amdgpu_buffer_rsrc_t to_ml = descriptor(a.ml + (size_t)part * (whole ? 0 : rows));
    for (int e = threadIdx.x; e < 16 * R * (D / 4); e += 256) {
        const int row = e / (D / 4), d = (e - row * (D / 4)) * 4;
        const int id = row_id[row];
        if (id < 0) continue;
        float top = -INFINITY;
        f32x2 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = ml[i * 16 * R + row];
            top = fmaxf(top, w[i].x);
        }
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
        if (top > -INFINITY) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = __builtin_amdgcn_exp2f(w[i].x - top);
                l += w[i].y * f;
                sum += *reinterpret_cast<const f32x4*>(sums + (i * 16 * R + row) * PITCH + d) * f;
            }
        }
        if (whole) {
            put_out<T>(to, (unsigned)id * D + d, l > 0.f ? sum / l : f32x4{0.f, 0.f, 0.f, 0.f});
        } else {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sum), to, (int)(((unsigned)id * D + d) * 4), 0, kThrough);
            if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(u32x2{as_word(top), as_word(l)}, to_ml, id * 8, 0, kThrough);
        }
    }
}

// Counts the workgroup in at each of its rows and puts together the rows at which it is the last.  (As in the convs' split reductions: parts
// are written through ahead of the count, and read past this workgroup's caches.)
template <typename T, int D>
__device__ __forceinline__ void join(const AttentionArgs& a, const int* row_id, int rows_here, int* done) {
    const int lane = threadIdx.x & 63;
    const int parts = a.prefix_splits + a.own_splits;
    __shared__ int count;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x < 64) {
        const int id = lane < rows_here ? row_id[lane] : -1;
        bool last = false;
        if (id >= 0) {
            last = __hip_atomic_fetch_add(a.counters + id, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)parts - 1;
            if (last) __hip_atomic_store(a.counters + id, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        const unsigned long long who = __ballot(last);
        if (last) done[__popcll(who & ((1ull << lane) - 1))] = id;
        if (lane == 0) count = __popcll(who);
    }
    __syncthreads();
    const int n = count;
    const size_t rows = (size_t)a.tokens * a.heads;
    const __amdgpu_buffer_rsrc_t to = descriptor(a.out);
    for (int e = threadIdx.x; e < n * (D / 4); e += 256) {
        const int row = e / (D / 4), d = (e - row * (D / 4)) * 4;
        const int id = done[row];
        float top = -INFINITY, l = 0.f;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int first = 0; first < parts; first += 8) {
            constexpr int N = 8;  // parts that are requested together
            u32x2 w[N];
            u32x4 x[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int part = min(first + i, parts - 1);
                w[i] = __builtin_amdgcn_raw_buffer_load_b64(descriptor(a.ml + part * rows), id * 8, 0, kThrough);
                x[i] = __builtin_amdgcn_raw_buffer_load_b128(descriptor(a.acc + part * rows * D), (int)(((unsigned)id * D + d) * 4), 0, kThrough);
            }
            float now = top;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (first + i < parts) now = fmaxf(now, as_float(w[i].x));
            if (now == -INFINITY) continue;
            const float shrink = __builtin_amdgcn_exp2f(top - now);
            sum *= shrink;
            l *= shrink;
            top = now;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (first + i >= parts) continue;
                const float f = __builtin_amdgcn_exp2f(as_float(w[i].x) - top);
                l += as_float(w[i].y) * f;
                sum += __builtin_bit_cast(f32x4, x[i]) * f;
            }
        }
        put_out<T>(to, (unsigned)id * D + d, l > 0.f ? sum / l : f32x4{0.f, 0.f, 0.f, 0.f});
    }
}

template <int D, int R>
constexpr int attention_lds() { return 4 * 16 * R * 8 + 4 * 16 * R * (D + 4) * 4; }

// RP, RO: 16-row tiles of a workgroup over the prefix / over a sequence's own tokens.
template <typename T, int D, int RP, int RO>
__global__ __launch_bounds__(256, 1) void prefix_attention_kernel(AttentionArgs a) {
    hook_entry(a.notifier, a.job_id);
    constexpr int RM = RP > RO ? RP : RO;
    __shared__ __attribute__((aligned(16))) char lds[attention_lds<D, RM>()];
    __shared__ int row_id[16 * RM], done[16 * RM];
    constexpr int STEP = AttentionTile<T, D, 1>::STEP;
    const int lane = threadIdx.x & 63;
    const int head_bytes = D * T::bytes;
    Keys s;
    s.page_bytes = (size_t)a.kv_heads * a.page_size * head_bytes;
    s.page_blocks = a.page_blocks;
    s.page_blocks_inv = a.page_blocks_inv;
    s.num_pages = (unsigned)a.num_pages;
    unsigned item = blockIdx.x;
    bool any = false;
    if (item < a.prefix_items) {
        // (key head, split) by tile: the tiles of one pair read the same keys, so they follow each other by 8 and share an XCD's cache
        const unsigned pairs = (unsigned)(a.kv_heads * a.prefix_splits), tiles = (unsigned)a.prefix_tiles;
        const unsigned eights = pairs / 8 * 8 * tiles;
        unsigned pair, tile;
        if (item < eights) {
            pair = item / (8 * tiles) * 8 + item % 8;
            tile = item % (8 * tiles) / 8;
        } else {
            const unsigned left = pairs % 8, i = item - eights;
            pair = pairs / 8 * 8 + i % left;
            tile = i / left;
        }
        const int h = (int)(pair / a.prefix_splits), split = (int)(pair % a.prefix_splits);
        const int group_rows = a.tokens * a.per_kv;
        const char* q_row[RP];
        int limit[RP];
#pragma unroll
        for (int r = 0; r < RP; ++r) {
            const int x = min((int)tile * 16 * RP + r * 16 + (lane & 15), group_rows - 1);
            const int t = x / a.per_kv;
            q_row[r] = a.q + t * a.q_stride + (h * a.per_kv + x - t * a.per_kv) * head_bytes;
            limit[r] = a.prefix_len;
        }
        // rows that belong to no sequence are left out; each of them by a wave of its own where the batch is ragged
        for (int r = (int)(threadIdx.x >> 6); r < 16 * RP; r += 4) {
            const int x = (int)tile * 16 * RP + r, t = x / a.per_kv;
            int seq, j;
            const bool owned = x < group_rows && row_owner(a.starts, a.sequences, a.max_new, t, lane, &seq, &j);
            if (lane == 0) row_id[r] = owned ? t * a.heads + h * a.per_kv + x - t * a.per_kv : -1;
        }
        __syncthreads();
        s.table = a.prefix_table;
        s.table_len = (a.prefix_len + a.page_size - 1) / a.page_size;
        s.k = a.k_cache + (size_t)h * a.page_size * head_bytes;
        s.v = a.v_cache + (size_t)h * a.page_size * head_bytes;
        const int steps = (a.prefix_len + STEP - 1) / STEP;
        const int per = (steps + a.prefix_splits - 1) / a.prefix_splits;
        const int begin = min(split * per, steps), end = min(begin + per, steps);
        attend<T, D, RP>(a, s, q_row, limit, a.prefix_len, a.prefix_len, begin, end, split, row_id, lds);
        any = true;
    } else {
        item -= a.prefix_items;
        // the key heads of one sequence side by side: they share the look-ups and, with eight of them, an XCD each
        const int h = (int)(item % a.kv_heads);
        item /= (unsigned)a.kv_heads;
        const int split = (int)(item % a.own_splits);
        item /= (unsigned)a.own_splits;
        const int tile = (int)(item % a.own_tiles), seq = (int)(item / a.own_tiles);
        int first = seq * a.max_new, count = a.max_new;
        if (a.starts) {
            first = min(max(__builtin_amdgcn_readfirstlane(a.starts[seq]), 0), a.tokens);
            count = min(min(__builtin_amdgcn_readfirstlane(a.starts[seq + 1]), a.tokens) - first, a.max_new);
        }
        const int group_rows = max(count, 0) * a.per_kv;
        any = tile * 16 * RO < group_rows;
        if (any) {
            const int capacity = (int)min((int64_t)a.max_pages * a.page_size, (int64_t)1 << 30);
            const int past = min(max(__builtin_amdgcn_readfirstlane(a.past[seq]), 0), capacity);
            const char* q_row[RO];
            int limit[RO];
#pragma unroll
            for (int r = 0; r < RO; ++r) {
                const int x = tile * 16 * RO + r * 16 + (lane & 15);
                const int y = min(x, group_rows - 1), j = y / a.per_kv, t = first + j;
                const int head = h * a.per_kv + y - j * a.per_kv;
                q_row[r] = a.q + t * a.q_stride + head * head_bytes;
                limit[r] = min(past + j + 1, capacity);
                if (threadIdx.x < 16) row_id[r * 16 + lane] = x < group_rows ? t * a.heads + head : -1;
            }
            __syncthreads();
            s.table = a.tables + (size_t)seq * a.max_pages;
            s.table_len = a.max_pages;
            s.k = a.k_cache + (size_t)h * a.page_size * head_bytes;
            s.v = a.v_cache + (size_t)h * a.page_size * head_bytes;
            const int least = min(past + tile * 16 * RO / a.per_kv + 1, capacity);
            const int most = min(past + min(tile * 16 * RO + 16 * RO - 1, group_rows - 1) / a.per_kv + 1, capacity);
            const int steps = (most + STEP - 1) / STEP;
            const int per = (steps + a.own_splits - 1) / a.own_splits;
            const int begin = min(split * per, steps), end = min(begin + per, steps);
            attend<T, D, RO>(a, s, q_row, limit, least, most, begin, end, a.prefix_splits + split, row_id, lds);
        }
    }
    if (any && a.counters) join<T, D>(a, row_id, blockIdx.x < a.prefix_items ? 16 * RP : 16 * RO, done);
    hook_exit(a.notifier, a.job_id);
}

using AttentionKernel = void (*)(AttentionArgs);

template <typename T, int D>
AttentionKernel attention_kernel_of(int rp, int ro) {
    if (rp == 1 && ro == 1) return prefix_attention_kernel<T, D, 1, 1>;
    if constexpr (D * T::bytes <= 512 && D <= 128) {
        if (rp == 2 && ro == 1) return prefix_attention_kernel<T, D, 2, 1>;
        if (rp == 2 && ro == 2) return prefix_attention_kernel<T, D, 2, 2>;
    }
    if constexpr (D * T::bytes <= 256) {
        if (rp == 4 && ro == 1) return prefix_attention_kernel<T, D, 4, 1>;
        if (rp == 4 && ro == 2) return prefix_attention_kernel<T, D, 4, 2>;
        if (rp == 4 && ro == 4) return prefix_attention_kernel<T, D, 4, 4>;
    }
    return nullptr;
}

template <typename T>
AttentionKernel attention_kernel(int dim, int rp, int ro) {
    return dim == 64 ? attention_kernel_of<T, 64>(rp, ro) : dim == 128 ? attention_kernel_of<T, 128>(rp, ro) : dim == 256 ? attention_kernel_of<T, 256>(rp, ro) : nullptr;
}

// The kernel of a type for a head size and numbers of 16-row tiles; nullptr where there is none.  Defined once per type.
AttentionKernel attention_kernel_f32(int dim, int rp, int ro);
AttentionKernel attention_kernel_bf16(int dim, int rp, int ro);
AttentionKernel attention_kernel_f16(int dim, int rp, int ro);

}  // namespace paella
