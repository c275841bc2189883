#pragma once
// Attention of a decoding step: every new token over a prefix that all sequences share and over its own sequence's tokens, both in a paged
// cache.  Included by one translation unit per element type, so that they compile side by side.
//
// out = sum_i p_i v_i / sum_i p_i with p_i = exp(scale * q . k_i - m): one pass over the keys with the running maximum m and sum, in 32 bits.
//
// Work.  A workgroup takes either a tile of query rows (a row: a head of a new token; all heads that share a key head, of all sequences, side by
// side) over a part of the prefix, or rows of one sequence over a part of its own tokens.  Few rows, or few keys: 16 rows, all four waves have them, each takes every
// fourth step of 32 (fp32: 16) keys, and their sums are put together in LDS.  Else each wave has 16 or 32 rows of its own, and the workgroup
// brings the keys to LDS for all of them.  What the workgroups of a row leave is put together by the one that arrives last at the row (a
// counter per row) or by a launch of its own, in the order of the parts, so results do not depend on who that is.
//
// Operands.  With v_mfma_*_16x16 and the products turned round (scores^T = K q^T, out^T = V^T p^T), every operand comes
// as it lies in the cache or from the other product's result: lane l of a wave holds query row l % 16 throughout; lane group l / 16 gets the scores
// of exactly the keys whose probabilities it has to supply to the second product (the key that row m of score tile t stands for is
// m / 4 * TPL + 4 t + m % 4, TPL = 4 * tiles), and of V a lane loads TPL whole keys by 16 bytes, its group's keys by 16 lanes' dimensions: the 16-bit
// types need one byte permutation per operand register to put a dimension's keys side by side, fp32 none.  The output's dimensions are
// permuted by the same rule.  Where the waves split the keys, K and V are therefore read once, in runs of 64 bytes and of whole keys, and wait in registers for
// one step while the other product runs.
//
// Bounds.  Few rows: the trips to memory in a row (length, page, keys, parts, count, parts), 7.7 us for 3 rows a head over 333 keys in fp32, 8.1 for 8 over 2011 in
// fp16.  Own tokens of many sequences: memory, 1.05 GB at 5.6 TB/s (a plain read of this size 6.2).  The prefix of 32 rows and more per
// key head: the matrix and vector units, which take turns; per 32 x 32 scores 34 matrix instructions of 16 cycles and some 90 vector ones of 4, 16 of
// them exponentials of 16; 69 GFLOP in 90 us at the 1.9 GHz that the power limit leaves.  Both at once, 64 sequences over 65536 shared and 2000 own keys on average
// (802 MB, 71 GFLOP): 162 us and the joining launch's 7 when the card is cool, 195 under load without a pause.

#include <hip/hip_runtime.h>

#include "decode_common.h"

namespace paella {

struct AttentionArgs {
    const char *q, *k_cache, *v_cache;
    char* out;
    const int *starts, *past, *tables, *prefix_table;
    int64_t q_stride;  // bytes
    int sequences, max_new, tokens, max_pages, prefix_len, prefix_pages;
    int heads, page_size, num_pages;
    Divisor kv_heads, per_kv, page_blocks;  // per_kv: query heads of a key head; page_blocks: blocks of 8 tokens in a page
    float scale_log2;                       // scale * log2(e): probabilities are powers of two
    Divisor eight_tiles, prefix_splits, own_tiles, own_splits;  // eight_tiles: 8 times the tiles over the prefix
    int prefix_per, prefix_pairs;                               // steps of a split; key heads by splits
    unsigned prefix_items;
    unsigned* counters;     // [key heads][rows of one, in whole cache lines], zero between launches; null where a launch of its own joins.  A workgroup's lie side by
                            // side, and other key heads' on other lines: counts on one line go one after the other
    unsigned counter_pitch;
    f32x2* ml;           // [splits][tokens * heads]: running maximum and sum of each part
    float* acc;          // [splits][tokens * heads][head_dim]
    uint32_t job_id;
    Notifier* notifier;
};

constexpr int kJoined = 16;     // parts of a row that the workgroup that joins it requests together
constexpr int kJoinRows = 256;  // outputs of a workgroup of the joining launch

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
    Divisor page_blocks;  // a block: 8 keys, which never lie in two pages
    unsigned num_pages;

    struct Place {
        unsigned entry, in;  // of the table, and the block's place in the page
    };
    // Where block b lies; beyond the table's end in the last entry (the caller's limits mask what is read).
    __device__ __forceinline__ Place place_of(unsigned b) const {
        const Quotient at = divide(b, page_blocks);
        return {min(at.q, (unsigned)table_len - 1), at.r};
    }
    __device__ __forceinline__ size_t page_at(int page) const { return ((unsigned)page < num_pages ? (unsigned)page : 0u) * page_bytes; }
};

// 16 R query rows of a wave: what they have summed so far.  Lane l holds row l % 16 of each 16.  STRAIGHT: V comes with its dimensions in order, 16 to a
// product, else by pieces of PER of them.
template <typename T, int D, int R, bool STRAIGHT>
struct AttentionRows {
    static constexpr bool F = T::bytes == 4;
    static constexpr int NT = F ? 1 : 2;              // score tiles of 16 keys per step
    static constexpr int TPL = 4 * NT;                // keys of a step that a lane group supplies to the second product
    static constexpr int STEP = 16 * NT;
    static constexpr int ROW = D * T::bytes;          // bytes of a key
    static constexpr int KC = ROW / 64;               // 16-byte pieces of a key per lane
    static constexpr int PER = D / 16 * T::bytes < 16 ? D / 16 : 16 / T::bytes;  // neighbouring dimensions that a lane has of V
    static constexpr int GRP = D / 16 / PER;
    static constexpr int VW = PER * T::bytes / 4;     // words of such a piece
    // Probabilities are taken relative to 2^m, m = the running maximum's exponent less BELOW, and m moves only for a score that is above it by more than BELOW +
    // SLACK.  fp16 has few exponents: weights lose bits under 2^-14 and are gone under 2^-25, and beside one key that has nearly all of the weight tens of thousands of
    // small ones still count (with the maximum at 2^0, keys at e^-16 of the largest came to 0.4 % too little, at e^-17 to 3 %).  2^15 above m (2^16 is infinite) leave all bits to
    // weights down to 2^-25 of the largest, and what is lost below that is at most 2^-36 of it each.  Of these 15, 4 for the maximum's moves cost no time, 2 would: 40.6 us
    // against 39.4 for 32 sequences of up to 5 tokens over 8190 + 1000 keys.  fp32 and bf16 have exponents enough for any.
    // Where scores are so large that they are in steps of a half and more, m and the exponentials' arguments are off by as much, and 2^8 is what fp16 has room for as well.
    static constexpr float BELOW = __is_same(T, F16) ? 11.f : 0.f, SLACK = __is_same(T, F16) ? 4.f : 8.f;
    static constexpr float LARGE = 4194304.f;  // 2^22
    static __device__ __forceinline__ float base_of(float top) { return __is_same(T, F16) && !(fabsf(top) < LARGE) ? top : top - BELOW; }
    static __device__ __forceinline__ float rise_of(float base) { return base + (__is_same(T, F16) && !(fabsf(base) < LARGE) ? 8.f : BELOW + SLACK); }

    f32x4 acc[R][GRP * PER];
    f32x4 total[R];  // sums of the probabilities; 16-bit types: of the rounded ones, so that what the rounding does to a row's largest weights cancels
    float m[R];
    float rise[R];   // the score above which m moves
    u32x4 q[R][KC];

    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            m[r] = rise[r] = -INFINITY;
            total[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < GRP * PER; ++d) acc[r][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }

    __device__ __forceinline__ void load_q(int r, const char* row, int lane) {
#pragma unroll
        for (int c = 0; c < KC; ++c) q[r][c] = *reinterpret_cast<const u32x4*>(row + c * 64 + (lane >> 4) * 16);
    }

    // x = K q^T of a step's keys; k(t, c): the lane's piece c of its key of score tile t
    template <typename K>
    __device__ __forceinline__ void scores(f32x4 (&x)[R][NT], K k) const {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < NT; ++t) x[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const u32x4 piece = k(t, c);
                if constexpr (F) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int r = 0; r < R; ++r) x[r][t] = mfma_f32(as_float(piece[e]), as_float(q[r][c][e]), x[r][t]);
                } else {
#pragma unroll
                    for (int r = 0; r < R; ++r) x[r][t] = Mfma<T>::go(piece, q[r][c], x[r][t]);
                }
            }
    }

    // Row r sees the keys below limit[r]; `first`: of the lane group's keys; absent: they are in no page
    __device__ __forceinline__ static void mask(f32x4 (&x)[R][NT], int first, bool absent, const int (&limit)[R]) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (absent || first + t * 4 + e >= limit[r]) x[r][t][e] = -INFINITY;
    }

    // Scores to probabilities, as operands of the second product: each the sum of PARTS numbers of its type.
    template <int PARTS>
    __device__ __forceinline__ void weigh(const f32x4 (&x)[R][NT], float scale, unsigned (&p)[PARTS][R][4]) {
        // Until a score is above the running maximum by 2^SLACK, neither the lanes' exchange nor the rescaling is needed.
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
            grown |= top[r] > rise[r];
        }
        if (__any(grown)) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float now = fmaxf(base_of(top[r]), m[r]);
                now = fmaxf(now, __shfl_xor(now, 16, 64));
                now = fmaxf(now, __shfl_xor(now, 32, 64));
                const float shrink = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - now);
                m[r] = now;
                rise[r] = rise_of(now);
                total[r] *= shrink;
#pragma unroll
                for (int d = 0; d < GRP * PER; ++d) acc[r][d] *= shrink;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float base = m[r] == -INFINITY ? 0.f : m[r];
            float y[TPL];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) y[t * 4 + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r][t][e], scale, -base));
            if constexpr (F) {
                static_assert(PARTS == 1);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[0][r][e] = as_word(y[e]);
                    total[r][0] += y[e];
                }
            } else {
                // Probabilities to the products' type, since both of a product's operands have one: half a step of relative error each (a weight that BELOW has not kept from
                // fp16's subnormals: half of their step), as much as the values they weigh have.  A second part has what the first leaves, and leaves half a step of half a step.
                constexpr unsigned one = __is_same(T, Bf16) ? 0x3F803F80u : 0x3C003C00u;
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p[part][r][e] = pack2<T>(y[2 * e], y[2 * e + 1]);
                        if (part + 1 < PARTS) {
                            const f32x2 had = unpack2<T>(p[part][r][e]);
                            y[2 * e] -= had.x;
                            y[2 * e + 1] -= had.y;
                        }
                    }
                    total[r] = Mfma<T>::go(u32x4{one, one, one, one}, u32x4{p[part][r][0], p[part][r][1], p[part][r][2], p[part][r][3]}, total[r]);  // every row of it the same sum
                }
            }
        }
    }

    // out += V^T p; v: the lane group's keys, PER dimensions of each in every group of 16 PER
    template <int PARTS>
    __device__ __forceinline__ void add_values(const unsigned (&v)[TPL][GRP * VW], const unsigned (&p)[PARTS][R][4]) {
#pragma unroll
        for (int d = 0; d < GRP * PER; ++d) {
            if constexpr (F) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int r = 0; r < R; ++r) acc[r][d] = mfma_f32(as_float(v[e][d]), as_float(p[0][r][e]), acc[r][d]);
            } else {
                u32x4 a;
                const int w = d / 2;
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] = __builtin_amdgcn_perm(v[2 * e + 1][w], v[2 * e][w], d & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int part = 0; part < PARTS; ++part)
#pragma unroll
                    for (int r = 0; r < R; ++r) acc[r][d] = Mfma<T>::go(a, u32x4{p[part][r][0], p[part][r][1], p[part][r][2], p[part][r][3]}, acc[r][d]);
            }
        }
    }

    // The same from V as the transposing reads of LDS bring it: v[d], dimensions 16 d on of the lane group's keys.
    __device__ __forceinline__ void add_straight(const u32x4 (&v)[D / 16], const unsigned (&p)[R][4]) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r][d] = Mfma<T>::go(v[d], u32x4{p[r][0], p[r][1], p[r][2], p[r][3]}, acc[r][d]);
    }

    __device__ __forceinline__ float sum_of(int r) const {
        float l = total[r][0];
        if constexpr (F) {  // the lane groups' parts
            l += __shfl_xor(l, 16, 64);
            l += __shfl_xor(l, 32, 64);
        }
        return l;
    }

    // Sums to a row of LDS (`to`: of the lane's row in 16 r), dimensions in order.
    __device__ __forceinline__ void put_sums(int r, float* to, int lane) const {
        if constexpr (STRAIGHT) {
#pragma unroll
            for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f32x4*>(to + d * 16 + (lane >> 4) * 4) = acc[r][d];
        } else {
#pragma unroll
            for (int g = 0; g < GRP; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < PER; e += 4) {
                        const int d = g * PER + e;
                        *reinterpret_cast<f32x4*>(to + g * 16 * PER + ((lane >> 4) * 4 + i) * PER + e) = f32x4{acc[r][d][i], acc[r][d + 1][i], acc[r][d + 2][i], acc[r][d + 3][i]};
                    }
        }
    }
};

// Few rows: a wave has all 16 of the workgroup's rows and every fourth step of its keys, which come straight from memory into registers.
template <typename T, int D>
struct NarrowWalk {
    using Rows = AttentionRows<T, D, 1, false>;
    static constexpr bool F = Rows::F;
    static constexpr int ROW = Rows::ROW, TPL = Rows::TPL, STEP = Rows::STEP;

    u32x4 k[Rows::NT][Rows::KC];
    unsigned v[TPL][Rows::GRP * Rows::VW];
    int page_k, page_v;   // of the step whose keys are loaded next, for the lane's keys of K and of V
    unsigned in_k, in_v;  // the blocks' places in the pages

    __device__ __forceinline__ void look_up(const Keys& s, unsigned b8, bool even, int lane) {
        if (even) {  // a step lies in one page: one look-up for all
            const Keys::Place at = s.place_of(__builtin_amdgcn_readfirstlane(b8));
            page_k = page_v = s.table[at.entry];
            in_k = in_v = at.in;
        } else {
            constexpr int BLOCK_LANES_K = F ? 8 : 4;  // rows of the score tile that lie in one block
            const Keys::Place at_k = s.place_of(b8 + (unsigned)(lane & 15) / BLOCK_LANES_K), at_v = s.place_of(b8 + (unsigned)(lane >> 4) * TPL / 8);
            page_k = s.table[at_k.entry];
            page_v = s.table[at_v.entry];
            in_k = at_k.in;
            in_v = at_v.in;
        }
    }

    __device__ __forceinline__ void load_k(const Keys& s, bool even, int lane) {
        const int mm = lane & 15;
        // the key of row mm of score tile 0: mm / 4 * TPL + mm % 4, the blocks before its own among them where one page holds the step
        const unsigned own = F ? (even ? mm : mm & 7) : (even ? (mm >> 2) * 8 + (mm & 3) : mm & 3);
        const char* p;
        if (even) p = s.k + s.page_at(__builtin_amdgcn_readfirstlane(page_k)) + __builtin_amdgcn_readfirstlane(in_k) * 8 * ROW + (own * ROW + (lane >> 4) * 16);
        else p = s.k + s.page_at(page_k) + (size_t)((in_k * 8 + own) * ROW + (lane >> 4) * 16);
#pragma unroll
        for (int t = 0; t < Rows::NT; ++t)
#pragma unroll
            for (int c = 0; c < Rows::KC; ++c) k[t][c] = *reinterpret_cast<const u32x4*>(p + t * 4 * ROW + c * 64);
    }

    __device__ __forceinline__ void load_v(const Keys& s, bool even, int lane) {
        const unsigned own = F ? (even ? (lane >> 4) * 4 : (lane >> 4 & 1) * 4) : (even ? (lane >> 4) * 8 : 0);
        const unsigned at = own * ROW + (lane & 15) * Rows::PER * T::bytes;
        const char* p;
        if (even) p = s.v + s.page_at(__builtin_amdgcn_readfirstlane(page_v)) + __builtin_amdgcn_readfirstlane(in_v) * 8 * ROW + at;
        else p = s.v + s.page_at(page_v) + (size_t)(in_v * 8 * ROW + at);
#pragma unroll
        for (int u = 0; u < TPL; ++u)
#pragma unroll
            for (int g = 0; g < Rows::GRP; ++g) {
                const char* from = p + u * ROW + g * 16 * Rows::PER * T::bytes;
                if constexpr (Rows::VW == 4) {
                    const u32x4 w = *reinterpret_cast<const u32x4*>(from);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[u][g * 4 + e] = w[e];
                } else {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(from);
                    v[u][g * 2] = w.x;
                    v[u][g * 2 + 1] = w.y;
                }
            }
    }

    // One step over the keys from `first` on.  `least` and `most` bound the limits of all rows, absent: this lane group's keys are in no page.
    // next(true) is called once K is no longer needed, next(false) once V is.
    template <typename Next>
    __device__ __forceinline__ void step(Rows& rows, int first, const bool absent, const int (&limit)[1], int least, int most, float scale, int lane, Next next) {
        f32x4 x[1][Rows::NT];
        rows.scores(x, [&](int t, int c) { return k[t][c]; });
        next(true);
        if (first + STEP > least || __any(absent)) {
            const int mine = first + (lane >> 4) * TPL;
            Rows::mask(x, mine, absent, limit);
            // what lies in places that no row may see can be anything, and 0 * NaN is NaN
#pragma unroll
            for (int u = 0; u < TPL; ++u)
                if (absent || mine + u >= most) {
#pragma unroll
                    for (int w = 0; w < Rows::GRP * Rows::VW; ++w) v[u][w] = 0;
                }
        }
        unsigned p[1][1][4];
        rows.weigh(x, scale, p);
        rows.add_values(v, p);
        next(false);
    }

    // Steps `at`, at + 4, ... below `end`.  Page numbers are asked for a step ahead of the keys.
    __device__ __forceinline__ void walk(Rows& rows, const Keys& s, int at, int end, const int (&limit)[1], int least, int most, float scale, int lane) {
        if (at >= end) return;
        const bool even = s.page_blocks.d % (STEP / 8) == 0;
        look_up(s, (unsigned)at * (STEP / 8), even, lane);
        load_k(s, even, lane);
        load_v(s, even, lane);
        bool absent = (unsigned)page_v >= s.num_pages;
        look_up(s, (unsigned)(at + 4) * (STEP / 8), even, lane);
        for (; at + 4 < end; at += 4) {
            step(rows, at * STEP, absent, limit, least, most, scale, lane, [&](bool k_is_free) {
                if (k_is_free) {
                    load_k(s, even, lane);
                } else {
                    load_v(s, even, lane);
                    absent = (unsigned)page_v >= s.num_pages;
                    look_up(s, (unsigned)(at + 8) * (STEP / 8), even, lane);
                }
            });
        }
        step(rows, at * STEP, absent, limit, least, most, scale, lane, [](bool) {});
    }
};

// Loads of memory into LDS without a register between, in the order of the lanes: 16 bytes (4) of `base` + each lane's offset, from `lds` on.  What has arrived is
// told by arrived(n): all but the wave's last n loads.  (Written out, because ahead of any read of LDS the compiler waits for all of such loads.  The wait states are
// those between a vector instruction's write of the base and the load.  m0 is named, though reserved, so that the compiler keeps nothing of its own in it across them.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ unsigned lds_address(const char* p) { return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char*)p; }
__device__ __forceinline__ void bring16(const char* base, unsigned offset, unsigned lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds) : "m0", "memory");
}
__device__ __forceinline__ void bring4(const void* base, unsigned offset, unsigned lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dword %0, %1" ::"v"(offset), "s"(base), "s"(lds) : "m0", "memory");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void arrived() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// All waves' accesses to LDS so far are done.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Many rows: each of the four waves has 16 R rows of its own, and all of them walk the same keys, which the workgroup brings to LDS step by step, AHEAD steps ahead
// of the one that is worked on, with one barrier a step.  (Through registers, one tile of 64 keys ahead with two barriers: 118 us for 256 rows a key head over
// 65536 keys, this 102, of which the launch that joins their 33 parts is 10.  The next step's K to registers ahead of the barrier as well: no change.)  16-byte piece
// c of key i lies at place c ^ turn(i), so that the 16 keys of a score tile, and the 8 keys by 32 bytes that half a wave reads of V, come from different
// banks.  16-bit V comes by transposing reads (of 4 keys by 16 dimensions, per 16 lanes), which save the vector unit the 32 permutations of a step.
template <typename T, int D, int R>
struct WideWalk {
    static constexpr bool F = T::bytes == 4;
    using Rows = AttentionRows<T, D, R, !F>;
    static constexpr int ROW = Rows::ROW, TPL = Rows::TPL, STEP = Rows::STEP;
    static constexpr int PIECES = ROW / 16;
    static constexpr int TILE = STEP;
    static constexpr int KEYS = 1024 / ROW, LOADS = TILE / KEYS / 4;    // keys of a wave's load, which lie in one block, and its loads of a tile's K, and of its V
    static constexpr int BUFFERS = 4, AHEAD = BUFFERS - 1;
    static constexpr int BUFFER = 2 * TILE * ROW, PAGES = BUFFERS * BUFFER;
    static constexpr int LDS = PAGES + 4 * 2 * 64 * 4;

    int page;              // lane i: of block `window` + i, and the block's place in it
    unsigned in;
    unsigned window;
    unsigned long long bad;  // bit i: block `window` + i is in no page
    unsigned long long bad_ahead;  // of the tiles brought and not yet worked on, the next one's blocks in the lowest bits
    unsigned odd;          // which half of the wave's place in LDS the next window's pages are in
    unsigned lane_at[LOADS];

    __device__ __forceinline__ static int turn(int key) {
        if constexpr (F) return key & 15;
        else if constexpr (PIECES >= 16) return (key >> 4 & 1) | (key & 3) << 1 | (key >> 3 & 1) << 3;
        else return (key >> 4 & 1) | (key >> 1 & 1) << 1 | (key >> 3 & 1) << 2;  // two keys make up the banks
    }

    __device__ __forceinline__ static int wave_of() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

    // The pages of the window behind, through LDS: 64 blocks are 8 tiles or more, so that they are there when they are asked for.
    __device__ __forceinline__ void look_ahead(const Keys& s, const char* lds, int lane) {
        bring4(s.table, s.place_of(window + 64 + lane).entry * 4u, lds_address(lds) + PAGES + (wave_of() * 2 + odd) * 256);
    }

    __device__ __forceinline__ void begin(const Keys& s, int first, const char* lds, int lane) {
        window = (unsigned)first / 8;
        const Keys::Place at = s.place_of(window + lane);
        page = s.table[at.entry];
        in = at.in;
        bad = __ballot((unsigned)page >= s.num_pages);
        bad_ahead = 0;
        odd = 0;
        look_ahead(s, lds, lane);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int key = (wave_of() * LOADS + i) * KEYS + lane / PIECES;
            lane_at[i] = (unsigned)(lane / PIECES * ROW + (lane % PIECES ^ turn(key)) * 16);
        }
    }

    // Asks for the tile from key `first` on, which `before` tiles that are not yet worked on precede.
    __device__ __forceinline__ void bring(const Keys& s, int first, int buffer, int before, const char* lds, int lane) {
        if ((unsigned)first / 8 == window + 64) {
            window += 64;
            page = reinterpret_cast<const int*>(lds + PAGES)[(wave_of() * 2 + odd) * 64 + lane];
            in = s.place_of(window + lane).in;
            bad = __ballot((unsigned)page >= s.num_pages);
            odd ^= 1;
            look_ahead(s, lds, lane);
        }
        const unsigned block = (unsigned)first / 8 - window;
        bad_ahead |= (bad >> block & ((1ull << TILE / 8) - 1)) << (before * (TILE / 8));
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int load = wave_of() * LOADS + i;
            const int lies = (int)block + load * KEYS / 8;
            const size_t at = s.page_at(__builtin_amdgcn_readlane(page, lies)) + (size_t)(((unsigned)__builtin_amdgcn_readlane((int)in, lies) * 8 + load * KEYS % 8) * ROW);
            const unsigned to = lds_address(lds) + buffer * BUFFER + load * 1024;
            bring16(s.k + at, lane_at[i], to);
            bring16(s.v + at, lane_at[i], to + TILE * ROW);
        }
    }

    // What lies in places of V that no row may see can be anything, and 0 * NaN is NaN.  (Each wave for the keys that it brought.)
    __device__ __forceinline__ void clear(int first, int most, unsigned gone, char* buffer, int lane) const {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int load = wave_of() * LOADS + i, key = load * KEYS + lane / PIECES;
            if (gone >> (key / 8) & 1 || first + key >= most) *reinterpret_cast<u32x4*>(buffer + TILE * ROW + load * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
        }
    }

    // Keys `first` (a multiple of STEP) to `end`; `least` and `most` bound the limits of the workgroup's rows.
    __device__ __forceinline__ void walk(Rows& rows, const Keys& s, int first, int end, const int (&limit)[R], int least, int most, float scale, int lane, char* lds) {
        if (first >= end) return;
        begin(s, first, lds, lane);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (first + i * TILE < end) bring(s, first + i * TILE, i, i, lds, lane);
        const int group = lane >> 4, mm = lane & 15;
        constexpr int V_PLACES = F ? 4 : PIECES < 16 ? PIECES / 2 : 8;
        int k_at[Rows::KC], v_at[V_PLACES];
        {
            const int key = F ? mm : (mm >> 2) * 8 + (mm & 3);
#pragma unroll
            for (int c = 0; c < Rows::KC; ++c) k_at[c] = key * ROW + ((c * 4 + group) ^ turn(key)) * 16;
#pragma unroll
            for (int u = 0; u < V_PLACES; ++u) {
                if constexpr (F) {  // key u of the lane group's, the lane's four dimensions
                    const int from = group * TPL + u;
                    v_at[u] = TILE * ROW + from * ROW + (mm ^ turn(from)) * 16;
                } else {  // key mm / 4 of the lane group's, dimensions 16 u + mm % 4 * 4 on
                    const int from = group * TPL + (mm >> 2);
                    v_at[u] = TILE * ROW + from * ROW + ((u * 2 + (mm >> 1 & 1)) ^ turn(from)) * 16 + (mm & 1) * 8;
                }
            }
        }
        int buffer = 0;
        for (; first < end; first += TILE) {
            if (first + (AHEAD - 1) * TILE < end) arrived<(AHEAD - 1) * 2 * LOADS>();
            else arrived<0>();
            char* const from = lds + buffer * BUFFER;
            const unsigned gone_blocks = (unsigned)(bad_ahead & ((1ull << TILE / 8) - 1));
            bad_ahead >>= TILE / 8;
            if (first + TILE > most || gone_blocks) clear(first, most, gone_blocks, from, lane);
            lds_barrier();  // the tile is there, and the one before it has been read
            if (first + AHEAD * TILE < end) bring(s, first + AHEAD * TILE, buffer == 0 ? BUFFERS - 1 : buffer - 1, AHEAD - 1, lds, lane);
            f32x4 x[R][Rows::NT];
            rows.scores(x, [&](int t, int c) { return *reinterpret_cast<const u32x4*>(from + k_at[c] + t * 4 * ROW); });
            unsigned w[TPL][Rows::GRP * Rows::VW];
            u32x4 straight[D / 16];
            // pieces and keys further on whose bits the turn leaves alone are at fixed distances
            if constexpr (F) {
#pragma unroll
                for (int u = 0; u < TPL; ++u)
#pragma unroll
                    for (int g = 0; g < Rows::GRP; ++g) {
                        const u32x4 y = *reinterpret_cast<const u32x4*>(from + v_at[u] + g * 256);
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[u][g * 4 + e] = y[e];
                    }
            } else {
                typedef short s16x4 __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) s16x4* LdsPointer;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    const char* const at = from + v_at[d % V_PLACES] + d / V_PLACES * 256;
                    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPointer)at));
                    const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPointer)(at + 4 * ROW)));
                    straight[d] = u32x4{a.x, a.y, b.x, b.y};
                }
            }
            const bool gone = gone_blocks >> (group * TPL / 8) & 1;
            if (first + STEP > least || gone_blocks) Rows::mask(x, first + group * TPL, gone, limit);
            unsigned p[1][R][4];
            rows.weigh(x, scale, p);
            if constexpr (F) rows.add_values(w, p);
            else rows.add_straight(straight, p[0]);
            buffer = buffer == BUFFERS - 1 ? 0 : buffer + 1;
        }
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

// A workgroup's form: how many 16-row tiles a wave has, and whether the waves share rows (16) and split the keys, or the other way round.
template <int TILES, bool WIDE_>
struct Form {
    static constexpr int R = TILES;
    static constexpr bool WIDE = WIDE_;
    static constexpr int ROWS = 16 * R * (WIDE ? 4 : 1);
};

template <typename T, int D, typename Fm>
constexpr int attention_lds() {
    constexpr int sums = 4 * 16 * (8 + (D + 4) * 4);
    return Fm::WIDE && WideWalk<T, D, Fm::R>::LDS > sums ? WideWalk<T, D, Fm::R>::LDS : sums;
}

// What the waves have summed for rows `row_id` (LDS; -1: none), to slot `part` (or, where there is one, as the output).
template <typename T, int D, typename Fm>
__device__ __forceinline__ void leave(const AttentionArgs& a, const AttentionRows<T, D, Fm::R, Fm::WIDE && T::bytes == 2>& rows, int part, const int* row_id, char* lds) {
    constexpr int R = Fm::R;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // Through LDS, so that a row's outputs leave side by side, 16 rows of each wave at a time: the waves' sums of one row where they split the keys
    constexpr int PITCH = D + 4;  // floats of a row in LDS: lanes of different rows on different banks
    f32x2* const ml = reinterpret_cast<f32x2*>(lds);                 // [4][16]
    float* const sums = reinterpret_cast<float*>(lds + 4 * 16 * 8);  // [4][16][PITCH]
    const size_t all = (size_t)a.tokens * a.heads;
    const bool whole = a.acc == nullptr;
    const __amdgpu_buffer_rsrc_t to = whole ? descriptor(a.out) : descriptor(a.acc + (size_t)part * all * D);
    const __amdgpu_buffer_rsrc_t to_ml = descriptor(a.ml + (size_t)part * (whole ? 0 : all));
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (Fm::WIDE) __syncthreads();  // the keys, or the rows before, have been read
        const float own = rows.sum_of(r);
        // (a NaN among a row's scores is no maximum: an infinite one makes NaN of whatever the sum meets further on)
        if (lane < 16) ml[wave * 16 + lane] = f32x2{own == own ? rows.m[r] : INFINITY, own};
        rows.put_sums(r, sums + (wave * 16 + (lane & 15)) * PITCH, lane);
        __syncthreads();
        for (int e = threadIdx.x; e < (Fm::WIDE ? 64 : 16) * (D / 4); e += 256) {
            const int row = e / (D / 4), d = (e - row * (D / 4)) * 4;
            const int id = row_id[Fm::WIDE ? (row >> 4) * 16 * R + r * 16 + (row & 15) : row];
            if (id < 0) continue;
            float top, l;
            f32x4 sum;
            if constexpr (Fm::WIDE) {
                const f32x2 w = ml[row];
                top = w.x;
                l = w.y;
                sum = *reinterpret_cast<const f32x4*>(sums + row * PITCH + d);
            } else {
                top = -INFINITY;
                l = 0.f;
                sum = f32x4{0.f, 0.f, 0.f, 0.f};
                f32x2 w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = ml[i * 16 + row];
                    top = fmaxf(top, w[i].x);
                }
                if (top > -INFINITY) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float f = __builtin_amdgcn_exp2f(w[i].x - top);
                        l += w[i].y * f;
                        sum += *reinterpret_cast<const f32x4*>(sums + (i * 16 + row) * PITCH + d) * f;
                    }
                }
            }
            if (whole) {
                put_out<T>(to, (unsigned)id * D + d, l == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : sum / l);
            } else {
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sum), to, (int)(((unsigned)id * D + d) * 4), 0, kThrough);
                if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(u32x2{as_word(top), as_word(l)}, to_ml, id * 8, 0, kThrough);
            }
        }
    }
}

// A workgroup's part: the rows of its tile over steps [begin, end) of `s`.
template <typename T, int D, typename Fm>
__device__ __forceinline__ void attend(const AttentionArgs& a, const Keys& s, const char* const (&q_row)[Fm::R], const int (&limit)[Fm::R], int least, int most,
                                       int begin, int end, int part, const int* row_id, char* lds) {
    constexpr int R = Fm::R;
    using Rows = AttentionRows<T, D, R, Fm::WIDE && T::bytes == 2>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Rows rows;
    rows.begin();
#pragma unroll
    for (int r = 0; r < R; ++r) rows.load_q(r, q_row[r], lane);
    if constexpr (Fm::WIDE) {
        WideWalk<T, D, R> keys;
        keys.walk(rows, s, begin * Rows::STEP, end * Rows::STEP, limit, least, most, a.scale_log2, lane, lds);
    } else {
        NarrowWalk<T, D> keys;
        keys.walk(rows, s, begin + wave, end, limit, least, most, a.scale_log2, lane);
    }
    leave<T, D, Fm>(a, rows, part, row_id, lds);
}

// What some parts of a row sum up to, four outputs from d on.
struct Joined {
    float top = -INFINITY, l = 0.f;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    __device__ __forceinline__ void add(float t, float n, f32x4 x) {
        const float f = __builtin_amdgcn_exp2f(t - top);
        l += n * f;
        sum += x * f;
    }
    __device__ __forceinline__ bool raise(float now) {  // the running maximum; false while there is nothing
        if (now == -INFINITY) return false;
        const float shrink = __builtin_amdgcn_exp2f(top - now);
        sum *= shrink;
        l *= shrink;
        top = now;
        return true;
    }
    __device__ __forceinline__ f32x4 out() const { return l == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : sum / l; }
};

// Parts first, first + every, ... of row `id`, in their order, N of them requested together.  (CACHE: kThrough where other workgroups of this launch
// wrote them.)
template <int D, int N, int CACHE>
__device__ __forceinline__ Joined join_parts(const AttentionArgs& a, int id, int d, int first, int every) {
    const int parts = (int)(a.prefix_splits.d + a.own_splits.d);
    const size_t rows = (size_t)a.tokens * a.heads;
    Joined all;
    for (; first < parts; first += N * every) {
        u32x2 w[N];
        u32x4 x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int part = min(first + i * every, parts - 1);
            w[i] = __builtin_amdgcn_raw_buffer_load_b64(descriptor(a.ml + part * rows), id * 8, 0, CACHE);
            x[i] = __builtin_amdgcn_raw_buffer_load_b128(descriptor(a.acc + part * rows * D), (int)(((unsigned)id * D + d) * 4), 0, CACHE);
        }
        float now = all.top;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (first + i * every < parts) now = fmaxf(now, as_float(w[i].x));
        if (!all.raise(now)) continue;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (first + i * every < parts) all.add(as_float(w[i].x), as_float(w[i].y), __builtin_bit_cast(f32x4, x[i]));
    }
    return all;
}

// Counts the workgroup in at each of its rows and puts together the rows at which it is the last.  (As in the convs' split reductions: parts
// are written through ahead of the count.)
template <typename T, int D, int MOST>
__device__ __forceinline__ void join_last(const AttentionArgs& a, const int* row_id, unsigned first_counter, int rows_here, int* done) {
    const int lane = threadIdx.x & 63, parts = (int)(a.prefix_splits.d + a.own_splits.d);
    __shared__ int count;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x < 64) {
        int n = 0;
#pragma unroll
        for (int first = 0; first < MOST; first += 64) {
            const int id = first + lane < rows_here ? row_id[first + lane] : -1;
            bool last = false;
            if (id >= 0) {
                unsigned* const counter = a.counters + first_counter + first + lane;
                last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)parts - 1;
                if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            const unsigned long long who = __ballot(last);
            if (last) done[n + __popcll(who & ((1ull << lane) - 1))] = id;
            n += __popcll(who);
        }
        if (lane == 0) count = n;
    }
    __syncthreads();
    const int n = count;
    const __amdgpu_buffer_rsrc_t to = descriptor(a.out);
    for (int e = threadIdx.x; e < n * (D / 4); e += 256) {
        const int id = done[e / (D / 4)], d = e % (D / 4) * 4;
        put_out<T>(to, (unsigned)id * D + d, join_parts<D, kJoined, kThrough>(a, id, d, 0, 1).out());
    }
}

// All rows' parts by a launch of its own: where a workgroup's rows are many, the one that arrives last would be at it for longer than that takes.  A quarter of
// a row's parts per group of lanes, all of them requested at once up to 32: 2048 rows of 128 in 34 parts, 36 MB, by whole rows in steps of
// eight 18 us.
template <typename T, int D>
__global__ __launch_bounds__(256) void prefix_attention_join_kernel(AttentionArgs a) {
    hook_entry(a.notifier, a.job_id);
    constexpr int LANES = D / 4, ROWS = kJoinRows / D;
    static_assert(ROWS * LANES == 64, "a wave per quarter");
    __shared__ f32x4 sums[4][ROWS * LANES];
    __shared__ f32x2 ml[4][ROWS * LANES];
    const int rows = (a.starts ? min(max(a.starts[a.sequences], 0), a.tokens) : a.tokens) * a.heads;
    const int at = (int)threadIdx.x % (ROWS * LANES), quarter = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);  // (a wave each: descriptors go by it)
    const int row = blockIdx.x * ROWS + at / LANES, d = at % LANES * 4;
    if (row < rows) {
        const Joined mine = join_parts<D, 8, 0>(a, row, d, quarter, 4);
        sums[quarter][at] = mine.sum;
        ml[quarter][at] = f32x2{mine.top, mine.l};
    }
    __syncthreads();
    if (quarter == 0 && row < rows) {
        Joined all;
        if (all.raise(fmaxf(fmaxf(ml[0][at].x, ml[1][at].x), fmaxf(ml[2][at].x, ml[3][at].x)))) {
#pragma unroll
            for (int i = 0; i < 4; ++i) all.add(ml[i][at].x, ml[i][at].y, sums[i][at]);
        }
        put_out<T>(descriptor(a.out), (unsigned)row * D + d, all.out());
    }
    hook_exit(a.notifier, a.job_id);
}

// FP, FO: the form of a workgroup over the prefix / over a sequence's own tokens.
template <typename T, int D, typename FP, typename FO>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void prefix_attention_kernel(AttentionArgs a) {
    hook_entry(a.notifier, a.job_id);
    constexpr int LP = attention_lds<T, D, FP>(), LO = attention_lds<T, D, FO>(), MOST = FP::ROWS > FO::ROWS ? FP::ROWS : FO::ROWS;
    __shared__ __attribute__((aligned(16))) char lds[LP > LO ? LP : LO];
    __shared__ int row_id[MOST], done[MOST];
    constexpr int STEP = AttentionRows<T, D, 1, false>::STEP;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int head_bytes = D * T::bytes;
    Keys s;
    s.page_bytes = (size_t)a.kv_heads.d * a.page_size * head_bytes;
    s.page_blocks = a.page_blocks;
    s.num_pages = (unsigned)a.num_pages;
    const bool over_prefix = blockIdx.x < a.prefix_items;
    const unsigned item = over_prefix ? blockIdx.x : blockIdx.x - a.prefix_items;
    bool any = true;
    unsigned first_counter = 0;
    if (over_prefix) {
        // (key head, split) by tile: the tiles of one pair read the same keys, so they follow each other by 8 and share an XCD's cache
        const unsigned eights = (unsigned)a.prefix_pairs / 8 * a.eight_tiles.d, left = (unsigned)a.prefix_pairs % 8;
        unsigned pair, tile;
        if (item < eights) {
            const Quotient at = divide(item, a.eight_tiles);
            pair = at.q * 8 + item % 8;
            tile = at.r / 8;
        } else {
            tile = (item - eights) / left;
            pair = (unsigned)a.prefix_pairs / 8 * 8 + (item - eights) - tile * left;
        }
        const Quotient who = divide(pair, a.prefix_splits);
        const int h = (int)who.q, split = (int)who.r, per_kv = (int)a.per_kv.d;
        // rows behind the last sequence are left out (their lanes take the last row's query)
        const int first_row = (int)tile * FP::ROWS, group_rows = (a.starts ? min(max(a.starts[a.sequences], 0), a.tokens) : a.tokens) * per_kv;
        first_counter = (unsigned)h * a.counter_pitch + (unsigned)first_row;
        const char* q_row[FP::R];
        int limit[FP::R];
#pragma unroll
        for (int r = 0; r < FP::R; ++r) {
            const int x = max(min(first_row + (FP::WIDE ? wave * 16 * FP::R : 0) + r * 16 + (lane & 15), group_rows - 1), 0);
            const Quotient at = divide((unsigned)x, a.per_kv);
            q_row[r] = a.q + at.q * a.q_stride + (h * per_kv + (int)at.r) * head_bytes;
            limit[r] = a.prefix_len;
        }
        if ((int)threadIdx.x < FP::ROWS) {
            const int x = first_row + (int)threadIdx.x;
            const Quotient at = divide((unsigned)x, a.per_kv);
            row_id[threadIdx.x] = x < group_rows ? (int)at.q * a.heads + h * per_kv + (int)at.r : -1;
        }
        __syncthreads();
        s.table = a.prefix_table;
        s.table_len = a.prefix_pages;
        s.k = a.k_cache + (size_t)h * a.page_size * head_bytes;
        s.v = a.v_cache + (size_t)h * a.page_size * head_bytes;
        const int steps = (a.prefix_len + STEP - 1) / STEP;
        const int begin = min(split * a.prefix_per, steps), end = min(begin + a.prefix_per, steps);
        attend<T, D, FP>(a, s, q_row, limit, a.prefix_len, a.prefix_len, begin, end, split, row_id, lds);
    } else {
        // the key heads of one sequence side by side: they share the look-ups and, with eight of them, an XCD each
        const Quotient by_head = divide(item, a.kv_heads), by_split = divide(by_head.q, a.own_splits), by_tile = divide(by_split.q, a.own_tiles);
        const int h = (int)by_head.r, split = (int)by_split.r, tile = (int)by_tile.r, seq = (int)by_tile.q, per_kv = (int)a.per_kv.d;
        int first = seq * a.max_new, count = a.max_new;
        if (a.starts) {
            first = min(max(__builtin_amdgcn_readfirstlane(a.starts[seq]), 0), a.tokens);
            count = min(min(__builtin_amdgcn_readfirstlane(a.starts[seq + 1]), a.tokens) - first, a.max_new);
        }
        const int first_row = tile * FO::ROWS, group_rows = max(count, 0) * per_kv;
        any = first_row < group_rows;
        first_counter = (unsigned)h * a.counter_pitch + (unsigned)(first * per_kv + first_row);
        if (any) {
            const int capacity = (int)min((int64_t)a.max_pages * a.page_size, (int64_t)1 << 30);
            const int past = min(max(__builtin_amdgcn_readfirstlane(a.past[seq]), 0), capacity);
            auto limit_of = [&](int row) { return min(past + (int)divide((unsigned)min(row, group_rows - 1), a.per_kv).q + 1, capacity); };
            const int wave_row = first_row + (FO::WIDE ? wave * 16 * FO::R : 0);
            const char* q_row[FO::R];
            int limit[FO::R];
#pragma unroll
            for (int r = 0; r < FO::R; ++r) {
                const Quotient at = divide((unsigned)min(wave_row + r * 16 + (lane & 15), group_rows - 1), a.per_kv);
                q_row[r] = a.q + (first + (int)at.q) * a.q_stride + (h * per_kv + (int)at.r) * head_bytes;
                limit[r] = min(past + (int)at.q + 1, capacity);
            }
            if ((int)threadIdx.x < FO::ROWS) {
                const int x = first_row + (int)threadIdx.x;
                const Quotient at = divide((unsigned)x, a.per_kv);
                row_id[threadIdx.x] = x < group_rows ? (first + (int)at.q) * a.heads + h * per_kv + (int)at.r : -1;
            }
            __syncthreads();
            s.table = a.tables + (size_t)seq * a.max_pages;
            s.table_len = a.max_pages;
            s.k = a.k_cache + (size_t)h * a.page_size * head_bytes;
            s.v = a.v_cache + (size_t)h * a.page_size * head_bytes;
            const int least = limit_of(wave_row), most = limit_of(first_row + FO::ROWS - 1);
            const int steps = (most + STEP - 1) / STEP;
            const int per = (int)divide((unsigned)steps + a.own_splits.d - 1, a.own_splits).q;
            const int begin = min(split * per, steps), end = min(begin + per, steps);
            attend<T, D, FO>(a, s, q_row, limit, least, most, begin, end, (int)a.prefix_splits.d + split, row_id, lds);
        }
    }
    if (any && a.counters) join_last<T, D, MOST>(a, row_id, first_counter, over_prefix ? FP::ROWS : FO::ROWS, done);
    hook_exit(a.notifier, a.job_id);
}

using AttentionKernel = void (*)(AttentionArgs);

// Which forms a type and head size have, by the rows of a workgroup: 16 (the waves split the keys), 64 and 128 (they split the rows).
template <typename T, int D>
AttentionKernel attention_kernel_of(int rp, int ro) {
    using N1 = Form<1, false>;
    using W1 = Form<1, true>;
    if (rp == 16 && ro == 16) return prefix_attention_kernel<T, D, N1, N1>;
    if (rp == 64 && ro == 16) return prefix_attention_kernel<T, D, W1, N1>;
    if (rp == 64 && ro == 64) return prefix_attention_kernel<T, D, W1, W1>;
    if constexpr (D * T::bytes <= 256) {  // what the registers hold without a spill
        using W2 = Form<2, true>;
        if (rp == 128 && ro == 16) return prefix_attention_kernel<T, D, W2, N1>;
        if (rp == 128 && ro == 128) return prefix_attention_kernel<T, D, W2, W2>;
    }
    return nullptr;
}

template <typename T>
AttentionKernel attention_kernel(int dim, int rp, int ro) {
    return dim == 64 ? attention_kernel_of<T, 64>(rp, ro) : dim == 128 ? attention_kernel_of<T, 128>(rp, ro) : dim == 256 ? attention_kernel_of<T, 256>(rp, ro) : nullptr;
}

template <typename T>
AttentionKernel attention_join(int dim) {
    return dim == 64 ? prefix_attention_join_kernel<T, 64> : dim == 128 ? prefix_attention_join_kernel<T, 128> : prefix_attention_join_kernel<T, 256>;
}

// The kernels of a type for a head size and rows per workgroup (nullptr where there is none), and for joining.  Defined once per type.
AttentionKernel attention_kernel_f32(int dim, int rp, int ro);
AttentionKernel attention_kernel_bf16(int dim, int rp, int ro);
AttentionKernel attention_kernel_f16(int dim, int rp, int ro);
AttentionKernel attention_join_f32(int dim);
AttentionKernel attention_join_bf16(int dim);
AttentionKernel attention_join_f16(int dim);

}  // namespace paella
