#pragma once
// What the operators of a decoding step share: element types, 16-byte loads, write-through stores, page lookups.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "paella_decode.h"
#include "paella_ops.h"
#include <llis/job/finished_block_notifier.h>

#include "launch.h"
#include "out_store.h"

namespace paella {

using Notifier = llis::job::FinishedBlockNotifier;

struct F32 { static constexpr int bytes = 4; };
struct Bf16 { static constexpr int bytes = 2; };
struct F16 { static constexpr int bytes = 2; };

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// By value: a bit cast of a vector's element in place reads element 0.
__device__ __forceinline__ float as_float(unsigned w) { return __builtin_bit_cast(float, w); }
__device__ __forceinline__ unsigned as_word(float f) { return __builtin_bit_cast(unsigned, f); }

// Two neighbouring 16-bit values of a word, and back (one rounding, to nearest even).
template <typename T> __device__ __forceinline__ f32x2 unpack2(unsigned w);
template <> __device__ __forceinline__ f32x2 unpack2<Bf16>(unsigned w) {
    return f32x2{as_float(w << 16), as_float(w & 0xFFFF0000u)};
}
template <> __device__ __forceinline__ f32x2 unpack2<F16>(unsigned w) { return __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2); }

template <typename T> __device__ __forceinline__ unsigned pack2(float a, float b);
template <> __device__ __forceinline__ unsigned pack2<Bf16>(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
template <> __device__ __forceinline__ unsigned pack2<F16>(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, f16x2));
}

// A value of 16 lanes side by side by the vector unit's own lane moves (an exchange through LDS takes ten times as long), and of all 64.
template <int CONTROL>
__device__ __forceinline__ float lane_move(float v) { return as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)as_word(v), CONTROL, 0xF, 0xF, false)); }
template <int CONTROL>
__device__ __forceinline__ double lane_move(double v) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)b, CONTROL, 0xF, 0xF, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), CONTROL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
template <typename V, typename Op>
__device__ __forceinline__ V row_all(V v, Op op) {
    v = op(v, lane_move<0xB1>(v));   // lane ^ 1
    v = op(v, lane_move<0x4E>(v));   // lane ^ 2
    v = op(v, lane_move<0x141>(v));  // the other half of eight, mirrored
    return op(v, lane_move<0x140>(v));  // the other half of sixteen, mirrored
}
// The sum over 2^log2 lanes side by side, which is the same for all of the wave.
__device__ __forceinline__ float lanes_sum(float v, int log2) {
    if (log2 > 0) v += lane_move<0xB1>(v);
    if (log2 > 1) v += lane_move<0x4E>(v);
    if (log2 > 2) v += lane_move<0x141>(v);
    if (log2 > 3) v += lane_move<0x140>(v);
    if (log2 > 4) v += __shfl_xor(v, 16, 64);
    if (log2 > 5) v += __shfl_xor(v, 32, 64);
    return v;
}
template <typename Op>
__device__ __forceinline__ float wave_all(float v, Op op) {
    v = row_all(v, op);
    const float a = as_float(__builtin_amdgcn_readlane(as_word(v), 0)), b = as_float(__builtin_amdgcn_readlane(as_word(v), 16));
    const float c = as_float(__builtin_amdgcn_readlane(as_word(v), 32)), d = as_float(__builtin_amdgcn_readlane(as_word(v), 48));
    return op(op(a, b), op(c, d));
}
__device__ __forceinline__ float wave_sum_f(float v) {
    return wave_all(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_max_f(float v) {
    return wave_all(v, [](float a, float b) { return fmaxf(a, b); });
}

// Division by a number that the host knows: with 2^32 over it, rounded down (all ones for 1), the product's upper half is the quotient or one less.  (A
// division costs some forty instructions; a workgroup of a small launch spends a microsecond on the half dozen that say what its work is.)
struct Divisor {
    unsigned d, inv;
};
inline Divisor divisor(unsigned d) { return {d, d <= 1 ? 0xFFFFFFFFu : (unsigned)(0x100000000ull / d)}; }
struct Quotient {
    unsigned q, r;
};
__device__ __forceinline__ Quotient divide(unsigned n, Divisor by) {
    unsigned q = __umulhi(n, by.inv), r = n - q * by.d;
    if (r >= by.d) {
        ++q;
        r -= by.d;
    }
    return {q, r};
}

// A descriptor over everything behind `base` (uniform over the wave); offsets are 32-bit, sc1 = 16 writes through / reads past this XCD's caches.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t descriptor(const void* base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0xFFFFFFFFu, 0x00027000);
}
constexpr int kThrough = 16;

// The sequence of row t and its index j among the sequence's new tokens, found by every wave for itself with one load per 64 sequences;
// false for rows that belong to none.  t is uniform over the wave.
__device__ __forceinline__ bool row_owner(const int* __restrict__ starts, int sequences, Divisor max_new, int t, int lane, int* seq, int* j) {
    if (!starts) {
        const Quotient at = divide((unsigned)t, max_new);
        *seq = (int)at.q;
        *j = (int)at.r;
        return *seq < sequences;
    }
    int b = 0;
    for (int at = 0; at < sequences; at += 64) {
        const int i = at + lane;
        const unsigned long long begun = __ballot(i < sequences && starts[i + 1] <= t);
        b += __popcll(begun);
        if (begun != ~0ull) break;
    }
    *seq = b;
    if (b >= sequences) return false;
    *j = t - starts[b];
    return *j >= 0 && *j < (int)max_new.d;
}

// Host side: what every entry point asks of a cache and a batch.
constexpr double kMostWorkgroups = 16777215.;  // of 256 threads in one launch: the runtime counts threads in 32 bits
inline int element_bytes(int dtype) { return dtype == PAELLA_F32 ? 4 : 2; }

inline bool cache_extents_ok(const paella_kv_cache* c) {
    if (!c || c->dtype < PAELLA_F32 || c->dtype > PAELLA_F16 || c->num_pages <= 0 || c->kv_heads <= 0 || c->page_size <= 0 || c->head_dim <= 0) return false;
    if (c->page_size % 8 || c->head_dim % 8 || c->head_dim > 512) return false;
    return (double)c->kv_heads * c->page_size * c->head_dim * element_bytes(c->dtype) < 2147483648.0;
}
inline bool cache_ok(const paella_kv_cache* c) { return cache_extents_ok(c) && c->k && c->v && (((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0; }

inline bool batch_extents_ok(const paella_kv_batch* b) {
    if (!b || b->sequences <= 0 || b->max_new <= 0 || b->tokens <= 0 || b->max_pages <= 0 || b->prefix_len < 0) return false;
    // rows and positions are 32-bit numbers
    if (b->max_new >= 1 << 30) return false;
    return (double)b->sequences * b->max_new < 2147483648.0 && (double)b->sequences * b->max_pages < 2147483648.0 && b->prefix_len < (1 << 30);
}
inline bool batch_ok(const paella_kv_batch* b) {
    if (!batch_extents_ok(b) || !b->past || !b->tables) return false;
    return b->starts != nullptr || (double)b->sequences * b->max_new == (double)b->tokens;
}

inline bool overlap(const void* a, double a_bytes, const void* b, double b_bytes) {
    const double x = (double)(uintptr_t)a, y = (double)(uintptr_t)b;
    return x < y + b_bytes && y < x + a_bytes;
}

// Of `rows` rows of row_bytes, row_stride bytes (not less) apart: whether any lies over the other memory.
inline bool rows_overlap(const void* a, int64_t rows, int64_t row_stride, int64_t row_bytes, const void* b, double b_bytes) {
    const double ahead = (double)(uintptr_t)b - (double)(uintptr_t)a - (double)row_bytes;  // the first row that ends behind b's beginning
    const double first = ahead < 0 ? 0 : std::floor(ahead / (double)row_stride) + 1;
    return first < (double)rows && (double)(uintptr_t)a + first * (double)row_stride < (double)(uintptr_t)b + b_bytes;
}

// Whether outputs lie over the cache.
inline bool over_cache(const paella_kv_cache* c, const void* out, double bytes) {
    const double size = (double)c->num_pages * c->kv_heads * c->page_size * c->head_dim * element_bytes(c->dtype);
    return overlap(c->k, size, out, bytes) || overlap(c->v, size, out, bytes);
}

inline void set_launch_dims(paella_launch_dims* d, unsigned grid, unsigned block, unsigned lds, unsigned vgprs) {
    d->grid = grid;
    d->block = block;
    d->lds_bytes = lds;
    d->vgprs = vgprs;
}

// Register count and static LDS of the kernel that a launch takes, where there is a device to ask; *dims is left as planned elsewhere.
inline void loaded_dims(const void* kernel, paella_launch_dims* dims) {
    hipFuncAttributes attr;
    if (hipFuncGetAttributes(&attr, kernel) != hipSuccess) {
        (void)hipGetLastError();
        return;
    }
    dims->vgprs = (unsigned)attr.numRegs;
    dims->lds_bytes += (unsigned)attr.sharedSizeBytes;
}

}  // namespace paella
