#pragma once
// The largest of many numbers, by one workgroup: which value the last one taken has, and the taken ones in the order of their places.

#include "decode_common.h"

namespace paella {

// Which of n places the threads of WAVES waves have: those of a wave lie side by side, so that what is taken comes out in order.  KEYS: places of a thread at most, whose values may
// then lie in registers, or 0 for any number.
template <int WAVES, int KEYS>
struct Span {
    unsigned begin, end;
    __device__ __forceinline__ explicit Span(unsigned n) {
        const unsigned wave = (unsigned)__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), per = (n + WAVES * 64 - 1) / (WAVES * 64) * 64;
        begin = min(wave * per, n);
        end = min(begin + per, n);
    }
    // each(u, i, value) for place i, the thread's u-th, and what get(u, i) has for it: 0 behind the last one, where whole waves come along.  Where that reads memory, several are read ahead.
    template <typename Get, typename Each>
    __device__ __forceinline__ void visit(Get get, Each each) const {
        const unsigned lane = threadIdx.x & 63;
        if constexpr (KEYS > 0) {
#pragma unroll
            for (int u = 0; u < KEYS; ++u)
                if (begin + u * 64 < end) each(u, begin + u * 64 + lane, get(u, begin + u * 64 + lane));
        } else {
            constexpr int AHEAD = 8;
            for (unsigned first = begin; first < end; first += AHEAD * 64) {
                decltype(get(0, 0u)) value[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) value[u] = get(0, min(first + u * 64 + lane, end - 1));
#pragma unroll
                for (int u = 0; u < AHEAD; ++u)
                    if (first + u * 64 < end) each(0, first + u * 64 + lane, first + u * 64 + lane < end ? value[u] : 0);
            }
        }
    }
    // Registers' first values: key(load(i)), all requested before the first is looked at.
    template <typename Value, typename Load, typename Key>
    __device__ __forceinline__ void hold(Value (&held)[KEYS ? KEYS : 1], Load load, Key key) const {
        if constexpr (KEYS > 0) {
            const unsigned lane = threadIdx.x & 63;
#pragma unroll
            for (int u = 0; u < KEYS; ++u)
                if (begin + u * 64 < end) held[u] = load(min(begin + u * 64 + lane, end - 1));
#pragma unroll
            for (int u = 0; u < KEYS; ++u)
                if (begin + u * 64 < end) held[u] = begin + u * 64 + lane < end ? key(held[u]) : 0;
        }
    }
};

constexpr unsigned kRanked = 128;  // candidates that are ranked against each other: that takes no longer than another histogram
constexpr int kDigit = 10;         // bits of a digit: of thousands of keys, few are left behind the first histogram

template <int WAVES>
struct PickSpace {
    __attribute__((aligned(16))) unsigned bins[1 << kDigit];
    unsigned long long list[kRanked];
    unsigned long long low[WAVES], high[WAVES], bound;
    unsigned count[3][WAVES];
    unsigned digit, size, left, found;
};

// Numbers as ones whose order is theirs, above 0, -0 and 0 alike; NaN as `nan`.
__device__ __forceinline__ unsigned number_key(float v, unsigned nan) {
    const unsigned b = as_word(v + 0.f);
    return v != v ? nan : b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float key_number(unsigned k) { return as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }
__device__ __forceinline__ unsigned long long number_key(double v, unsigned long long nan) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v + 0.0);
    return v != v ? nan : b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
}

// How many lanes say so: counted by the scalar unit.
__device__ __forceinline__ unsigned wave_count(bool b) { return (unsigned)__popcll(__ballot(b)); }

// op of all lanes' whole numbers, the same for the whole wave.
template <typename Op>
__device__ __forceinline__ unsigned wave_all(unsigned v, Op op) {
    v = row_all(v, op);
    return op(op((unsigned)__builtin_amdgcn_readlane((int)v, 0), (unsigned)__builtin_amdgcn_readlane((int)v, 16)),
              op((unsigned)__builtin_amdgcn_readlane((int)v, 32), (unsigned)__builtin_amdgcn_readlane((int)v, 48)));
}
template <typename Op>
__device__ __forceinline__ unsigned long long wave_all(unsigned long long v, Op op) {
    v = row_all(v, op);
    auto at = [&](int lane) {
        return (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), lane) << 32 | (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, lane);
    };
    return op(op(at(0), at(16)), op(at(32), at(48)));
}
struct Least {
    template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return min(a, b); }
};
struct Most {
    template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return max(a, b); }
};
struct Sum {
    template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
// Of the waves' values in LDS.
template <int WAVES, typename V, typename Op>
__device__ __forceinline__ V waves_all(const V (&of)[WAVES], Op op) {
    if constexpr (WAVES == 16) {
        return row_all(of[threadIdx.x & 15], op);
    } else {
        V v = of[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v = op(v, of[w]);
        return v;
    }
}
template <typename V> __device__ __forceinline__ V uniform(V v) { return v; }
template <> __device__ __forceinline__ unsigned uniform(unsigned v) { return (unsigned)__builtin_amdgcn_readfirstlane((int)v); }
template <> __device__ __forceinline__ unsigned long long uniform(unsigned long long v) {
    return (unsigned long long)uniform((unsigned)(v >> 32)) << 32 | uniform((unsigned)v);
}

// The least and largest of the keys that are not 0, and how many there are, over all threads.
template <typename Key>
struct Range {
    Key least = ~(Key)0, most = 0;  // (the least one less, until they are joined)
    unsigned some = 0;  // of the wave, until they are joined
    __device__ __forceinline__ void add(Key k) {  // by whole waves
        least = min(least, (Key)(k - 1));  // (none is the largest)
        most = max(most, k);
        some += wave_count(k != 0);
    }
    template <int WAVES>
    __device__ __forceinline__ void join(PickSpace<WAVES>& s) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        least = wave_all(least, Least());
        most = wave_all(most, Most());
        __syncthreads();
        if (lane == 0) {
            s.low[wave] = least;
            s.high[wave] = most;
            s.count[0][wave] = some;
        }
        __syncthreads();
        least = (Key)uniform(waves_all(s.low, Least())) + 1;
        most = (Key)uniform(waves_all(s.high, Most()));
        some = uniform(waves_all(s.count[0], Sum()));
    }
    // Of joined ranges: whether k is among the keys, or beyond them all.
    __device__ __forceinline__ bool holds(Key k) const { return k - least <= most - least; }
};

// What is taken: keys above `bound`, and the first `left` of those equal to it (all of them where left is ~0).
template <typename Key>
struct Bound {
    Key bound;
    unsigned left;
};

// Of the keys get(u, i) within `range`, which is theirs (others may lie below and above it): the `want` largest.  Digit by digit from the highest one in which the keys differ, by a histogram of the
// keys that agree with the bound so far, until they are so few that each is ranked against all others.  Called by all threads.
template <int WAVES, int KEYS, typename Key, typename Get>
__device__ __forceinline__ Bound<Key> find_bound(const Span<WAVES, KEYS>& span, const Range<Key>& range, unsigned want, PickSpace<WAVES>& s, Get get) {
    if (range.some <= want) return {1, ~0u};
    const int lane = threadIdx.x & 63;
    const int differ = range.least == range.most ? 0 : 64 - __clzll((unsigned long long)(range.least ^ range.most));  // bits; those above are the same in all keys
    if (!differ) return {range.most, want};
    int shift = max(differ - kDigit, 0);
    Key known = shift + kDigit < (int)sizeof(Key) * 8 ? (Key)(~(Key)0 << (shift + kDigit)) : (Key)0;  // the bits that the bound has so far
    Key bound = range.most & known;
    unsigned left = want, size = range.some;
    while (size > kRanked) {
        __syncthreads();
        for (unsigned b = threadIdx.x; b < 1u << kDigit; b += WAVES * 64) s.bins[b] = 0;
        __syncthreads();
        span.visit(get, [&](int, unsigned, Key k) {
            if (range.holds(k) && (k & known) == bound) atomicAdd(&s.bins[(unsigned)(k >> shift) & ((1u << kDigit) - 1)], 1u);
        });
        __syncthreads();
        if (threadIdx.x < 64) {  // some digits a lane, the highest first
            constexpr int EACH = (1 << kDigit) / 64;
            const u32x4* const mine = reinterpret_cast<const u32x4*>(s.bins) + (63 - lane) * (EACH / 4);
            u32x4 c[EACH / 4];
            unsigned sum = 0;
#pragma unroll
            for (int e = 0; e < EACH / 4; ++e) {
                c[e] = mine[e];
                sum += c[e].x + c[e].y + c[e].z + c[e].w;
            }
            unsigned upto = sum;
            for (int off = 1; off < 64; off <<= 1) {
                const unsigned other = __shfl_up((int)upto, off, 64);
                if (lane >= off) upto += other;
            }
            unsigned before = upto - sum;
            if (before < left && left <= upto) {
#pragma unroll
                for (int e = EACH - 1; e >= 0; --e) {
                    const unsigned here = c[e / 4][e % 4];
                    if (before < left && left <= before + here) {
                        s.digit = (63 - lane) * EACH + e;
                        s.left = left - before;
                        s.size = here;
                    }
                    before += here;
                }
            }
        }
        __syncthreads();
        bound |= (Key)s.digit << shift;
        left = s.left;
        size = s.size;
        known |= (Key)((1u << kDigit) - 1) << shift;
        if (size == left) return {bound, ~0u};  // all that begin so
        if (shift == 0) return {bound, left};
        shift = max(shift - kDigit, 0);
    }
    __syncthreads();
    if (threadIdx.x == 0) s.found = 0;
    __syncthreads();
    span.visit(get, [&](int, unsigned, Key k) {
        if (range.holds(k) && (k & known) == bound) s.list[atomicAdd(&s.found, 1u)] = k;
    });
    __syncthreads();
    if (threadIdx.x < size) {
        const Key mine = (Key)s.list[threadIdx.x];
        unsigned above = 0, equal = 0;
#pragma unroll 8
        for (unsigned o = 0; o < size; ++o) {
            const Key other = (Key)s.list[o];
            above += other > mine;
            equal += other == mine;
        }
        if (above < left && left <= above + equal) {  // the same for all that are equal
            s.bound = mine;
            s.left = above + equal == left ? ~0u : left - above;
        }
    }
    __syncthreads();
    return {(Key)s.bound, s.left};
}

// Sum of the waves' numbers in LDS ahead of this wave's, and of all.
template <int WAVES>
__device__ __forceinline__ unsigned ahead_of(const unsigned (&of)[WAVES], int wave, unsigned* all) {
    unsigned ahead = 0, sum = 0;
    if constexpr (WAVES == 16) {
        const unsigned v = of[threadIdx.x & 15];
        sum = row_all(v, Sum());
        ahead = row_all((int)(threadIdx.x & 15) < wave ? v : 0u, Sum());
    } else {
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            ahead += w < wave ? of[w] : 0;
            sum += of[w];
        }
    }
    *all = uniform(sum);
    return uniform(ahead);
}

// take(place, i) for the places whose value is mine(value), in order, the wave's from `place` on.
template <int WAVES, int KEYS, typename Get, typename Mine, typename Take>
__device__ __forceinline__ void emit_from(const Span<WAVES, KEYS>& span, unsigned place, Get get, Mine mine, Take take) {
    const unsigned long long before = (1ull << (threadIdx.x & 63)) - 1;
    span.visit(get, [&](int, unsigned i, auto k) {
        const bool is = mine(k);
        const unsigned long long who = __ballot(is);
        if (who) {
            if (is) take(place + (unsigned)__popcll(who & before), i);
            place += (unsigned)__popcll(who);
        }
    });
}

// take(place, i) for every place whose value above(value), and for the first `left` of those whose value is tied(value), in order; returns how many.
template <int WAVES, int KEYS, typename Get, typename Above, typename Tied, typename Take>
__device__ __forceinline__ unsigned emit(const Span<WAVES, KEYS>& span, PickSpace<WAVES>& s, Get get, Above above, Tied tied, unsigned left, Take take) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    unsigned more = 0, equal = 0;
    span.visit(get, [&](int, unsigned, auto k) {
        more += wave_count(above(k));
        if (left) equal += wave_count(tied(k));
    });
    __syncthreads();
    if (lane == 0) {
        s.count[1][wave] = more;
        s.count[2][wave] = equal;
    }
    __syncthreads();
    unsigned all, ties_all = 0, ties = 0;
    unsigned place = ahead_of(s.count[1], wave, &all);
    if (left) ties = ahead_of(s.count[2], wave, &ties_all);
    place += min(ties, left);
    all += min(ties_all, left);
    const unsigned long long before = (1ull << lane) - 1;
    emit_from(span, place, get, [&](auto k) {
        bool mine = above(k);
        if (left) {
            const unsigned long long who = __ballot(tied(k));
            mine |= tied(k) && ties + (unsigned)__popcll(who & before) < left;
            ties += (unsigned)__popcll(who);
        }
        return mine;
    }, take);
    return all;
}

template <int WAVES, int KEYS, typename Key, typename Get, typename Take>
__device__ __forceinline__ unsigned emit_taken(const Span<WAVES, KEYS>& span, Bound<Key> b, PickSpace<WAVES>& s, Get get, Take take) {
    const Key from = b.left == ~0u ? b.bound : b.bound + 1;  // (no bound of which only some are taken is all ones)
    return emit(span, s, get, [&](Key k) { return k >= from; }, [&](Key k) { return k == b.bound; }, b.left == ~0u ? 0u : b.left, take);
}

}  // namespace paella
