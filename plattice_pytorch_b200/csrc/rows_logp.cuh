// rows_logp.cuh -- log probabilities of given labels, entropy and the best
// alternatives of rows of scores, and the scores' gradient.
//
//   m = max x, s = log sum exp(x - m);  log p_j = (x_j - m) - s
//   entropy = -sum p log p = s - sum exp(x - m) (x - m) / sum exp(x - m)
//   grad_j = g_l ([j = label] - p_j) - g_e p_j (log p_j + entropy) + g_z p_j
//
// m and s are kept apart: their sum would lose s beside a large m (rows whose
// scores are all the type's lowest value, say).  s is log1p of the sum without one 1 of
// the largest score.  Where that rest is below 1/16 the 1 is left out from the start, so
// that confident answers keep their precision; else it is added with the others and taken
// off again, which is off by about one rounding of the sum (relative to a rest of 1/16,
// four bits: the log probability is then about -1/16, and off by 2^-24).
//
// A row is read once and held: few classes by a thread out of shared memory, up to
// five accesses a lane by a warp in registers, more by the warps of a CTA or a
// cluster, each with a share of its own; rows that no cluster holds are taken in
// rounds.  So a thread, a warp or a share knows its largest score before the first
// exponential, and an element costs a bound, a multiply-add, the exponential and two
// sums, most of them in pairs.  The special function units take 16 elements a clock
// and SM, 60 us for the 268 M of 8192 x 32768, which take 83 us to read at the copy
// rate and 100 here (108 to 112 behind a kernel whose writes are still in the L2).
#pragma once
#include <cooperative_groups.h>

#include "plattice_runtime.h"
#include "rows_host.h"
#include "rows_logp.h"
#include "rows_vec.cuh"

namespace plr {

namespace cg = cooperative_groups;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -200.f;   // of an exponent of 2: the hardware's exponential is 0 from below -126 on

__device__ __forceinline__ int label_of(const LogpArgs& p, int64_t row) { return Labels{p.labels, p.labels_wide}.at(row, p.n); }
template <typename T> __device__ __forceinline__ const T* lo_of(const LogpArgs& p) { return static_cast<const T*>(p.x); }
template <typename T> __device__ __forceinline__ const T* hi_of(const LogpArgs& p) { return static_cast<const T*>(p.x) + p.rows * p.n; }

// ------------------------------------------------------------- rows in registers

// 16 bytes of a row: kN elements.  Accesses lie on 16-byte boundaries of memory,
// the first of a row perhaps before its start: `shift` elements.  Elements
// outside the row are -inf.
template <typename T> struct Piece {
    static constexpr int kN = 16 / (int)sizeof(T);
    uint4 q;
    static __device__ __forceinline__ int shift_of(const T* x) { return (int)((uintptr_t)x & 15) / (int)sizeof(T); }
    static __device__ __forceinline__ uint32_t closed() {
        if (std::is_same<T, float>::value) return 0xff800000u;
        return std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    }
    // Elements first.. of the row x[0..n), which lies in a tensor lo..hi.
    template <typename Int> __device__ __forceinline__ void load(const T* x, Int first, Int n, const T* lo, const T* hi) {
        const T* at = x + first;
        if (first >= 0 && first + kN <= n) {
            q = *reinterpret_cast<const uint4*>(at);
            return;
        }
        if (first <= -kN || first >= n) {
            q = make_uint4(closed(), closed(), closed(), closed());
            return;
        }
        union { uint4 u; T e[kN]; uint16_t h[8]; uint32_t w[4]; } r;
        r.u = make_uint4(closed(), closed(), closed(), closed());
        if (at >= lo && at + kN <= hi) {   // the neighbouring rows' elements come along
            r.u = *reinterpret_cast<const uint4*>(at);
#pragma unroll
            for (int i = 0; i < kN; ++i)
                if (first + i < 0 || first + i >= n) {
                    if constexpr (sizeof(T) == 4) r.w[i] = closed();
                    else r.h[i] = (uint16_t)closed();
                }
        } else {
#pragma unroll
            for (int i = 0; i < kN; ++i)
                if (first + i >= 0 && first + i < n) r.e[i] = x[first + i];
        }
        q = r.u;
    }
    // The same where all rows begin on 16-byte boundaries: there are no parts.
    template <typename Int> __device__ __forceinline__ void load_whole(const T* x, Int first, Int n) {
        if (first < n) q = *reinterpret_cast<const uint4*>(x + first);
        else q = make_uint4(closed(), closed(), closed(), closed());
    }
    __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w; }
    __device__ __forceinline__ float2 pair(int i) const {   // elements 2 i, 2 i + 1
        if constexpr (std::is_same<T, float>::value) {
            return make_float2(__uint_as_float(word(2 * i)), __uint_as_float(word(2 * i + 1)));
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            return make_float2(__uint_as_float(word(i) << 16), __uint_as_float(word(i) & 0xffff0000u));
        } else {
            const uint32_t w = word(i);
            return __half22float2(*reinterpret_cast<const __half2*>(&w));
        }
    }
    // Puts -inf in the place of elements equal to m; gives their number.
    __device__ __forceinline__ int take(float m) {
        int count = 0;
        if constexpr (std::is_same<T, float>::value) {
            uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (__uint_as_float(w[i]) == m) w[i] = closed(), ++count;
            q = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            typedef typename Pair<T>::type P;
            P both_m;
            pair_from(both_m, m, m);
            uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t same = __heq2_mask(*reinterpret_cast<const P*>(&w[i]), both_m);
                w[i] = (w[i] & ~same) | (same & closed());
                count += __popc(same) >> 4;
            }
            q = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return count;
    }
    template <int K> static __device__ __forceinline__ float most(const Piece (&all)[K]) {
        if constexpr (std::is_same<T, float>::value) {
            float m = all[0].most();
#pragma unroll
            for (int k = 1; k < K; ++k) m = max_nan(m, all[k].most());
            return m;
        } else {
            typedef typename Pair<T>::type P;
            P m[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w = all[0].word(i);
                m[i] = *reinterpret_cast<const P*>(&w);
            }
#pragma unroll
            for (int k = 1; k < K; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t w = all[k].word(i);
                    m[i] = __hmax2_nan(m[i], *reinterpret_cast<const P*>(&w));
                }
            const float2 f = pair_f32(__hmax2_nan(__hmax2_nan(m[0], m[1]), __hmax2_nan(m[2], m[3])));
            return max_nan(f.x, f.y);
        }
    }
    __device__ __forceinline__ float most() const {   // NaN where there is one
        if constexpr (std::is_same<T, float>::value) {
            return max_nan(max_nan(__uint_as_float(q.x), __uint_as_float(q.y)), max_nan(__uint_as_float(q.z), __uint_as_float(q.w)));
        } else {
            typedef typename Pair<T>::type P;
            const P* p = reinterpret_cast<const P*>(&q);
            const P a = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
            const float2 f = pair_f32(a);
            return max_nan(f.x, f.y);
        }
    }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {   // NaN where there is one
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
// Sums of two values over the warp: in the lanes of one half a's, of the other b's.
__device__ __forceinline__ void warp_sums(float& a, float& b) {
    const int lane = threadIdx.x & 31;
    float keep = lane < 16 ? a : b;
    keep += __shfl_xor_sync(0xffffffffu, lane < 16 ? b : a, 16);
#pragma unroll
    for (int d = 8; d; d >>= 1) keep += __shfl_xor_sync(0xffffffffu, keep, d);
    a = __shfl_sync(0xffffffffu, keep, 0);
    b = __shfl_sync(0xffffffffu, keep, 16);
}

// t = (x - m) log2(e) + delta in one multiply-add: delta, what the rounding of m
// log2(e) leaves, is the same for all of a row and taken out of its sums.  Scores
// so far below m that their exponential is 0 anyway (-inf among them, which would
// give 0 times infinity) are held at `bound`, 16-bit ones before they are widened:
// 140 or |m| / 64 below, which their own rounding leaves at least 100.
template <typename T> struct Exponents {
    float c, delta, whole;   // whole: 2^-delta
    uint32_t bound;
    bool fast;    // m is small enough for that, and far from the type's lowest (the same for a row)
    __device__ __forceinline__ explicit Exponents(float m) {
        c = -(m * kLog2e);
        delta = fmaf(m, kLog2e, c);
        whole = exp2_fast(-delta);
        fast = fabsf(m) < 1e6f;   // delta is below 2^-24 1.5 |m|
        if constexpr (sizeof(T) == 2) {
            typename Pair<T>::type b;
            const float low = m - fmaxf(140.f, fabsf(m) * (1.f / 64.f));
            pair_from(b, low, low);
            bound = *reinterpret_cast<const uint32_t*>(&b);
            if (std::is_same<T, __half>::value) fast = m > -60000.f && m < INFINITY;
        }
    }
    __device__ __forceinline__ uint64_t at(const Piece<T>& q, int i) const {   // of elements 2 i, 2 i + 1
        if constexpr (sizeof(T) == 2) {
            typedef typename Pair<T>::type P;
            const uint32_t w = q.word(i);
            const P held = __hmax2(*reinterpret_cast<const P*>(&w), *reinterpret_cast<const P*>(&bound));
            const float2 v = pair_f32(held);
            return fma2(pair_of(v.x, v.y), both(kLog2e), both(c));
        } else {
            const float2 v = q.pair(i);
            float a, b;
            pair_to(fma2(pair_of(v.x, v.y), both(kLog2e), both(c)), a, b);
            return pair_of(fmaxf(a, kLowest), fmaxf(b, kLowest));
        }
    }
};
__device__ __forceinline__ uint64_t exp2_pair(uint64_t t) {
    float a, b;
    pair_to(t, a, b);
    return pair_of(exp2_fast(a), exp2_fast(b));
}
__device__ __forceinline__ float both_added(uint64_t v) {
    float a, b;
    pair_to(v, a, b);
    return a + b;
}

// What a set of scores adds up to beside a largest score m: the exponentials of
// the scores below m, those times their exponents of 2, and the scores equal to m.
struct Sums {
    float below, weighted;
    int equal;
};

// The sums of all scores of the pieces, those equal to m with them.
template <typename T, int K>
__device__ __forceinline__ void add_all(Sums& s, const Piece<T> (&q)[K], const Exponents<T>& x, float m) {
    constexpr int kPairs = Piece<T>::kN / 2;
    if (x.fast) {
        uint64_t sum = 0ull, weighted = 0ull;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                const uint64_t t = x.at(q[k], i), e = exp2_pair(t);
                sum = add2(sum, e);
                weighted = fma2(e, t, weighted);
            }
        const float b = both_added(sum) * x.whole;
        s.below += b;
        s.weighted += fmaf(both_added(weighted), x.whole, -x.delta * b);
    } else {
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < 2 * kPairs; ++i) {
                const float2 v = q[k].pair(i / 2);
                const float t = fmaxf(((i % 2 ? v.y : v.x) - m) * kLog2e, kLowest), e = exp2_fast(t);
                s.below += e;
                s.weighted = fmaf(e, t, s.weighted);
            }
    }
}

// `own`: the largest of these scores.  The few threads that hold the largest of
// the row first take it out.
template <typename T, int K>
__device__ __forceinline__ void add_up(Sums& s, Piece<T> (&q)[K], float m, float own) {
    if (own == m) {
#pragma unroll
        for (int k = 0; k < K; ++k) s.equal += q[k].take(m);
    }
    add_all(s, q, Exponents<T>(m), m);
}

// A row's numbers from its sums, written by one thread.
struct Row {
    float m, s;
    bool empty, lost;   // -inf only; with a NaN or +inf
    __device__ __forceinline__ Row(float most, float below, int equal) : m(most) {
        empty = m == -INFINITY;
        lost = !(m < INFINITY);
        s = lost ? __int_as_float(0x7fffffff) : empty ? 0.f : log1pf(below + (float)(equal - 1));
    }
    __device__ __forceinline__ float logp(float x) const { return empty ? -INFINITY : (x - m) - s; }
    template <typename T>
    __device__ __forceinline__ void write(const LogpArgs& p, int64_t row, const T* x, const Sums& t, int label) const {
        p.stats[row] = make_float2(m, s);
        if (p.lse) p.lse[row] = m + s;
        if (p.entropy) p.entropy[row] = empty ? 0.f : s - t.weighted * kLn2 / (t.below + (float)t.equal);
        if (p.logp) p.logp[row] = label < 0 ? 0.f : logp(to_f32(x[label]));
    }
};

// ------------------------------------------------------------- the best alternatives

// Scores in order as unsigned numbers (-0 as 0, NaN below all), the class behind
// them so that of equal scores the lowest class is the greatest.  0: none.
__device__ __forceinline__ uint64_t ranked(float v, int64_t j) {
    const unsigned b = __float_as_uint(v + 0.f);
    const unsigned u = v != v ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return (uint64_t)u << 32 | (unsigned)~(unsigned)j;
}
__device__ __forceinline__ int class_of(uint64_t key) { return (int)~(unsigned)key; }
__device__ __forceinline__ float score_of(uint64_t key) {
    const unsigned u = (unsigned)(key >> 32);
    return u == 0 ? __int_as_float(0x7fffffff) : __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint64_t warp_best(uint64_t v) {
    const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(v >> 32));
    const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(v >> 32) == hi ? (unsigned)v : 0u);
    return (uint64_t)hi << 32 | lo;
}

// The `top` best of `count` distinct keys, out[i] the i-th; by a warp.
__device__ __forceinline__ void in_order(uint64_t* out, const uint64_t* keys, int count, int top) {
    for (int i = threadIdx.x & 31; i < count; i += 32) {
        const uint64_t mine = keys[i];
        int greater = 0;
#pragma unroll 4
        for (int j = 0; j < count; ++j) greater += keys[j] > mine;
        if (greater < top) out[greater] = mine;
    }
}

constexpr int kWarpRoom = 96;   // candidates of a warp, and a list so far

// Bits of a lane's scores that are at least `bound` (closed places are not).
template <typename T, int K> struct Hits {
    static constexpr int kN = Piece<T>::kN;
    static_assert(4 * K <= 32, "two masks of 16 words");
    uint32_t lo = 0, hi = 0;   // 16-bit: words 0-15, 16-31, a bit of each half for either element of a word
    __device__ __forceinline__ Hits(const Piece<T> (&q)[K], float bound) {
        if constexpr (sizeof(T) == 2) {
            typedef typename Pair<T>::type P;
            P at;
            pair_from(at, bound, bound);
#pragma unroll
            for (int w = 0; w < 4 * K; ++w) {
                const uint32_t v = q[w / 4].word(w % 4);
                const uint32_t bits = __hge2_mask(*reinterpret_cast<const P*>(&v), at) & (0x10001u << (w & 15));
                if (w < 16) lo |= bits;
                else hi |= bits;
            }
        } else {
#pragma unroll
            for (int w = 0; w < 4 * K; ++w) lo |= (__uint_as_float(q[w / 4].word(w % 4)) >= bound ? 1u : 0u) << w;
        }
    }
    __device__ __forceinline__ bool some() const { return (lo | hi) != 0; }
    // One of them, taken out: element kN k + i.
    __device__ __forceinline__ int next() {
        if constexpr (sizeof(T) == 4) {
            const int b = __ffs(lo) - 1;
            lo &= lo - 1;
            return b;
        }
        const bool low = lo != 0;
        const uint32_t m = low ? lo : hi;
        const int b = __ffs(m) - 1;
        if (low) lo &= lo - 1;
        else hi &= hi - 1;
        return ((b & 15) + (low ? 0 : 16)) * 2 + (b >> 4);
    }
};

// The best by a bound: the scores that are at least the top-th largest of the
// lanes' largest ones hold them, and mostly they are few more.  With the list so far
// (null: none) in order to `out`; false where they are too many or too few.
// fetch(e): the lane's element e; element kN k + i is class first + k step + i.
template <typename T, int K, typename F>
__device__ __forceinline__ bool best_by_bound(uint64_t* out, const uint64_t* list, const Piece<T> (&q)[K], int first, int step, float own,
                                              int top, uint64_t* room, const F& fetch) {
    constexpr int kN = Piece<T>::kN;
    const int lane = threadIdx.x & 31;
    float bound = 0.f, v = own;
    for (int k = 0; k < top; ++k) {
        bound = warp_max(v);
        const unsigned at = __ballot_sync(0xffffffffu, v == bound);
        if (lane == __ffs(at) - 1) v = -INFINITY;
    }
    bound = fmaxf(bound, sizeof(T) == 4 ? -3.4028234e38f : std::is_same<T, __half>::value ? -65504.f : -3.3895314e38f);   // not -inf
    Hits<T, K> hits(q, bound);
    int count = 0;
    for (;;) {
        const bool some = hits.some();
        const unsigned at = __ballot_sync(0xffffffffu, some);
        if (!at || count > kWarpRoom) break;
        if (some) {
            const int e = hits.next(), to = count + __popc(at & ((1u << lane) - 1));
            if (to < kWarpRoom) room[to] = ranked(fetch(e), first + e / kN * step + e % kN);
        }
        count += __popc(at);
    }
    const int old = list ? top : 0;
    if (count + old > kWarpRoom || count + old < top) return false;
    if (lane < old) room[count + lane] = list[lane];
    __syncwarp();
    in_order(out, room, count + old, top);
    __syncwarp();
    return true;
}

// A lane's element e out of its registers.
template <typename T, int K> struct FromRegisters {
    const Piece<T> (&q)[K];
    __device__ __forceinline__ float operator()(int e) const {
        uint32_t w = q[0].word(0);
        const int at = sizeof(T) == 2 ? e / 2 : e;
#pragma unroll
        for (int i = 1; i < 4 * K; ++i) w = at == i ? q[i / 4].word(i % 4) : w;
        if constexpr (sizeof(T) == 4) return __uint_as_float(w);
        const uint16_t h = (uint16_t)(e % 2 ? w >> 16 : w);
        return to_f32(*reinterpret_cast<const T*>(&h));
    }
};

// The best key below `before` of the pieces first, first + step, .. < end of a row,
// read again: for rows whose scores are so alike (or so many -inf) that no bound
// keeps the candidates few.
template <typename T>
__device__ __forceinline__ uint64_t best_below(const LogpArgs& p, const T* x, int64_t first, int64_t step, int64_t end, uint64_t before) {
    constexpr int kN = Piece<T>::kN;
    uint64_t b = 0;
#pragma unroll 1
    for (; first < end; first += step) {
        Piece<T> q;
        q.load(x, first, end, lo_of<T>(p), hi_of<T>(p));
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int64_t j = first + i;
            const float2 f = q.pair(i / 2);
            const uint64_t v = j >= 0 && j < end ? ranked(i % 2 ? f.y : f.x, j) : 0;
            if (v < before && v > b) b = v;
        }
    }
    return b;
}

__device__ __forceinline__ void write_top(const LogpArgs& p, int64_t row, int place, uint64_t key, float m, float s) {
    p.top_ids[row * p.top + place] = class_of(key);
    p.top_logp[row * p.top + place] = m == -INFINITY ? -INFINITY : (score_of(key) - m) - s;
}

// ------------------------------------------------------------- a row by a warp
//
// Up to 32 neighbouring rows one after the other, the next one's loads under way;
// lane r keeps row r's sums, and the logarithms, quotients and stores of all of
// them are made together at the end (one by one they cost more than the
// exponentials of 256 classes).

constexpr int kWarpRows = 32;

// The best of 16-bit scores: class and score make a key of 32 bits, whose largest
// of the warp is one instruction; a lane's next largest is that of key - taken
// (mod 2^32, where those that were taken are smallest).  Up to two accesses a lane: 262144 x 256, 4 alternatives, 103 us,
// 120 by the bound above.
template <typename T, int K, bool kWhole>
__device__ __forceinline__ void best_of_16(uint64_t* out, const Piece<T> (&q)[K], int first, int n, int top) {
    typedef typename Pair<T>::type P;
    uint32_t key[8 * K];
    const P zero = {};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t raw = q[k].word(i);
            const P v = __hadd2(*reinterpret_cast<const P*>(&raw), zero);   // -0 as 0
            const uint32_t w = *reinterpret_cast<const uint32_t*>(&v);
            uint32_t u = w ^ (((w >> 15) & 0x00010001u) * 0xffffu | 0x80008000u);
            const int j = first + k * 256 + 2 * i;
            const uint32_t classes = (uint32_t)(0xfffe - j) << 16 | ((uint32_t)(0xffff - j) & 0xffffu);   // of both
            if (kWhole) {
                if (first + k * 256 >= n) u = 0;   // -inf has 0x7f or more
                key[8 * k + 2 * i] = __byte_perm(u, classes, 0x1054);
                key[8 * k + 2 * i + 1] = __byte_perm(u, classes, 0x3276);
            } else {
                key[8 * k + 2 * i] = (unsigned)j < (unsigned)n ? __byte_perm(u, classes, 0x1054) : 0u;
                key[8 * k + 2 * i + 1] = (unsigned)(j + 1) < (unsigned)n ? __byte_perm(u, classes, 0x3276) : 0u;
            }
        }
    uint32_t best = 0, mine = 0;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 8 * K; ++i) best = max(best, key[i]);
    for (int t = 0; t < top; ++t) {
        const uint32_t taken = __reduce_max_sync(0xffffffffu, best);
        if (lane == t) mine = taken;
        uint32_t left = 0;
#pragma unroll
        for (int i = 0; i < 8 * K; ++i) left = __viaddmax_u32(key[i], 0u - taken, left);
        left += taken;
        if (best == taken) best = left < taken ? left : 0u;   // another lane's best stays
    }
    if (lane < top) {
        const uint16_t u = (uint16_t)(mine >> 16), h = u & 0x8000 ? u ^ 0x8000 : ~u;
        out[lane] = ranked(to_f32(*reinterpret_cast<const T*>(&h)), 0xffff - (int)(mine & 0xffff));
    }
}

template <typename T, int K, bool kTop, bool kWhole>
__global__ void __launch_bounds__(128) k_logp_warp(const __grid_constant__ LogpArgs p, int rows_each) {
    __shared__ uint64_t room[4][kWarpRoom];
    extern __shared__ uint64_t staged[];   // [4][rows_each][top]
    constexpr int kN = Piece<T>::kN;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = p.n;
    uint64_t* best = staged + (size_t)warp * rows_each * p.top;
    const int64_t all = (p.rows + rows_each - 1) / rows_each;
    for (int64_t group = (int64_t)blockIdx.x * 4 + warp; group < all; group += (int64_t)gridDim.x * 4) {
        const int64_t base = group * rows_each;
        const int rows = p.rows - base < rows_each ? (int)(p.rows - base) : rows_each;
        const T* x = static_cast<const T*>(p.x) + base * n;
        Piece<T> q[K], next[K];
        int first = 0, first_next;
        const auto load = [&](int r) {
            const T* y = x + r * n;
            first_next = lane * kN - (kWhole ? 0 : Piece<T>::shift_of(y));
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int at = first_next + k * 32 * kN, end = r < rows ? n : -kN;
                if (kWhole) next[k].load_whole(y, at, end);
                else next[k].load(y, at, end, lo_of<T>(p), hi_of<T>(p));
            }
        };
        load(0);
        const int label = lane < rows && p.logp ? label_of(p, base + lane) : -1;
        float most = 0.f;
        Sums sums = {0.f, 0.f, 0};
        for (int r = 0; r < rows; ++r) {
#pragma unroll
            for (int k = 0; k < K; ++k) q[k] = next[k];
            first = first_next;
            load(r + 1);
            const float own = Piece<T>::most(q);
            const float m = warp_max(own);
            const bool plain = m < INFINITY && m > -INFINITY;
            if (kTop) {
                uint64_t* out = best + r * p.top;
                bool done = plain;
                if (plain) {
                    if constexpr (sizeof(T) == 2 && K <= 2) best_of_16<T, K, kWhole>(out, q, first, n, p.top);
                    else done = best_by_bound(out, nullptr, q, first, 32 * kN, own, p.top, room[warp], FromRegisters<T, K>{q});
                }
                if (!done) {
                    uint64_t before = ~0ull;
                    for (int k = 0; k < p.top; ++k) {
                        before = warp_best(best_below(p, x + r * n, first, 32 * kN, n, before));
                        if (lane == 0) out[k] = before;
                    }
                }
            }
            Sums t = {0.f, 0.f, 0};
            if (plain) {
                // The largest scores are added with the others; where little is left beside
                // one of them (the warp agrees), again without.
                add_all(t, q, Exponents<T>(m), m);
                warp_sums(t.below, t.weighted);
                t.below -= 1.f;
                t.equal = 1;
                if (t.below < 0.0625f) {
                    t = Sums{0.f, 0.f, 0};
                    add_up(t, q, m, own);
                    warp_sums(t.below, t.weighted);
                    t.equal = (int)__reduce_add_sync(0xffffffffu, (unsigned)t.equal);
                }
            }
            if (lane == r) {
                most = m;
                sums = t;
            }
        }
        const Row mine(most, sums.below, sums.equal);
        if (lane < rows) mine.write(p, base + lane, x + lane * n, sums, label);
        if (kTop) {
            __syncwarp();
            for (int i = 0; i < rows * p.top; i += 32) {
                const int e = i + lane, r = e / p.top;
                const float m = __shfl_sync(0xffffffffu, mine.m, r & 31), s = __shfl_sync(0xffffffffu, mine.s, r & 31);
                if (e < rows * p.top) write_top(p, base + r, e - r * p.top, best[e], m, s);
            }
            __syncwarp();
        }
    }
}

// ------------------------------------------------------------- a row by CTAs
//
// A CTA, or a cluster of per_row of them, goes through rows; each warp has a share
// of a row, kPieces accesses a lane, and knows no other warp's: it leaves the sums
// of its share relative to its own largest score, and its best alternatives, in
// shared memory, and goes on to the next row.  After kBatch rows the CTAs meet, and
// every row's shares are put together by a warp.  (Meeting twice a row, to share the
// largest score first, took 115 us for 8192 x 32768 and 281 for 2000 x 100003.)
//
// kAhead > 0: the next rows' accesses are under way as asynchronous copies, to
// places in shared memory that only the thread itself reads, so that they need no
// barrier.  kAhead 0: rows that no cluster holds; a warp takes its share in rounds.

constexpr int kBatch = 32, kTopBatch = 8;

__device__ __forceinline__ void copy16(uint4* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

// A share's largest score and its sums relative to it.
struct alignas(16) Share {
    float m;
    Sums sums;
    // Of both: the one with the smaller largest score is scaled to the other.
    __device__ __forceinline__ void join(const Share& o) {
        const Share &hi = o.m > m ? o : *this, &lo = o.m > m ? *this : o;
        Share r = hi;
        if (lo.m == hi.m) {
            r.sums.below += lo.sums.below;
            r.sums.weighted += lo.sums.weighted;
            r.sums.equal += lo.sums.equal;
        } else if (lo.m > -INFINITY) {
            const float t = fmaxf((lo.m - hi.m) * kLog2e, kLowest), e = exp2_fast(t), all = lo.sums.below + (float)lo.sums.equal;
            r.sums.below = fmaf(all, e, r.sums.below);
            r.sums.weighted += e * fmaf(t, all, lo.sums.weighted);
        }
        r.m = max_nan(m, o.m);
        *this = r;
    }
};

// The sums of a warp's pieces relative to m, its largest score: in all lanes.
template <typename T, int K>
__device__ __forceinline__ Sums warp_add_up(Piece<T> (&q)[K], float m, float own) {
    Sums t = {0.f, 0.f, 0};
    if (!(m < INFINITY && m > -INFINITY)) return t;
    // The largest scores are added with the others; where little is left beside one of
    // them (the warp agrees), again without.
    add_all(t, q, Exponents<T>(m), m);
    warp_sums(t.below, t.weighted);
    t.below -= 1.f;
    t.equal = 1;
    if (t.below < 0.0625f) {
        t = Sums{0.f, 0.f, 0};
        add_up(t, q, m, own);
        warp_sums(t.below, t.weighted);
        t.equal = (int)__reduce_add_sync(0xffffffffu, (unsigned)t.equal);
    }
    return t;
}

template <typename T, int kThreads, int kPieces, int kAhead, bool kTop>
__global__ void __launch_bounds__(kThreads, kThreads == 512 ? 2 : kThreads == 256 ? 3 : 6) k_logp_ctas(
    const __grid_constant__ LogpArgs p, int share, int rounds, int per_row) {
    constexpr bool kLoop = kAhead == 0;
    constexpr int kWarps = kThreads / 32, kN = Piece<T>::kN, step = 32 * kN, kRows = kTop ? kTopBatch : kBatch;
    extern __shared__ uint4 ring[];   // [kAhead][kPieces][kThreads], then keys [kRows][kWarps][top]
    __shared__ uint64_t room[kTop ? kWarps : 1][kWarpRoom];
    __shared__ Share shares[kRows][kWarps];
    __shared__ float2 stats[kTop ? kRows : 1];
    uint64_t* lists = reinterpret_cast<uint64_t*>(ring + kAhead * kPieces * kThreads);
    const cg::cluster_group cluster = cg::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = per_row > 1 ? (int)cluster.block_rank() : 0;
    const int64_t rows_at = gridDim.x / per_row, row0 = blockIdx.x / per_row;
    const auto row_of = [&](int64_t row) { return static_cast<const T*>(p.x) + row * p.n; };
    // The warp's share of a row: `share` accesses from a multiple of it on (a row's
    // classes are fewer than 2^30: offsets in it fit 32 bits).
    const int64_t begin = (int64_t)(rank * kWarps + warp) * share * kN;
    const auto start_of = [&](const T* x) { return (int)(begin < p.n + kN ? begin : p.n + kN) + lane * kN - Piece<T>::shift_of(x); };
    const auto end_of = [&](const T* x) {
        const int64_t e = begin + (int64_t)share * kN - Piece<T>::shift_of(x);
        return e < p.n ? (int)e : p.n;
    };
    const auto ahead = [&](int64_t row, int stage) {
        if (row < p.rows) {
            const T* x = row_of(row);
            const int first = start_of(x), end = end_of(x);
            uint4* to = ring + stage * kPieces * kThreads + threadIdx.x;
            if (first >= 0 && first + (kPieces - 1) * step + kN <= end) {
#pragma unroll
                for (int k = 0; k < kPieces; ++k) copy16(to + k * kThreads, x + first + k * step);
            } else {
#pragma unroll 1
                for (int k = 0; k < kPieces; ++k, to += kThreads) {
                    const int at = first + k * step;
                    if (at >= 0 && at + kN <= end) {
                        copy16(to, x + at);
                    } else {
                        Piece<T> q;
                        q.load(x, at, end, lo_of<T>(p), hi_of<T>(p));
                        *to = q.q;
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const auto meet = [&] {
        if (per_row > 1) cluster.sync();
        else __syncthreads();
    };
    const auto best_slowly = [&](uint64_t* out, const T* x, int first, int end) {
        uint64_t before = ~0ull;
        for (int k = 0; k < p.top; ++k) {
            before = warp_best(best_below(p, x, (int64_t)first, step, end, before));
            if (lane == 0) out[k] = before;
        }
        __syncwarp();
    };
    // The rows of a batch, row0 + (i0 + i) rows_at, every per_row-th of which is this CTA's:
    // a warp a row where there are enough, else a lane a row.  Then the alternatives, a warp a row.
    const auto finish = [&](int64_t i0, int n) {
        meet();
        const bool wide = n <= kWarps * per_row;
        if (wide || warp == 0) {
            const int i = (wide ? warp : lane) * per_row + rank;
            if (i < n) {
                const int64_t row = row0 + (i0 + i) * rows_at;
                const int label = p.logp ? label_of(p, row) : -1;
                Share all = {-INFINITY, {0.f, 0.f, 0}};
#pragma unroll 4
                for (int k = wide ? lane : 0; k < kWarps * per_row; k += wide ? 32 : 1) {
                    const Share* from = &shares[i][k % kWarps];
                    all.join(per_row > 1 ? *cluster.map_shared_rank(from, k / kWarps) : *from);
                }
                if (wide) {
#pragma unroll
                    for (int d = 16; d; d >>= 1) {
                        Share o;
                        o.m = __shfl_xor_sync(0xffffffffu, all.m, d);
                        o.sums.below = __shfl_xor_sync(0xffffffffu, all.sums.below, d);
                        o.sums.weighted = __shfl_xor_sync(0xffffffffu, all.sums.weighted, d);
                        o.sums.equal = __shfl_xor_sync(0xffffffffu, all.sums.equal, d);
                        all.join(o);
                    }
                }
                const Row done(all.m, all.sums.below, all.sums.equal);
                if (!wide || lane == 0) {
                    done.write(p, row, row_of(row), all.sums, label);
                    if (kTop) stats[i] = make_float2(done.m, done.s);
                }
            }
        }
        if constexpr (kTop) {
            __syncthreads();
            for (int i = warp * per_row + rank; i < n; i += kWarps * per_row) {
                // Lists that fall: the best of all is among their heads.
                const int many = kWarps * per_row;
                const uint64_t* from[4];
                uint64_t head[4];
                int taken[4] = {0, 0, 0, 0};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int k = lane + 32 * u;
                    from[u] = lists + (i * kWarps + k % kWarps) * p.top;
                    if (per_row > 1 && k < many) from[u] = cluster.map_shared_rank(from[u], k / kWarps);
                    head[u] = k < many ? from[u][0] : 0;
                }
                uint64_t mine = 0;
                for (int t = 0; t < p.top; ++t) {
                    uint64_t b = head[0];
#pragma unroll
                    for (int u = 1; u < 4; ++u) b = head[u] > b ? head[u] : b;
                    b = warp_best(b);
                    if (lane == t) mine = b;
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (head[u] == b && b) head[u] = ++taken[u] < p.top ? from[u][taken[u]] : 0;   // keys differ: one list
                }
                if (lane < p.top) write_top(p, row0 + (i0 + i) * rows_at, lane, mine, stats[i].x, stats[i].y);
            }
        }
        meet();
    };
    if (!kLoop) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ahead(row0 + i * rows_at, i);
    }
    int64_t it = 0;
    int held = 0;
    for (int64_t row = row0; row < p.rows; row += rows_at, ++it) {
        const T* x = row_of(row);
        const int start = start_of(x), end = end_of(x);
        uint64_t* out = lists + (held * kWarps + warp) * p.top;
        Piece<T> q[kPieces];
        Share all;
        if constexpr (kLoop) {
            all = Share{-INFINITY, {0.f, 0.f, 0}};
            bool listed = kTop;
            for (int round = 0; round < rounds; ++round) {
                const int first = start + round * kPieces * step;
#pragma unroll
                for (int k = 0; k < kPieces; ++k) q[k].load(x, first + k * step, end, lo_of<T>(p), hi_of<T>(p));
                const float own = Piece<T>::most(q);
                Share one;
                one.m = warp_max(own);
                if (listed && !(round && one.m == -INFINITY))
                    listed = one.m < INFINITY && best_by_bound(out, round ? out : nullptr, q, first, step, own, p.top, room[warp],
                                                               FromRegisters<T, kPieces>{q});
                one.sums = warp_add_up(q, one.m, own);
                all.join(one);
            }
            if (kTop && !listed) best_slowly(out, x, start, end);
        } else {
            constexpr int kSlots = kAhead > 0 ? kAhead : 1;
            const int slot = (int)(it % kSlots);
            asm volatile("cp.async.wait_group %0;" ::"n"(kSlots - 1) : "memory");
            const uint4* from = ring + slot * kPieces * kThreads + threadIdx.x;
#pragma unroll
            for (int k = 0; k < kPieces; ++k) q[k].q = from[k * kThreads];
            const float own = Piece<T>::most(q);
            all.m = warp_max(own);
            if (kTop) {
                const auto fetch = [&](int e) { return to_f32(reinterpret_cast<const T*>(from + e / kN * kThreads)[e % kN]); };
                if (!(all.m < INFINITY && all.m > -INFINITY) ||
                    !best_by_bound(out, nullptr, q, start, step, own, p.top, room[warp], fetch))
                    best_slowly(out, x, start, end);
            }
            ahead(row + kSlots * rows_at, slot);   // the places have been read
            all.sums = warp_add_up(q, all.m, own);
        }
        if (lane == 0) shares[held][warp] = all;
        if (++held == kRows) {
            finish(it - held + 1, held);
            held = 0;
        }
    }
    if (held) finish(it - held, held);
}

// ------------------------------------------------------------- few classes

// A thread a row, up to 256 bytes of classes: 858914 x 73 in float16 with 3
// alternatives 126 us, a warp a row 390; 198959 x 48 in float32 with 20, for each of
// which a thread looks through its row again, 113 us and 267.
constexpr int kFewBytes = 256, kTileRows = 128;

// A tile of rows lies in memory as one stretch: 16 bytes at a time (its start
// allows that when the tensor's does) to shared memory, where rows are `pitch`
// apart, so that a thread a row meets few others in its banks: an odd number of
// words, or a word and a half more or less.
template <typename T> __host__ __device__ inline int pitch_of(int n) {
    return sizeof(T) == 4 ? n | 1 : n % 4 == 0 ? n + 2 : n;
}

struct Place {   // of an element of a tile: at most 128 x 128 of them, so the quotient is exact
    int row, j;
    __device__ __forceinline__ Place(int i, int n) {
        row = (int)(((unsigned)i * ((1u << 22) / (unsigned)n + 1u)) >> 22);
        j = i - row * n;
    }
    __device__ __forceinline__ void next(int n) {
        if (++j == n) j = 0, ++row;
    }
};

// kIn: memory to tile, else back.
template <typename T, bool kIn>
__device__ __forceinline__ void tile_copy(T* tile, T* x, int count, int n, bool vec) {
    constexpr int kN = 16 / (int)sizeof(T);
    const int pitch = pitch_of<T>(n);
    const int whole = vec ? count / kN : 0;
    for (int i = threadIdx.x; i < whole; i += kTileRows) {
        if (pitch == n) {
            if (kIn) copy16(reinterpret_cast<uint4*>(tile) + i, reinterpret_cast<const uint4*>(x) + i);
            else reinterpret_cast<uint4*>(x)[i] = reinterpret_cast<const uint4*>(tile)[i];
            continue;
        }
        union { uint4 u; T e[kN]; } r;
        Place at(i * kN, n);
        if (kIn) r.u = reinterpret_cast<const uint4*>(x)[i];
#pragma unroll
        for (int k = 0; k < kN; ++k, at.next(n)) {
            if (kIn) tile[at.row * pitch + at.j] = r.e[k];
            else r.e[k] = tile[at.row * pitch + at.j];
        }
        if (!kIn) reinterpret_cast<uint4*>(x)[i] = r.u;
    }
    for (int i = whole * kN + threadIdx.x; i < count; i += kTileRows) {
        const Place at(i, n);
        if (kIn) tile[at.row * pitch + at.j] = x[i];
        else x[i] = tile[at.row * pitch + at.j];
    }
    if (kIn) asm volatile("cp.async.wait_all;" ::: "memory");
}

// f(x, j) of a row's classes in order; 16-bit ones two at a time where n is even (rows
// then begin on words).  Four steps' classes are read together.
template <typename T, typename F> __device__ __forceinline__ void each_class(const T* x, int n, const F& f) {
    if (sizeof(T) == 2 && n % 2 == 0) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(x);
#pragma unroll 4
        for (int j = 0; j < n; j += 2, ++w) {
            Vec<T, 2> v;
            v.r.w[0] = *w;
            f(v.at(0), j);
            f(v.at(1), j + 1);
        }
    } else {
#pragma unroll 4
        for (int j = 0; j < n; ++j) f(to_f32(x[j]), j);
    }
}

template <typename T>
__global__ void __launch_bounds__(kTileRows) k_logp_few(const __grid_constant__ LogpArgs p, bool vec) {
    extern __shared__ uint4 memory[];
    T* tile = reinterpret_cast<T*>(memory);
    for (int64_t base = (int64_t)blockIdx.x * kTileRows; base < p.rows; base += (int64_t)gridDim.x * kTileRows) {
        const int rows = p.rows - base < kTileRows ? (int)(p.rows - base) : kTileRows, n = p.n;
        const int64_t row = base + threadIdx.x;
        const bool here = (int)threadIdx.x < rows;
        const int label = here && p.logp ? label_of(p, row) : -1;
        tile_copy<T, true>(tile, const_cast<T*>(static_cast<const T*>(p.x)) + base * n, rows * n, n, vec);
        __syncthreads();
        if (here) {
            const T* x = tile + threadIdx.x * pitch_of<T>(n);
            float m = -INFINITY;
            each_class(x, n, [&](float v, int) { m = max_nan(m, v); });
            const bool plain = m < INFINITY && m > -INFINITY;
            Sums t = {0.f, 0.f, 0};
            if (plain)
                each_class(x, n, [&](float v, int) {
                    const float d = v - m, e2 = fmaxf(d * kLog2e, kLowest), e = exp2_fast(e2);
                    t.equal += d == 0.f;
                    t.below += d == 0.f ? 0.f : e;
                    t.weighted = fmaf(e, e2, t.weighted);
                });
            const Row done(m, t.below, t.equal);
            done.write(p, row, x, t, label);
            float value = INFINITY;   // of the alternative before, and its class
            int at = -1;
            uint64_t before = ~0ull;
            for (int k = 0; k < p.top; ++k) {
                if (plain) {
                    float b = -INFINITY;
                    int j = n;
                    each_class(x, n, [&](float v, int i) {
                        const bool left = v < value || (v == value && i > at);
                        if (left && (v > b || j == n)) b = v, j = i;
                    });
                    value = b;
                    at = j;
                } else {
                    uint64_t b = 0;
                    each_class(x, n, [&](float v, int i) {
                        const uint64_t r = ranked(v, i);
                        if (r < before && r > b) b = r;
                    });
                    before = b;
                    value = score_of(b);
                    at = class_of(b);
                }
                p.top_ids[row * p.top + k] = at;
                p.top_logp[row * p.top + k] = done.logp(value);
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------- the gradient

// What the elements of a row have in common: p (all - ge log p), and gl more at
// the label.
struct RowGrad {
    float m, s, all, ge, gl;
    float rest;   // of all without gl: at the label
    int label;
    __device__ __forceinline__ RowGrad(const LogpArgs& p, int64_t row) {
        const float2 st = p.stats[row];
        m = st.x;
        s = st.y;
        label = p.gl ? label_of(p, row) : -1;
        gl = label >= 0 ? p.gl[row] : 0.f;
        ge = p.ge ? p.ge[row] : 0.f;
        rest = (p.gz ? p.gz[row] : 0.f) - (p.ge ? ge * p.entropy[row] : 0.f);
        all = rest - gl;
    }
    // The label's own 1 - p would lose what a confident answer leaves.
    __device__ __forceinline__ float at_label(float x) const {
        const float lp = (x - m) - s, t = max_nan(lp * kLog2e, kLowest);
        return m == -INFINITY ? 0.f : fmaf(exp2_fast(t), fmaf(-ge * kLn2, t, rest), -gl * expm1f(lp));
    }
    __device__ __forceinline__ float at(float x) const {
        const float t = max_nan(((x - m) - s) * kLog2e, kLowest);   // NaN of a row that has one stays
        return m == -INFINITY ? 0.f : exp2_fast(t) * fmaf(-ge * kLn2, t, all);
    }
};

// The gradients of a piece at class `at` of its row.  log2 p = t - kappa with t of
// Exponents and kappa = delta + s log2(e), so that p (all - ge log p) = 2^t (a + b t).
template <typename T> struct PieceGrad {
    static constexpr int kN = Piece<T>::kN;
    RowGrad g;
    Exponents<T> x;
    float a, b;
    __device__ __forceinline__ explicit PieceGrad(const RowGrad& g_) : g(g_), x(g_.m) {
        const float kappa = fmaf(g.s, kLog2e, x.delta), f = exp2_fast(-kappa), e = g.ge * kLn2;
        a = f * fmaf(e, kappa, g.all);
        b = -f * e;
    }
    __device__ __forceinline__ void of(float (&v)[kN], const Piece<T>& q, int64_t at) const {
        if (x.fast) {
#pragma unroll
            for (int i = 0; i < kN / 2; ++i) {
                const uint64_t t = x.at(q, i);
                pair_to(mul2(exp2_pair(t), fma2(t, both(b), both(a))), v[2 * i], v[2 * i + 1]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const float2 f = q.pair(i / 2);
                v[i] = g.at(i % 2 ? f.y : f.x);
            }
        }
        const int64_t l = g.label - at;
        if (l >= 0 && l < kN && g.label >= 0) {
            float own = 0.f;
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const float2 f = q.pair(i / 2);
                own = i == l ? (i % 2 ? f.y : f.x) : own;
            }
            own = g.at_label(own);
#pragma unroll
            for (int i = 0; i < kN; ++i) v[i] = i == l ? own : v[i];
        }
    }
};

// `whole`: all of the piece is in the row and the gradient's row lies as the scores' does.
template <typename T>
__device__ __forceinline__ void store_piece(T* gx, const float (&v)[Piece<T>::kN], int64_t at, int64_t n, bool whole) {
    constexpr int kN = Piece<T>::kN;
    if (whole) {
        Vec<T, kN> o;
        o.from(v);
        o.store(gx + at);
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (at + i >= 0 && at + i < n) gx[at + i] = from_f32<T>(v[i]);
    }
}

template <typename T>
__global__ void __launch_bounds__(kTileRows) k_logp_few_grad(const __grid_constant__ LogpArgs p, bool vec, bool vec_out) {
    extern __shared__ uint4 memory[];
    T* tile = reinterpret_cast<T*>(memory);
    for (int64_t base = (int64_t)blockIdx.x * kTileRows; base < p.rows; base += (int64_t)gridDim.x * kTileRows) {
        const int rows = p.rows - base < kTileRows ? (int)(p.rows - base) : kTileRows, n = p.n;
        tile_copy<T, true>(tile, const_cast<T*>(static_cast<const T*>(p.x)) + base * n, rows * n, n, vec);
        __syncthreads();
        if ((int)threadIdx.x < rows) {
            const RowGrad g(p, base + threadIdx.x);
            T* x = tile + threadIdx.x * pitch_of<T>(n);
            const float label = g.label >= 0 ? to_f32(x[g.label]) : 0.f;
            for (int j = 0; j < n; ++j) x[j] = from_f32<T>(g.at(to_f32(x[j])));
            if (g.label >= 0) x[g.label] = from_f32<T>(g.at_label(label));
        }
        __syncthreads();
        tile_copy<T, false>(tile, static_cast<T*>(p.gx) + base * n, rows * n, n, vec_out);
        __syncthreads();
    }
}

// A warp a row, up to 32 neighbouring ones after another; lane r reads what row r's
// elements have in common.  kAtOnce accesses are under way together.
constexpr int kAtOnce = 4;

template <typename T, bool kWhole>
__global__ void __launch_bounds__(128) k_logp_grad_warp(const __grid_constant__ LogpArgs p, int rows_each, int pieces, bool same) {
    constexpr int kN = Piece<T>::kN;
    const int lane = threadIdx.x & 31, n = p.n;
    const int64_t all = (p.rows + rows_each - 1) / rows_each;
    for (int64_t group = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); group < all; group += (int64_t)gridDim.x * 4) {
        const int64_t base = group * rows_each;
        const int rows = p.rows - base < rows_each ? (int)(p.rows - base) : rows_each;
        const T* x = static_cast<const T*>(p.x) + base * n;
        T* gx = static_cast<T*>(p.gx) + base * n;
        const RowGrad own(p, base + (lane < rows ? lane : rows - 1));
        const int count = rows * pieces;   // piece i: of row i / pieces
        for (int i0 = 0, r0 = 0, k0 = 0; i0 < count; i0 += kAtOnce) {
            Piece<T> q[kAtOnce];
            int row[kAtOnce], at[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const T* y = x + r0 * n;
                row[u] = r0;
                at[u] = (k0 * 32 + lane) * kN - (kWhole ? 0 : Piece<T>::shift_of(y));
                const int end = r0 < rows ? n : -kN;
                if (kWhole) q[u].load_whole(y, at[u], end);
                else q[u].load(y, at[u], end, lo_of<T>(p), hi_of<T>(p));
                if (++k0 == pieces) k0 = 0, ++r0;
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                if (row[u] >= rows) break;
                RowGrad g = own;
                g.m = __shfl_sync(0xffffffffu, own.m, row[u]);
                g.s = __shfl_sync(0xffffffffu, own.s, row[u]);
                g.all = __shfl_sync(0xffffffffu, own.all, row[u]);
                g.ge = __shfl_sync(0xffffffffu, own.ge, row[u]);
                g.gl = __shfl_sync(0xffffffffu, own.gl, row[u]);
                g.rest = __shfl_sync(0xffffffffu, own.rest, row[u]);
                g.label = __shfl_sync(0xffffffffu, own.label, row[u]);
                float v[kN];
                PieceGrad<T>(g).of(v, q[u], at[u]);
                if (at[u] < n)
                    store_piece<T>(gx + row[u] * n, v, at[u], n, same && (kWhole || (at[u] >= 0 && at[u] + kN <= n)));
            }
        }
    }
}

// A CTA a share of a row: kAtOnce accesses a thread (8192 x 32768 in bfloat16: 209 us with
// 10 CTAs of 128 threads an SM, 216 with 4 of 256).
constexpr int kShareThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kShareThreads, 10) k_logp_grad(const __grid_constant__ LogpArgs p, int64_t shares, bool same) {
    constexpr int kN = Piece<T>::kN;
    const int64_t all = p.rows * shares;
    for (int64_t share = blockIdx.x; share < all; share += gridDim.x) {
        const int64_t row = all >> 32 ? share / shares : (unsigned)share / (unsigned)shares;
        const T* x = static_cast<const T*>(p.x) + row * p.n;
        const int64_t first = ((share - row * shares) * (kShareThreads * kAtOnce) + threadIdx.x) * kN - Piece<T>::shift_of(x), n = p.n;
        Piece<T> q[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) q[k].load(x, first + k * kShareThreads * kN, n, lo_of<T>(p), hi_of<T>(p));
        const PieceGrad<T> g(RowGrad(p, row));
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const int64_t at = first + k * kShareThreads * kN;
            if (at >= n) break;
            float v[kN];
            g.of(v, q[k], at);
            store_piece<T>(static_cast<T*>(p.gx) + row * n, v, at, n, same && at >= 0 && at + kN <= n);
        }
    }
}

// ------------------------------------------------------------------ host side

template <typename T> static bool whole_rows(const LogpArgs& a) { return a.n % Piece<T>::kN == 0 && aligned16(a.x); }
template <typename T> static int64_t vectors_of(const LogpArgs& a) {   // of a row, wherever it begins
    return ceil_div((int64_t)a.n + (whole_rows<T>(a) ? 0 : Piece<T>::kN - 1), Piece<T>::kN);
}

static unsigned grid_of(int64_t ctas) { return (unsigned)(ctas < (1 << 30) ? ctas : 1 << 30); }

// As many CTAs as are resident at a time (in clusters of per_row).
template <typename T, int kThreads, int kPieces, int kAhead, bool kTop>
static cudaError_t launch_ctas(const LogpArgs& a, int64_t nv, int per_row, cudaStream_t s) {
    const auto kernel = k_logp_ctas<T, kThreads, kPieces, kAhead, kTop>;
    constexpr int kRing = kAhead * kPieces * kThreads * 16, kLists = kTop ? kTopBatch * (kThreads / 32) * 8 : 0;   // keys: times top
    const int share = (int)ceil_div(ceil_div(nv, per_row * (kThreads / 32)), 32) * 32;   // accesses of a warp
    const size_t smem = kRing + (size_t)kLists * a.top;
    int resident = 1;
    cudaError_t e = pl::kernel_once(
        reinterpret_cast<const void*>(kernel),
        [](int*) {
            return cudaFuncSetAttribute(k_logp_ctas<T, kThreads, kPieces, kAhead, kTop>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        kRing + kLists * PLATTICE_MAX_TOP);
        },
        &resident);
    if (e == cudaSuccess && a.rows * per_row > sm_count())
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, kThreads, smem);
    if (e != cudaSuccess) return e;
    int64_t rows = (int64_t)(resident > 0 ? resident : 1) * sm_count() / per_row;   // few rows: one CTA an SM, at most
    if (rows < 1) rows = 1;
    if (rows > a.rows) rows = a.rows;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((unsigned)(rows * per_row));
    c.blockDim = dim3(kThreads);
    c.dynamicSmemBytes = smem;
    c.stream = s;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)per_row;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    c.attrs = &attr;
    c.numAttrs = per_row > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&c, kernel, a, share, (int)ceil_div(share, kPieces * 32), per_row);
}

template <typename T, int kThreads, int kPieces, int kAhead>
static cudaError_t launch_ctas(const LogpArgs& a, int64_t nv, int per_row, cudaStream_t s) {
    return a.top ? launch_ctas<T, kThreads, kPieces, kAhead, true>(a, nv, per_row, s)
                 : launch_ctas<T, kThreads, kPieces, kAhead, false>(a, nv, per_row, s);
}

// Rows a warp takes one after the other: as many as give whole rounds of the CTAs
// (of 4 warps) that are resident at a time, `most` at most.
template <typename F> static cudaError_t rows_each(int* each, F* kernel, size_t smem, int64_t rows, int most) {
    int resident = 0;
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, 128, smem);
    const int64_t warps = 4 * (int64_t)sm_count() * (resident > 0 ? resident : 1), rounds = ceil_div(rows, warps * most);
    *each = (int)ceil_div(rows, warps * rounds);
    return e;
}

template <typename T, int K, bool kTop>
static cudaError_t launch_warp(const LogpArgs& a, cudaStream_t s) {
    const auto kernel = whole_rows<T>(a) ? k_logp_warp<T, K, kTop, true> : k_logp_warp<T, K, kTop, false>;
    int each = 0;
    const cudaError_t e = rows_each(&each, kernel, (size_t)4 * kWarpRows * a.top * 8, a.rows, kWarpRows);
    if (e != cudaSuccess) return e;
    kernel<<<grid_of(ceil_div(a.rows, 4 * each)), 128, (size_t)4 * each * a.top * 8, s>>>(a, each);
    return cudaGetLastError();
}
template <typename T, int K>
static cudaError_t launch_warp(const LogpArgs& a, cudaStream_t s) {
    return a.top ? launch_warp<T, K, true>(a, s) : launch_warp<T, K, false>(a, s);
}

template <typename T>
cudaError_t logp_forward(const LogpArgs& a, cudaStream_t s) {
    if (a.n * sizeof(T) <= kFewBytes) {
        k_logp_few<T><<<grid_of(ceil_div(a.rows, kTileRows)), kTileRows, kTileRows * pitch_of<T>(a.n) * sizeof(T), s>>>(
            a, aligned16(a.x));
        return cudaGetLastError();
    }
    const int64_t nv = vectors_of<T>(a);
    if (nv <= 32) return launch_warp<T, 1>(a, s);
    if (nv <= 64) return launch_warp<T, 2>(a, s);
    if (nv <= 96) return launch_warp<T, 3>(a, s);
    if (nv <= 128) return launch_warp<T, 4>(a, s);
    if (nv <= 160) return launch_warp<T, 5>(a, s);
    // The smallest cluster that holds the row; a larger one where the rows leave SMs without work.
    int per_row = 1;
    while (per_row < 8 && (nv > 4096 * (int64_t)per_row || (a.rows * per_row * 2 <= sm_count() && nv >= 1024 * (int64_t)per_row)))
        per_row *= 2;
    const int64_t share = ceil_div(nv, per_row);
    if (share <= 512) return launch_ctas<T, 128, 4, 3>(a, nv, per_row, s);
    if (share <= 1024) return launch_ctas<T, 128, 8, 2>(a, nv, per_row, s);
    if (share <= 2048) return launch_ctas<T, 256, 8, 2>(a, nv, per_row, s);
    if (share <= 4096) return launch_ctas<T, 512, 8, 1>(a, nv, per_row, s);
    return launch_ctas<T, 512, 8, 0>(a, nv, per_row, s);
}

template <typename T>
cudaError_t logp_backward(const LogpArgs& a, cudaStream_t s) {
    if (a.n * sizeof(T) <= kFewBytes) {
        k_logp_few_grad<T><<<grid_of(ceil_div(a.rows, kTileRows)), kTileRows, kTileRows * pitch_of<T>(a.n) * sizeof(T), s>>>(
            a, aligned16(a.x), aligned16(a.gx));
        return cudaGetLastError();
    }
    const int64_t nv = vectors_of<T>(a);
    const bool same = (((uintptr_t)a.x ^ (uintptr_t)a.gx) & 15) == 0;
    if (nv <= 512) {
        const auto kernel = whole_rows<T>(a) ? k_logp_grad_warp<T, true> : k_logp_grad_warp<T, false>;
        int each = 0;
        const cudaError_t e = rows_each(&each, kernel, 0, a.rows, 32);
        if (e != cudaSuccess) return e;
        kernel<<<grid_of(ceil_div(a.rows, 4 * each)), 128, 0, s>>>(a, each, (int)ceil_div(nv, 32), same);
    } else {
        const int64_t shares = ceil_div(nv, kShareThreads * kAtOnce);
        k_logp_grad<T><<<grid_of(a.rows * shares), kShareThreads, 0, s>>>(a, shares, same);
    }
    return cudaGetLastError();
}

}  // namespace plr
