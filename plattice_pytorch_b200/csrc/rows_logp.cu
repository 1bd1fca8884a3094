// rows_logp.cu -- log probabilities of given labels, entropy and the best
// alternatives of rows of scores, and the scores' gradient.
//
//   m = max x, s = log sum exp(x - m);  log p_j = (x_j - m) - s
//   entropy = -sum p log p = s - sum exp(x - m) (x - m) / sum exp(x - m)
//   grad_j = g_l ([j = label] - p_j) - g_e p_j (log p_j + entropy) + g_z p_j
//
// m and s are kept apart: their sum would lose s beside a large m (rows whose
// scores are all the type's lowest value, say).  The sum leaves one 1 of the
// largest score out, so that s = log1p(rest) and the log probability of a
// confident answer keep their precision.
//
// A row is read once and held: few classes by a thread out of shared memory,
// up to kWarpVectors accesses a lane by a warp in registers, more by a CTA or a
// cluster of them in registers, and only rows that no cluster holds are read
// again.  So the largest score is known before the first exponential, which
// costs a subtraction, a product, a bound, the exponential and two sums (five
// instructions an element in pairs; the special function unit takes one element
// in 16 a clock and SM, 60 us for the 268 M of 8192 x 32768, which take 83 us to
// read).
#include <cooperative_groups.h>

#include "plattice_runtime.h"
#include "rows_host.h"
#include "rows_vec.cuh"

namespace plr {

namespace cg = cooperative_groups;

struct LogpArgs {
    const void* x;
    Labels labels;         // p null: none
    float *logp, *entropy;
    float2* stats;
    float* lse;
    float* top_logp;
    long long* top_ids;
    const float *gl, *ge, *gz;
    void* gx;
    int64_t rows;
    int n, top;
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -200.f;   // of an exponent of 2: beyond it the exponential is 0

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
    __device__ __forceinline__ void load(const T* x, int64_t first, int n) {
        if (first >= 0 && first + kN <= n) {
            q = *reinterpret_cast<const uint4*>(x + first);
        } else {
            q = make_uint4(closed(), closed(), closed(), closed());
            if (first > -kN && first < n) {
                union { uint4 u; T e[kN]; } r;
                r.u = q;
#pragma unroll
                for (int i = 0; i < kN; ++i)
                    if (first + i >= 0 && first + i < n) r.e[i] = x[first + i];
                q = r.u;
            }
        }
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

// What a set of scores adds up to beside a largest score m: the exponentials of
// the scores below m, those times their exponents of 2, and the scores equal to m.
struct Sums {
    float below, weighted;
    int equal;
};

template <typename T, int K>
__device__ __forceinline__ void add_up(Sums& s, const Piece<T> (&q)[K], float m, float own) {
    constexpr int kPairs = Piece<T>::kN / 2;
    const uint64_t minus = both(-m), scale = both(kLog2e);
    if (own < m) {   // no score of this thread's is the largest
        uint64_t sum = 0ull, weighted = 0ull;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                const float2 v = q[k].pair(i);
                float a, b;
                pair_to(mul2(add2(pair_of(v.x, v.y), minus), scale), a, b);
                a = fmaxf(a, kLowest);
                b = fmaxf(b, kLowest);
                const uint64_t e = pair_of(exp2_fast(a), exp2_fast(b));
                sum = add2(sum, e);
                weighted = fma2(e, pair_of(a, b), weighted);
            }
        float a, b;
        pair_to(sum, a, b);
        s.below += a + b;
        pair_to(weighted, a, b);
        s.weighted += a + b;
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < 2 * kPairs; ++i) {
                const float2 v = q[k].pair(i / 2);
                const float d = (i % 2 ? v.y : v.x) - m, t = fmaxf(d * kLog2e, kLowest), e = exp2_fast(t);
                if (d == 0.f) {
                    ++s.equal;
                } else {
                    s.below += e;
                    s.weighted = fmaf(e, t, s.weighted);
                }
            }
    }
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
    __device__ __forceinline__ void write(const LogpArgs& p, int64_t row, const T* x, const Sums& t) const {
        p.stats[row] = make_float2(m, s);
        if (p.lse) p.lse[row] = m + s;
        if (p.entropy) p.entropy[row] = empty ? 0.f : s - t.weighted * kLn2 / (t.below + (float)t.equal);
        if (p.logp) {
            const int l = p.labels.at(row, p.n);
            p.logp[row] = l < 0 ? 0.f : logp(to_f32(x[l]));
        }
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

constexpr int kCandidates = 96;   // of a warp

// The `top` best of `count` keys in shared memory: lane i gets the i-th (0 where
// there are fewer).
__device__ __forceinline__ uint64_t best_of(const uint64_t* keys, int count, int top) {
    const int lane = threadIdx.x & 31;
    uint64_t mine = 0, before = ~0ull;
    for (int k = 0; k < top; ++k) {
        uint64_t b = 0;
        for (int i = lane; i < count; i += 32) {
            const uint64_t v = keys[i];
            if (v < before && v > b) b = v;
        }
        before = warp_best(b);
        if (lane == k) mine = before;
    }
    return mine;
}

// The `top` best of a warp's pieces (element i of piece k is class first + k step
// + i) and of a list from before, held as the result.  The scores that are at
// least the top-th largest of the lanes' own largest ones hold them all; mostly
// they are few more, and only they are put in order.
template <typename T, int K>
__device__ __forceinline__ uint64_t best_of_pieces(const Piece<T> (&q)[K], int64_t first, int64_t step, int n, float own, bool plain,
                                                   int top, uint64_t list, uint64_t* room, int* count) {
    constexpr int kN = Piece<T>::kN;
    const int lane = threadIdx.x & 31;
    if (plain) {
        float bound = 0.f, v = own;
        for (int k = 0; k < top; ++k) {
            bound = warp_max(v);
            const unsigned at = __ballot_sync(0xffffffffu, v == bound);
            if (lane == __ffs(at) - 1) v = -INFINITY;
        }
        if (lane == 0) *count = 0;
        __syncwarp();
        if (bound > -INFINITY) {
            if (own >= bound) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (!(q[k].most() >= bound)) continue;
#pragma unroll
                    for (int i = 0; i < kN; ++i) {
                        const float2 f = q[k].pair(i / 2);
                        const float x = i % 2 ? f.y : f.x;
                        if (x >= bound) {   // never outside the row
                            const int at = atomicAdd(count, 1);   // in any order: all keys differ
                            if (at < kCandidates) room[at] = ranked(x, first + k * step + i);
                        }
                    }
                }
            }
            __syncwarp();
            const int c = *count;
            if (c + 32 <= kCandidates) {
                room[c + lane] = list;
                __syncwarp();
                const uint64_t got = best_of(room, c + 32, top);
                __syncwarp();
                return got;
            }
        }
        __syncwarp();
    }
    uint64_t mine = 0, before = ~0ull;
    for (int t = 0; t < top; ++t) {
        uint64_t b = list < before ? list : 0;
#pragma unroll 1
        for (int k = 0; k < K; ++k) {
            Piece<T> piece = q[0];
#pragma unroll
            for (int o = 1; o < K; ++o)
                if (o == k) piece = q[o];
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int64_t j = first + k * step + i;
                const float2 f = piece.pair(i / 2);
                const uint64_t v = j >= 0 && j < n ? ranked(i % 2 ? f.y : f.x, j) : 0;
                if (v < before && v > b) b = v;
            }
        }
        before = warp_best(b);
        if (lane == t) mine = before;
    }
    return mine;
}

__device__ __forceinline__ void write_top(const LogpArgs& p, int64_t row, const Row& r, uint64_t mine) {
    const int lane = threadIdx.x & 31;
    if (lane < p.top) {
        p.top_ids[row * p.top + lane] = class_of(mine);
        p.top_logp[row * p.top + lane] = r.logp(score_of(mine));
    }
}

// ------------------------------------------------------------- a row by a warp

constexpr int kWarpVectors = 5;

template <typename T, int K, int kRows>
__global__ void __launch_bounds__(256) k_logp_warp(const __grid_constant__ LogpArgs p) {
    __shared__ uint64_t room[8][kCandidates];
    __shared__ int count[8];
    constexpr int kN = Piece<T>::kN;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t base = ((int64_t)blockIdx.x * 8 + warp) * kRows; base < p.rows; base += (int64_t)gridDim.x * 8 * kRows) {
        Piece<T> q[kRows][K];
        int64_t first[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const T* x = static_cast<const T*>(p.x) + (base + r) * p.n;
            first[r] = (int64_t)lane * kN - Piece<T>::shift_of(x);
            const int n = base + r < p.rows ? p.n : 0;
#pragma unroll
            for (int k = 0; k < K; ++k) q[r][k].load(x, first[r] + k * 32 * kN, n);
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int64_t row = base + r;
            if (row >= p.rows) break;
            float own = q[r][0].most();
#pragma unroll
            for (int k = 1; k < K; ++k) own = max_nan(own, q[r][k].most());
            const float m = warp_max(own);
            const bool plain = m < INFINITY && m > -INFINITY;
            Sums t = {0.f, 0.f, 0};
            if (plain) {
                add_up(t, q[r], m, own);
                warp_sums(t.below, t.weighted);
                t.equal = (int)__reduce_add_sync(0xffffffffu, (unsigned)t.equal);
            }
            const Row done(m, t.below, t.equal);
            if (lane == 0) done.write(p, row, static_cast<const T*>(p.x) + row * p.n, t);
            if (p.top)
                write_top(p, row, done, best_of_pieces(q[r], first[r], 32 * kN, p.n, own, plain, p.top, 0, room[warp], &count[warp]));
        }
    }
}

// ------------------------------------------------------------- a row by a cluster

// CTAs of kThreads threads, gridDim a multiple of the cluster.  Each holds K
// pieces a thread at a time, `rounds` times; a row of one round is read once.
template <typename T, int K, int kThreads>
__global__ void __launch_bounds__(kThreads) k_logp_cluster(const __grid_constant__ LogpArgs p, int rounds, int per_row) {
    constexpr int kWarps = kThreads / 32, kN = Piece<T>::kN;
    __shared__ uint64_t room[kWarps][kCandidates], lists[(kWarps > 8 ? kWarps : 8) * 32], best[32];   // lists: of the warps, then of the CTAs
    __shared__ int count[kWarps];
    __shared__ float part_m[kWarps], cta_m;
    __shared__ Sums part[kWarps], cta;
    const cg::cluster_group cluster = cg::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = per_row > 1 ? (int)cluster.block_rank() : 0;
    const auto sync = [&] {
        if (per_row > 1) cluster.sync();
        else __syncthreads();
    };
    for (int64_t row = blockIdx.x / per_row; row < p.rows; row += gridDim.x / per_row) {
        const T* x = static_cast<const T*>(p.x) + row * p.n;
        const int64_t step = (int64_t)kThreads * kN, start = ((int64_t)rank * rounds * K * kThreads + threadIdx.x) * kN - Piece<T>::shift_of(x);
        Piece<T> q[K];
        const auto load = [&](int round) {
#pragma unroll
            for (int k = 0; k < K; ++k) q[k].load(x, start + ((int64_t)round * K + k) * step, p.n);
        };
        const auto most = [&] {
            float v = q[0].most();
#pragma unroll
            for (int k = 1; k < K; ++k) v = max_nan(v, q[k].most());
            return v;
        };
        float own = -INFINITY, m;
        for (int round = 0; round < rounds; ++round) {
            load(round);
            own = max_nan(own, most());
        }
        m = warp_max(own);
        if (lane == 0) part_m[warp] = m;
        __syncthreads();
        m = part_m[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) m = max_nan(m, part_m[w]);
        if (per_row > 1) {
            if (threadIdx.x == 0) cta_m = m;
            cluster.sync();
            for (int c = 0; c < per_row; ++c) m = max_nan(m, *cluster.map_shared_rank(&cta_m, c));
        }
        const bool plain = m < INFINITY && m > -INFINITY;
        Sums t = {0.f, 0.f, 0};
        uint64_t list = 0;
        for (int round = 0; round < rounds; ++round) {
            if (rounds > 1) {
                load(round);
                own = most();
            }
            if (plain) add_up(t, q, m, own);
            if (p.top) list = best_of_pieces(q, start + (int64_t)round * K * step, step, p.n, own, plain, p.top, list, room[warp], &count[warp]);
        }
        warp_sums(t.below, t.weighted);
        t.equal = (int)__reduce_add_sync(0xffffffffu, (unsigned)t.equal);
        if (lane == 0) part[warp] = t;
        if (lane < p.top) lists[warp * p.top + lane] = list;
        __syncthreads();
        if (warp == 0) {
            Sums all = part[0];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) {
                all.below += part[w].below;
                all.weighted += part[w].weighted;
                all.equal += part[w].equal;
            }
            uint64_t mine = p.top ? best_of(lists, kWarps * p.top, p.top) : 0;
            if (per_row > 1) {
                if (lane == 0) cta = all;
                best[lane] = mine;
            }
            if (per_row == 1) {
                const Row done(m, all.below, all.equal);
                if (lane == 0) done.write(p, row, x, all);
                if (p.top) write_top(p, row, done, mine);
            }
        }
        if (per_row > 1) {
            cluster.sync();
            if (rank == 0 && warp == 0) {
                Sums all = cta;
                for (int c = 1; c < per_row; ++c) {
                    const Sums o = *cluster.map_shared_rank(&cta, c);
                    all.below += o.below;
                    all.weighted += o.weighted;
                    all.equal += o.equal;
                }
                const Row done(m, all.below, all.equal);
                if (lane == 0) done.write(p, row, x, all);
                if (p.top) {
                    for (int c = 0; c < per_row; ++c)
                        if (lane < p.top) lists[c * p.top + lane] = cluster.map_shared_rank(best, c)[lane];
                    __syncwarp();
                    write_top(p, row, done, best_of(lists, per_row * p.top, p.top));
                }
            }
        }
        sync();   // what was shared may be written again, and outlives its readers
    }
}

// ------------------------------------------------------------- few classes

constexpr int kFewClasses = 64, kTileRows = 128;

// A tile of rows lies in memory as one stretch: 16 bytes at a time (its start
// allows that when the tensor's does) to shared memory, where rows are `pitch`
// apart, so that a thread a row meets few others in its banks: an odd number of
// words, or a word and a half more or less.
template <typename T> __host__ __device__ inline int pitch_of(int n) {
    return sizeof(T) == 4 ? n | 1 : n % 4 == 0 ? n + 2 : n;
}

struct Place {   // of an element of a tile: at most 128 x 64 of them, so the quotient is exact
    int row, j;
    __device__ __forceinline__ Place(int i, int n) {
        row = (int)(((unsigned)i * ((1u << 20) / (unsigned)n + 1u)) >> 20);
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
            if (kIn) reinterpret_cast<uint4*>(tile)[i] = reinterpret_cast<const uint4*>(x)[i];
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
}

template <typename T>
__global__ void __launch_bounds__(kTileRows) k_logp_few(const __grid_constant__ LogpArgs p, bool vec) {
    extern __shared__ uint4 memory[];
    T* tile = reinterpret_cast<T*>(memory);
    for (int64_t base = (int64_t)blockIdx.x * kTileRows; base < p.rows; base += (int64_t)gridDim.x * kTileRows) {
        const int rows = p.rows - base < kTileRows ? (int)(p.rows - base) : kTileRows, n = p.n;
        tile_copy<T, true>(tile, const_cast<T*>(static_cast<const T*>(p.x)) + base * n, rows * n, n, vec);
        __syncthreads();
        if ((int)threadIdx.x < rows) {
            const int64_t row = base + threadIdx.x;
            const T* x = tile + threadIdx.x * pitch_of<T>(n);
            float m = -INFINITY;
            for (int j = 0; j < n; ++j) m = max_nan(m, to_f32(x[j]));
            Sums t = {0.f, 0.f, 0};
            if (m < INFINITY && m > -INFINITY)
                for (int j = 0; j < n; ++j) {
                    const float d = to_f32(x[j]) - m, e2 = fmaxf(d * kLog2e, kLowest), e = exp2_fast(e2);
                    t.equal += d == 0.f;
                    t.below += d == 0.f ? 0.f : e;
                    t.weighted = fmaf(e, e2, t.weighted);
                }
            const Row done(m, t.below, t.equal);
            done.write(p, row, x, t);
            uint64_t before = ~0ull;
            for (int k = 0; k < p.top; ++k) {
                uint64_t b = 0;
                for (int j = 0; j < n; ++j) {
                    const uint64_t v = ranked(to_f32(x[j]), j);
                    if (v < before && v > b) b = v;
                }
                before = b;
                p.top_ids[row * p.top + k] = class_of(b);
                p.top_logp[row * p.top + k] = done.logp(score_of(b));
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------- the gradient

// What the elements of a row have in common.
struct RowGrad {
    float m, s, all, ge, gl;   // p (all - ge log p), and gl more at the label
    float rest;                // of all without gl: at the label
    int label;
    bool empty;
    __device__ __forceinline__ RowGrad(const LogpArgs& p, int64_t row) {
        const float2 st = p.stats[row];
        m = st.x;
        s = st.y;
        empty = m == -INFINITY;
        label = p.gl ? p.labels.at(row, p.n) : -1;
        gl = label >= 0 ? p.gl[row] : 0.f;
        ge = p.ge ? p.ge[row] : 0.f;
        rest = (p.gz ? p.gz[row] : 0.f) - (p.ge ? ge * p.entropy[row] : 0.f);
        all = rest - gl;
    }
    // The label's own 1 - p would lose what a confident answer leaves.
    __device__ __forceinline__ float at_label(float x) const {
        const float lp = (x - m) - s, t = max_nan(lp * kLog2e, kLowest);
        return empty ? 0.f : fmaf(exp2_fast(t), fmaf(-ge * kLn2, t, rest), -gl * expm1f(lp));
    }
    __device__ __forceinline__ float at(float x) const {
        const float t = max_nan(((x - m) - s) * kLog2e, kLowest);   // NaN of a row that has one stays
        return empty ? 0.f : exp2_fast(t) * fmaf(-ge * kLn2, t, all);
    }
};

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

// kLanes neighbouring threads a row (32, or the CTA); each takes pieces kLanes apart,
// blockIdx.y gives the first of its `pieces` ones.
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) k_logp_grad(const __grid_constant__ LogpArgs p, int pieces, bool same) {
    constexpr int kN = Piece<T>::kN, kUnroll = 4;
    const int64_t rows_at = gridDim.x * (int64_t)(256 / kLanes);
    for (int64_t row = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes; row < p.rows; row += rows_at) {
        const T* x = static_cast<const T*>(p.x) + row * p.n;
        T* gx = static_cast<T*>(p.gx) + row * p.n;
        const RowGrad g(p, row);
        const int shift = Piece<T>::shift_of(x);
        const uint64_t minus = both(-g.m), less = both(-g.s), scale = both(kLog2e), ge = both(-g.ge * kLn2), all = both(g.all);
        for (int piece = 0; piece < pieces; piece += kUnroll) {
            const int64_t first = (((int64_t)blockIdx.y * pieces + piece) * kLanes + threadIdx.x % kLanes) * kN - shift;
            if (first - (int64_t)(threadIdx.x % kLanes) * kN >= p.n) break;
            Piece<T> q[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) q[k].load(x, first + k * kLanes * kN, piece + k < pieces ? p.n : 0);
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                const int64_t at = first + k * kLanes * kN;
                if (piece + k >= pieces || at >= p.n) continue;
                float v[kN];
#pragma unroll
                for (int i = 0; i < kN / 2; ++i) {
                    const float2 f = q[k].pair(i);
                    float a, b;
                    pair_to(mul2(add2(add2(pair_of(f.x, f.y), minus), less), scale), a, b);
                    a = max_nan(a, kLowest);
                    b = max_nan(b, kLowest);
                    pair_to(mul2(pair_of(exp2_fast(a), exp2_fast(b)), fma2(pair_of(a, b), ge, all)), v[2 * i], v[2 * i + 1]);
                }
                const int64_t l = g.label - at;
                if (g.label >= 0 && l >= 0 && l < kN) {
                    const float own = g.at_label(to_f32(x[g.label]));
#pragma unroll
                    for (int i = 0; i < kN; ++i) v[i] = i == l ? own : v[i];
                }
                if (g.empty)
#pragma unroll
                    for (int i = 0; i < kN; ++i) v[i] = 0.f;
                if (same && at >= 0 && at + kN <= p.n) {
                    Vec<T, kN> o;
                    o.from(v);
                    o.store(gx + at);
                } else {
#pragma unroll
                    for (int i = 0; i < kN; ++i)
                        if (at + i >= 0 && at + i < p.n) gx[at + i] = from_f32<T>(v[i]);
                }
            }
        }
    }
}

// ------------------------------------------------------------------ host side

static int64_t vectors_of(const LogpArgs& a, int kn) {   // of a row, wherever it begins
    const bool aligned = a.n % kn == 0 && aligned16(a.x);
    return ceil_div((int64_t)a.n + (aligned ? 0 : kn - 1), kn);
}

static unsigned grid_of(int64_t ctas) { return (unsigned)(ctas < (1 << 30) ? ctas : 1 << 30); }

template <typename T, int K, int kThreads>
static cudaError_t launch_cluster(const LogpArgs& a, int rounds, int per_row, cudaStream_t s) {
    cudaLaunchConfig_t c = {};
    const int64_t rows = a.rows < (1 << 24) ? a.rows : 1 << 24;
    c.gridDim = dim3((unsigned)(rows * per_row));
    c.blockDim = dim3(kThreads);
    c.stream = s;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)per_row;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    c.attrs = &attr;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, k_logp_cluster<T, K, kThreads>, a, rounds, per_row);
}

template <typename T, int K>
static cudaError_t launch_warp(const LogpArgs& a, cudaStream_t s) {
    constexpr int kRows = K == 1 ? 2 : 1;
    k_logp_warp<T, K, kRows><<<grid_of(ceil_div(a.rows, 8 * kRows)), 256, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t forward(const LogpArgs& a, cudaStream_t s) {
    constexpr int kN = Piece<T>::kN;
    if (a.n <= kFewClasses) {
        k_logp_few<T><<<grid_of(ceil_div(a.rows, kTileRows)), kTileRows, kTileRows * pitch_of<T>(a.n) * sizeof(T), s>>>(a, aligned16(a.x));
        return cudaGetLastError();
    }
    const int64_t nv = vectors_of(a, kN);
    if (nv <= 32) return launch_warp<T, 1>(a, s);
    if (nv <= 64) return launch_warp<T, 2>(a, s);
    if (nv <= 96) return launch_warp<T, 3>(a, s);
    if (nv <= 32 * kWarpVectors) return launch_warp<T, kWarpVectors>(a, s);
    // The smallest cluster that holds the row; a larger one where the rows leave SMs without work.
    int per_row = 1;
    while (per_row < 8 && (nv > 4096 * (int64_t)per_row || (a.rows * per_row * 2 <= sm_count() && nv >= 1024 * (int64_t)per_row)))
        per_row *= 2;
    const int64_t each = ceil_div(nv, per_row);
    if (each <= 512) return launch_cluster<T, 4, 128>(a, 1, per_row, s);
    if (each <= 1024) return launch_cluster<T, 4, 256>(a, 1, per_row, s);
    if (each <= 2048) return launch_cluster<T, 4, 512>(a, 1, per_row, s);
    return launch_cluster<T, 8, 512>(a, (int)ceil_div(each, 4096), per_row, s);
}

template <typename T>
static cudaError_t backward(const LogpArgs& a, cudaStream_t s) {
    constexpr int kN = Piece<T>::kN;
    if (a.n <= kFewClasses) {
        k_logp_few_grad<T><<<grid_of(ceil_div(a.rows, kTileRows)), kTileRows, kTileRows * pitch_of<T>(a.n) * sizeof(T), s>>>(
            a, aligned16(a.x), aligned16(a.gx));
        return cudaGetLastError();
    }
    const int64_t nv = vectors_of(a, kN);
    const bool same = (((uintptr_t)a.x ^ (uintptr_t)a.gx) & 15) == 0;
    if (nv <= 32 * 8) {
        k_logp_grad<T, 32><<<grid_of(ceil_div(a.rows, 8)), 256, 0, s>>>(a, (int)ceil_div(nv, 32), same);
    } else {
        int64_t pieces = 4, y = ceil_div(nv, 256 * pieces);
        if (y > 65535) y = 65535, pieces = ceil_div(ceil_div(nv, 256), y);
        k_logp_grad<T, 256><<<dim3(grid_of(a.rows), (unsigned)y), 256, 0, s>>>(a, (int)pieces, same);
    }
    return cudaGetLastError();
}

}  // namespace plr

using namespace plr;

extern "C" {

static bool logp_ok(const plattice_log_probs_args* q) {
    return q && dtype_ok(q->dtype) && q->rows >= 0 && q->n >= 1 && q->n <= (1 << 30) && q->top >= 0 &&
           q->top <= PLATTICE_MAX_TOP && q->top <= q->n && fits(q->rows, q->n) &&
           (!q->labels || (uintptr_t)q->labels % (q->labels_wide ? 8 : 4) == 0);
}

static LogpArgs logp_args(const plattice_log_probs_args* q) {
    return {q->logits, {q->labels, q->labels_wide}, q->logp, q->entropy, reinterpret_cast<float2*>(q->stats), q->lse, q->top_logp,
            q->top_ids, q->grad_logp, q->grad_entropy, q->grad_lse, q->grad_logits, q->rows, q->n, q->top};
}

int plattice_log_probs(const plattice_log_probs_args* q, void* stream) {
    if (!logp_ok(q)) return PLATTICE_ERR_INVALID;
    if (q->rows == 0) return PLATTICE_OK;
    if (!q->logits || (uintptr_t)q->logits % dtype_size(q->dtype) || !q->stats || (uintptr_t)q->stats % 8 ||
        (q->logp && !q->labels) || (q->top && (!q->top_logp || !q->top_ids)))
        return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const LogpArgs a = logp_args(q);
    const cudaError_t e = q->dtype == PLATTICE_F32    ? forward<float>(a, s)
                          : q->dtype == PLATTICE_BF16 ? forward<__nv_bfloat16>(a, s)
                                                      : forward<__half>(a, s);
    return rows_status(e, "plattice_log_probs");
}

int plattice_log_probs_backward(const plattice_log_probs_args* q, void* stream) {
    if (!logp_ok(q)) return PLATTICE_ERR_INVALID;
    if (q->rows == 0) return PLATTICE_OK;
    if (!q->logits || (uintptr_t)q->logits % dtype_size(q->dtype) || !q->stats || (uintptr_t)q->stats % 8 || !q->grad_logits ||
        (uintptr_t)q->grad_logits % dtype_size(q->dtype) || (q->grad_logp && !q->labels) || (q->grad_entropy && !q->entropy))
        return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const LogpArgs a = logp_args(q);
    const cudaError_t e = q->dtype == PLATTICE_F32    ? backward<float>(a, s)
                          : q->dtype == PLATTICE_BF16 ? backward<__nv_bfloat16>(a, s)
                                                      : backward<__half>(a, s);
    return rows_status(e, "plattice_log_probs_backward");
}

}  // extern "C"
