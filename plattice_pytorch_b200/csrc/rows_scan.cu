// rows_scan.cu -- gated linear recurrence along lines of rows, and its gradients.
//
//   h[t] = a[t] h[t-1] + u[t],    u = x or (1 - a) x
//   G[t] = g[t] + a[t+1] G[t+1];  grad_x = G or (1 - a) G,
//   grad_a[t] = G[t] (h[t-1] or h[t-1] - x[t])
//
// A thread walks the steps of V neighbouring channels of a line in blocks of 16
// (PLATTICE_SCAN_KEEP), whose loads are in flight together.  The forward keeps
// the float32 state before each block (4 bytes per 16 steps: 3 % of what a pass
// over 16-bit rows moves), from which the backward computes h again: in float32
// and without reading h.
#include "plattice_runtime.h"
#include "rows_host.h"
#include "rows_vec.cuh"

namespace plr {

constexpr int kSteps = PLATTICE_SCAN_KEEP;
constexpr int kThreads = 128;

// Cut lines: what steps together do to a state, s -> f s + r.  A product of gates leaves
// float32 long before states do (0.5 for 120 steps and 2 for 200 take a state of 1 to
// 2^80, and the last 128 steps' product alone is infinite; an infinite state stays
// infinite however small the product), so f has an exponent of its own: m 2^e, where e
// is a multiple of 60 and m between 2^-60 and 2^60 (at most 1 with e < 0, at least 1 with
// e > 0), or m is 0, with e = 0.
constexpr float kSmall = 0x1p-60f, kLarge = 0x1p60f;
constexpr int kPart = 60, kFar = kPart << 20;   // e goes no farther: nothing comes back from there

__device__ __forceinline__ bool medium(float v) { return fabsf(v) >= kSmall && fabsf(v) <= kLarge; }

struct Factor {
    float m;
    int e;
    __device__ __forceinline__ void hold() {   // after a product: m is between 2^-120 and 2^120, or 0
        const bool small = fabsf(m) < kSmall, large = fabsf(m) > kLarge;
        m *= small ? kLarge : large ? kSmall : 1.f;
        e += small ? -kPart : large ? kPart : 0;
        const bool over = e < 0 && fabsf(m) > 1.f, under = e > 0 && fabsf(m) < 1.f;
        m *= over ? kSmall : under ? kLarge : 1.f;
        e += over ? kPart : under ? -kPart : 0;
        e = m == 0.f ? 0 : max(min(e, kFar), -kFar);
    }
    __device__ __forceinline__ void times(const Factor& o) {
        m = m == 0.f ? 0.f : m * o.m;   // the state before a gate of 0 is of no consequence
        e += o.e;
        hold();
    }
    __device__ __forceinline__ void times(float gate) {   // of any size
        const float a = fabsf(gate);
        times(a < kSmall && a > 0.f ? Factor{gate * kLarge * kLarge, -2 * kPart}
              : a > kLarge          ? Factor{gate * kSmall * kSmall, 2 * kPart}
                                    : Factor{gate, 0});
    }
};
// Out of line, as it is there for few blocks: gates that leave 2^+-120 within eight steps.
struct Eight { float g[8]; };
__device__ __noinline__ Factor times_slowly(Factor f, Eight q) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f.times(q.g[i]);
    return f;
}

struct alignas(16) Map {
    Factor f;
    float r;
};
// A state of 0 stays r, whatever the factor.
__device__ __forceinline__ float apply(const Map& m, float s) {
    float v = m.f.m * s;
    int e = m.f.e;
#pragma unroll
    for (int i = 0; i < 3; ++i) {   // in parts that float32 has: of more than 6 60 nothing is left, or infinity
        const int part = max(min(e, 2 * kPart), -2 * kPart);
        v *= __int_as_float((127 + part) << 23);
        e -= part;
    }
    return s == 0.f ? m.r : v + m.r;
}
// The map of both.  Without branches: one for what stays within 2^+-60 took a line of 3000 x 8
// in bfloat16 0.9 us more, whose 64 pieces soon leave it.
__device__ __forceinline__ Map then(Map first, const Map& second) {
    first.f.times(second.f);
    first.r = apply(second, first.r);
    return first;
}

// Nearly all maps are tame: |f| <= 1 and |r| <= 2^24.  Where all of a line's are, and the
// state it begins with, a map is two numbers of float32: what f loses below 2^-126 is
// never multiplied up again, and its product with a state, which grows by 2^24 a map at
// most, is below 2^-85.  f is NaN for a map that is not tame, and so is every product with it;
// the state is then found from the maps as they are (1000003 x 16 in float32: 70 us, and 81
// from a state of 1e8; 3 lines of 5000 x 64 in bfloat16 9.4 and 17).
constexpr float kTame = 0x1p24f;
__device__ __forceinline__ float2 plain(const Map& m) {
    const bool tame = m.f.e <= 0 && fabsf(m.f.m) <= 1.f && fabsf(m.r) <= kTame;
    const float f = m.f.e == 0 ? m.f.m : m.f.e == -kPart ? m.f.m * kSmall : m.f.e == -2 * kPart ? m.f.m * kSmall * kSmall : 0.f;
    return make_float2(tame ? f : __int_as_float(0x7fffffff), m.r);
}
__device__ __forceinline__ float2 then(float2 first, float2 second) {
    return make_float2(first.x * second.x, fmaf(second.x, first.y, second.y));
}

struct ScanArgs {
    const void *x, *a;
    const float* state;
    void* h;
    float *last, *states;
    const void* g;
    const float* grad_last;
    void *gx, *ga;
    float* gs;
    Map* sums;               // cut lines: [line][piece][c]
    Map* tile_sums;          // [line][tile][c], of a CTA's pieces together
    float2 *plain_sums, *plain_tiles;   // the same as plain()
    int64_t lines, steps, blocks;   // blocks of kSteps in a line
    int64_t tiles;           // CTAs a line's steps are cut over
    int c, reverse;
    int lanes, pieces;       // of a CTA: lanes x pieces = kThreads
    int piece_blocks;        // blocks of a piece
};

// What a thread works on: V channels of a line, blocks first..end-1 of it.  Whole
// lines: neighbouring threads take neighbouring channels, of several lines where
// a line has few.  Cut lines: a CTA has `pieces` pieces of its lanes' channels.
template <int V, bool kCut> struct Work {
    int64_t line, col, piece, first, end, tile;
    int lane, own;           // of the CTA's lanes, pieces
    bool here;
    __device__ __forceinline__ Work(const ScanArgs& p, int64_t tile_) : tile(tile_) {
        const int units = p.c / V;
        if (!kCut) {
            const int64_t index = (int64_t)blockIdx.x * kThreads + threadIdx.x;
            lane = own = 0;
            line = index / units;
            col = (index - line * units) * V;
            here = line < p.lines;
            piece = first = 0;
            end = p.blocks;
            return;
        }
        lane = threadIdx.x % p.lanes;
        own = threadIdx.x / p.lanes;
        const int wide = (units + p.lanes - 1) / p.lanes;
        line = blockIdx.x / wide;
        col = ((int64_t)(blockIdx.x - line * wide) * p.lanes + lane) * V;
        here = col < p.c;
        piece = tile * p.pieces + own;
        first = piece * p.piece_blocks;
        end = first + p.piece_blocks < p.blocks ? first + p.piece_blocks : p.blocks;
    }
};

// Element of the first step of block b of a line, and from a step to the next.
__device__ __forceinline__ int64_t stride_of(const ScanArgs& p) { return p.reverse ? -(int64_t)p.c : p.c; }
__device__ __forceinline__ int64_t start_of(const ScanArgs& p, int64_t line, int64_t col, int64_t b) {
    const int64_t t = b * kSteps;
    int64_t o = (line * p.steps + (p.reverse ? p.steps - 1 - t : t)) * p.c + col;
    asm volatile("" : "+l"(o));   // one offset a block: otherwise 16 addresses a tensor are carried along in registers
    return o;
}
__device__ __forceinline__ int steps_of(const ScanArgs& p, int64_t b) {
    const int64_t left = p.steps - b * kSteps;
    return left < kSteps ? (int)left : kSteps;
}

// A block's steps of a thread.  `run`: the thread has all channels of its line, and the
// steps lie in one stretch of kSteps V elements: 16 bytes at a time where the stretch
// allows it (lines of one channel: 184 x 18219 in bfloat16 and back took 142 us element
// by element, for each of which a warp's threads meet in no two sectors).
template <typename T, int V> struct Block {
    Vec<T, V> v[kSteps];
    static constexpr int kWords = kSteps * V * (int)sizeof(T) / 4;
    static __device__ __forceinline__ bool stretch(const T* low, int n, bool run) {
        return run && n == kSteps && ((uintptr_t)low & 15) == 0;
    }
    // What lies behind the n-th step is 0, or `fill`.
    __device__ __forceinline__ void load(const void* base, int64_t o, int64_t stride, int n, bool run, float fill = 0.f) {
        const T* p = static_cast<const T*>(base) + o;
        const T* low = stride < 0 ? p + (kSteps - 1) * stride : p;
        if (stretch(low, n, run)) {
            uint32_t w[kWords];
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const uint4 q = reinterpret_cast<const uint4*>(low)[i / 4];
                w[i] = q.x, w[i + 1] = q.y, w[i + 2] = q.z, w[i + 3] = q.w;
            }
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const Vec<T, V> up = part(w, i), down = part(w, kSteps - 1 - i);
                v[i] = stride < 0 ? down : up;
            }
        } else if (n == kSteps) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i, p += stride) v[i].load(p);
        } else {
#pragma unroll
            for (int i = 0; i < kSteps; ++i, p += stride) {
                if (i < n) {
                    v[i].load(p);
                } else {
                    float all[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) all[j] = fill;
                    v[i].from(all);
                }
            }
        }
    }
    __device__ __forceinline__ void store(void* base, int64_t o, int64_t stride, int n, bool run) const {
        T* p = static_cast<T*>(base) + o;
        T* low = stride < 0 ? p + (kSteps - 1) * stride : p;
        if (stretch(low, n, run)) {
            uint32_t w[kWords];
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = 0;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                Vec<T, V> one;
#pragma unroll
                for (int k = 0; k < Vec<T, V>::kWords; ++k) one.r.w[k] = stride < 0 ? v[kSteps - 1 - i].r.w[k] : v[i].r.w[k];
                put(w, i, one);
            }
#pragma unroll
            for (int i = 0; i < kWords; i += 4) reinterpret_cast<uint4*>(low)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < kSteps; ++i, p += stride)
                if (i < n) v[i].store(p);
        }
    }

private:
    static __device__ __forceinline__ Vec<T, V> part(const uint32_t (&w)[kWords], int i) {
        Vec<T, V> r;
        if constexpr (Vec<T, V>::kBytes == 2) {
            r.r.w[0] = (uint16_t)(w[i / 2] >> (i % 2 * 16));
        } else {
#pragma unroll
            for (int k = 0; k < Vec<T, V>::kWords; ++k) r.r.w[k] = w[i * Vec<T, V>::kWords + k];
        }
        return r;
    }
    static __device__ __forceinline__ void put(uint32_t (&w)[kWords], int i, const Vec<T, V>& one) {
        if constexpr (Vec<T, V>::kBytes == 2) {
            w[i / 2] |= (uint32_t)one.r.w[0] << (i % 2 * 16);
        } else {
#pragma unroll
            for (int k = 0; k < Vec<T, V>::kWords; ++k) w[i * Vec<T, V>::kWords + k] = one.r.w[k];
        }
    }
};

template <bool kBlend> __device__ __forceinline__ float input(float a, float x) { return kBlend ? (1.f - a) * x : x; }

// ---------------------------------------------------------------- cut lines
//
// Lines that do not fill the device by themselves are cut: a thread takes a
// piece, a CTA `pieces` neighbouring ones of its lanes.  The first kernel gives
// for each piece and for the CTA's pieces together what it does to a state.  The
// second one's CTAs each go through the CTAs before them, then through their own
// pieces, and know every piece's first state.

__device__ __forceinline__ void set_identity(Map& m) { m = Map{{1.f, 0}, 0.f}; }
__device__ __forceinline__ void set_identity(float2& m) { m = make_float2(1.f, 0.f); }

// The maps of a CTA's pieces (`place`: in the order they are gone through), each after
// all before it, are left in `shared`: in pairs, so that many pieces of few channels
// take as many steps as their number has bits (one by one: 169 lines of 2661 x 2, 28 us).
// kSets sets of maps, each with places of its own.
template <typename M, int V, int kSets>
__device__ __forceinline__ void scan_maps(M (&m)[kSets][V], M (*shared)[kThreads * V], const int (&place)[kSets], int lane,
                                          const ScanArgs& p) {
    for (int d = 1;; d <<= 1) {
#pragma unroll
        for (int q = 0; q < kSets; ++q)
#pragma unroll
            for (int j = 0; j < V; ++j) shared[q][(place[q] * p.lanes + lane) * V + j] = m[q][j];
        __syncthreads();
        if (d >= p.pieces) return;
#pragma unroll
        for (int q = 0; q < kSets; ++q)
            if (place[q] >= d)
#pragma unroll
                for (int j = 0; j < V; ++j) m[q][j] = then(shared[q][((place[q] - d) * p.lanes + lane) * V + j], m[q][j]);
        __syncthreads();
    }
}

// Pieces of a backward pass are gone through from the last on.
template <typename T, int V, bool kBlend, bool kGrad>
__global__ void __launch_bounds__(kThreads) k_scan_sums(const __grid_constant__ ScanArgs p) {
    __shared__ Map shared[1][kThreads * V];
    const Work<V, true> w(p, blockIdx.y);
    Factor f[V];
    float r[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        f[j] = Factor{1.f, 0};
        r[j] = 0.f;
    }
    if (w.here) {
        const int64_t stride = stride_of(p);
        for (int64_t k = w.first; k < w.end; ++k) {
            const int64_t b = kGrad ? w.first + w.end - 1 - k : k, o = start_of(p, w.line, w.col, b);
            const int n = steps_of(p, b);
            Block<T, V> x, a;
            x.load(kGrad ? p.g : p.x, o, stride, n, p.c == V);
            a.load(p.a, o, stride, n, p.c == V, 1.f);   // of steps that are not there: r 1 + 0
#pragma unroll
            for (int j = 0; j < V; ++j) {
                Factor& q = f[j];
#pragma unroll
                for (int first = 0; first < kSteps; first += 8) {
                    const float m0 = q.m;
                    float least = INFINITY;
                    Eight eight;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int t = kGrad ? kSteps - 1 - first - i : first + i;
                        const float gate = a.v[t].at(j), v = x.v[t].at(j);
                        r[j] = kGrad ? gate * (v + r[j]) : fmaf(gate, r[j], input<kBlend>(gate, v));
                        q.m *= gate;
                        least = fminf(least, fabsf(q.m));
                        eight.g[i] = gate;
                    }
                    if (least >= kSmall * kSmall && fabsf(q.m) <= kLarge * kLarge) {
                        if (q.e != 0 || !medium(q.m)) q.hold();
                    } else {
                        bool closed = m0 == 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) closed |= eight.g[i] == 0.f;
                        q = closed ? Factor{0.f, 0} : times_slowly(Factor{m0, q.e}, eight);
                    }
                }
            }
        }
        if (w.first < p.blocks)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int64_t at = (w.line * p.tiles * p.pieces + w.piece) * p.c + w.col + j;
                p.sums[at] = Map{f[j], r[j]};
                p.plain_sums[at] = plain(Map{f[j], r[j]});
            }
    }
    Map m[1][V];
#pragma unroll
    for (int j = 0; j < V; ++j) m[0][j] = Map{f[j], r[j]};
    const int place[1] = {kGrad ? p.pieces - 1 - w.own : w.own};
    scan_maps<Map, V, 1>(m, shared, place, w.lane, p);
    if (w.own == 0 && w.here)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int64_t at = (w.line * p.tiles + w.tile) * p.c + w.col + j;
            const Map all = shared[0][((p.pieces - 1) * p.lanes + w.lane) * V + j];
            p.tile_sums[at] = all;
            p.plain_tiles[at] = plain(all);
        }
}

// The maps of all CTAs before, and of the CTA's pieces before the thread's.  Of the first a
// thread takes a part, one of as many as the CTA has pieces.
template <typename M, int V, bool kGrad>
__device__ __forceinline__ void maps_before(M (&tiles)[V], M (&own)[V], const M* tile_sums, const M* sums, M (*shared)[kThreads * V],
                                            const ScanArgs& p, const Work<V, true>& w) {
    constexpr int kAtOnce = sizeof(M) == sizeof(float2) ? 8 : 2;
    const int64_t before = kGrad ? p.tiles - 1 - w.tile : w.tile, part = (before + p.pieces - 1) / p.pieces;
    M m[2][V];   // of the CTAs; of the piece
#pragma unroll
    for (int j = 0; j < V; ++j) {
        set_identity(m[0][j]);
        set_identity(m[1][j]);
    }
    if (w.here) {
        const int64_t to = (w.own + 1) * part < before ? (w.own + 1) * part : before;
        const M* from = tile_sums + w.line * p.tiles * p.c + w.col;
        for (int64_t k = w.own * part; k < to; k += kAtOnce) {
            M ahead[kAtOnce][V];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    set_identity(ahead[i][j]);
                    if (k + i < to) ahead[i][j] = from[(kGrad ? p.tiles - 1 - k - i : k + i) * p.c + j];
                }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) m[0][j] = then(m[0][j], ahead[i][j]);
        }
        if (w.first < p.blocks)
#pragma unroll
            for (int j = 0; j < V; ++j) m[1][j] = sums[((w.line * p.tiles + w.tile) * p.pieces + w.own) * p.c + w.col + j];
    }
    const int place[2] = {w.own, kGrad ? p.pieces - 1 - w.own : w.own};
    scan_maps<M, V, 2>(m, shared, place, w.lane, p);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        tiles[j] = shared[0][((p.pieces - 1) * p.lanes + w.lane) * V + j];
        if (place[1]) own[j] = shared[1][((place[1] - 1) * p.lanes + w.lane) * V + j];
        else set_identity(own[j]);
    }
}

// The state that the thread's piece starts from, of the line's s: where a map is not tame.
template <int V> struct States { float s[V]; };
template <int V, bool kGrad>
__device__ __noinline__ States<V> first_state_slowly(States<V> s, const ScanArgs& p, int64_t tile) {
    const Work<V, true> w(p, tile);
    __shared__ Map shared[2][kThreads * V];
    Map tiles[V], own[V];
    maps_before<Map, V, kGrad>(tiles, own, p.tile_sums, p.sums, shared, p, w);
#pragma unroll
    for (int j = 0; j < V; ++j) s.s[j] = apply(own[j], apply(tiles[j], s.s[j]));
    return s;
}
template <int V, bool kGrad>
__device__ __forceinline__ void first_state(float (&s)[V], const ScanArgs& p, const Work<V, true>& w) {
    __shared__ float2 shared[2][kThreads * V];
    float2 tiles[V], own[V];
    maps_before<float2, V, kGrad>(tiles, own, p.plain_tiles, p.plain_sums, shared, p, w);
    bool tame = true;
    States<V> line;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        line.s[j] = s[j];
        tame &= fabsf(s[j]) <= kTame && tiles[j].x == tiles[j].x && own[j].x == own[j].x;
        s[j] = fmaf(own[j].x, fmaf(tiles[j].x, s[j], tiles[j].y), own[j].y);
    }
    if (__syncthreads_or(!tame)) {
        line = first_state_slowly<V, kGrad>(line, p, w.tile);
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = line.s[j];
    }
}

// ---------------------------------------------------------------- the passes

template <typename T, int V, bool kBlend, bool kCut>
__global__ void __launch_bounds__(kThreads, 6) k_scan(const __grid_constant__ ScanArgs p) {
    const Work<V, kCut> w(p, kCut ? (int64_t)gridDim.y - 1 - blockIdx.y : 0);   // what was read last may still be in the L2
    float h[V];
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = w.here && p.state ? p.state[w.line * p.c + w.col + j] : 0.f;
    if constexpr (kCut) first_state<V, false>(h, p, w);
    if (!w.here || w.first >= p.blocks) return;
    const int64_t stride = stride_of(p);
    for (int64_t b = w.first; b < w.end; ++b) {
        const int n = steps_of(p, b);
        const int64_t o = start_of(p, w.line, w.col, b);
        Block<T, V> x, a;
        x.load(p.x, o, stride, n, p.c == V);
        a.load(p.a, o, stride, n, p.c == V);
        if (p.states) {
            float* s = p.states + (w.line * p.blocks + b) * p.c + w.col;
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] = h[j];
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            if (i < n) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float gate = a.v[i].at(j);
                    h[j] = fmaf(gate, h[j], input<kBlend>(gate, x.v[i].at(j)));
                }
            }
            x.v[i].from(h);
        }
        x.store(p.h, o, stride, n, p.c == V);
    }
    if (p.last && w.end == p.blocks)
#pragma unroll
        for (int j = 0; j < V; ++j) p.last[w.line * p.c + w.col + j] = h[j];
}

template <typename T, int V, bool kBlend, bool kCut>
__global__ void __launch_bounds__(kThreads, 4) k_scan_grad(const __grid_constant__ ScanArgs p) {
    const Work<V, kCut> w(p, kCut ? blockIdx.y : 0);
    float r[V];   // what reaches h from later steps
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = w.here && p.grad_last ? p.grad_last[w.line * p.c + w.col + j] : 0.f;
    if constexpr (kCut) first_state<V, true>(r, p, w);
    if (!w.here || w.first >= p.blocks) return;
    const int64_t stride = stride_of(p);
    for (int64_t b = w.end - 1; b >= w.first; --b) {
        const int n = steps_of(p, b);
        const int64_t o = start_of(p, w.line, w.col, b);
        Block<T, V> x, a, g;
        float h[V], d[kSteps][V];   // d: h[t-1], or h[t-1] - x[t]
        const float* s = p.states + (w.line * p.blocks + b) * p.c + w.col;
#pragma unroll
        for (int j = 0; j < V; ++j) h[j] = s[j];
        x.load(p.x, o, stride, n, p.c == V);
        a.load(p.a, o, stride, n, p.c == V);
        g.load(p.g, o, stride, n, p.c == V);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float gate = a.v[i].at(j), v = x.v[i].at(j);
                d[i][j] = kBlend ? h[j] - v : h[j];
                h[j] = fmaf(gate, h[j], input<kBlend>(gate, v));
            }
#pragma unroll
        for (int i = kSteps - 1; i >= 0; --i)
            if (i < n) {
                float fx[V], fa[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float gate = a.v[i].at(j), whole = g.v[i].at(j) + r[j];
                    fx[j] = kBlend ? (1.f - gate) * whole : whole;
                    fa[j] = whole * d[i][j];
                    r[j] = gate * whole;
                }
                g.v[i].from(fx);
                x.v[i].from(fa);
            }
        g.store(p.gx, o, stride, n, p.c == V);
        x.store(p.ga, o, stride, n, p.c == V);
    }
    if (p.gs && w.first == 0)
#pragma unroll
        for (int j = 0; j < V; ++j) p.gs[w.line * p.c + w.col + j] = r[j];
}

// ---------------------------------------------------------------- single steps
//
// One step of every line, as where a state is kept between calls: no line to walk,
// V channels of any line a thread (4679 lines of 792 bfloat16 channels forward and
// back: 85 us as blocks of a step).

template <typename T, int V, bool kBlend>
__global__ void __launch_bounds__(256) k_scan_step(const __grid_constant__ ScanArgs p, int64_t units) {
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x, at = u * V;
    if (u >= units) return;
    Vec<T, V> x, a;
    Vec<float, V> s;
    x.load(static_cast<const T*>(p.x) + at);
    a.load(static_cast<const T*>(p.a) + at);
    s.zero();
    if (p.state) s.load(p.state + at);
    if (p.states) s.store(p.states + at);
    float h[V];
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = fmaf(a.at(j), s.at(j), input<kBlend>(a.at(j), x.at(j)));
    Vec<T, V> y;
    y.from(h);
    y.store(static_cast<T*>(p.h) + at);
    s.from(h);
    if (p.last) s.store(p.last + at);
}

template <typename T, int V, bool kBlend>
__global__ void __launch_bounds__(256) k_scan_step_grad(const __grid_constant__ ScanArgs p, int64_t units) {
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x, at = u * V;
    if (u >= units) return;
    Vec<T, V> x, a, g, gx, ga;
    Vec<float, V> s, r;
    x.load(static_cast<const T*>(p.x) + at);
    a.load(static_cast<const T*>(p.a) + at);
    g.load(static_cast<const T*>(p.g) + at);
    s.load(p.states + at);
    r.zero();
    if (p.grad_last) r.load(p.grad_last + at);
    float fx[V], fa[V], fs[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float gate = a.at(j), whole = g.at(j) + r.at(j);
        fx[j] = kBlend ? (1.f - gate) * whole : whole;
        fa[j] = whole * (kBlend ? s.at(j) - x.at(j) : s.at(j));
        fs[j] = gate * whole;
    }
    gx.from(fx);
    ga.from(fa);
    gx.store(static_cast<T*>(p.gx) + at);
    ga.store(static_cast<T*>(p.ga) + at);
    r.from(fs);
    if (p.gs) r.store(p.gs + at);
}

// ------------------------------------------------------------------ host side

// Threads that fill the device (each has 16 steps of two or three tensors in flight;
// one round of the backward's CTAs: 1000003 x 16 in bfloat16 30 us with 384 an SM, 42
// with 512), and those below which lines are cut: a cut line is read twice.
constexpr int64_t kEnough = kPlanSms * 512, kEnoughGrad = kPlanSms * 384, kFew = kPlanSms * 192;

struct ScanPlan {
    int v, lanes, pieces, piece_blocks;
    int64_t wide, tiles, cells, bytes;   // wide: CTAs beside one another; cells: maps of all tiles
    bool cut;
};

static ScanPlan scan_plan(const plattice_scan_args* q, bool grad) {
    ScanPlan p = {};
    uintptr_t bits = (uintptr_t)q->x | (uintptr_t)q->gate;
    bits |= grad ? (uintptr_t)q->grad_h | (uintptr_t)q->grad_x | (uintptr_t)q->grad_gate : (uintptr_t)q->h;
    const int v = widest(q->c, dtype_size(q->dtype), bits);
    p.v = q->dtype != PLATTICE_F32 && v >= 2 ? 2 : 1;
    const int64_t units = q->c / p.v, blocks = ceil_div(q->steps, kSteps), threads = q->lines * units;
    p.cut = threads < kFew && blocks >= 8;
    p.tiles = 1;
    if (!p.cut) {
        p.wide = ceil_div(threads, kThreads);
        return p;
    }
    p.lanes = 1;
    while (p.lanes < 32 && p.lanes < units) p.lanes <<= 1;
    const int64_t length = blocks / ceil_div(grad ? kEnoughGrad : kEnough, threads);
    p.piece_blocks = length < 1 ? 1 : length > (1 << 20) ? 1 << 20 : (int)length;
    p.pieces = kThreads / p.lanes;
    p.wide = q->lines * ceil_div(units, p.lanes);
    p.tiles = ceil_div(blocks, (int64_t)p.piece_blocks * p.pieces);
    p.cells = q->lines * p.tiles * q->c;
    p.bytes = p.cells * (p.pieces + 1) * (int64_t)(sizeof(Map) + sizeof(float2));
    return p;
}

template <typename T, int V, bool kBlend>
static cudaError_t launch(const ScanArgs& a, const ScanPlan& p, bool grad, cudaStream_t s) {
    if (p.wide > 0x7fffffff || p.tiles > 65535) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)p.wide, (unsigned)p.tiles);
    if (grad) {
        if (p.cut) {
            k_scan_sums<T, V, kBlend, true><<<grid, kThreads, 0, s>>>(a);
            k_scan_grad<T, V, kBlend, true><<<grid, kThreads, 0, s>>>(a);
        } else {
            k_scan_grad<T, V, kBlend, false><<<grid, kThreads, 0, s>>>(a);
        }
    } else if (p.cut) {
        k_scan_sums<T, V, kBlend, false><<<grid, kThreads, 0, s>>>(a);
        k_scan<T, V, kBlend, true><<<grid, kThreads, 0, s>>>(a);
    } else {
        k_scan<T, V, kBlend, false><<<grid, kThreads, 0, s>>>(a);
    }
    return cudaGetLastError();
}

template <typename T>
static cudaError_t launch(const ScanArgs& a, const ScanPlan& p, bool blend, bool grad, cudaStream_t s) {
    constexpr int kPair = sizeof(T) == 2 ? 2 : 1;
    if (p.v == kPair) return blend ? launch<T, kPair, true>(a, p, grad, s) : launch<T, kPair, false>(a, p, grad, s);
    return blend ? launch<T, 1, true>(a, p, grad, s) : launch<T, 1, false>(a, p, grad, s);
}

template <typename T, int V>
static cudaError_t launch_step(const ScanArgs& a, bool blend, bool grad, cudaStream_t s) {
    const int64_t units = a.lines * a.c / V, ctas = ceil_div(units, 256);
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    const auto kernel = grad ? (blend ? k_scan_step_grad<T, V, true> : k_scan_step_grad<T, V, false>)
                             : (blend ? k_scan_step<T, V, true> : k_scan_step<T, V, false>);
    kernel<<<(unsigned)ctas, 256, 0, s>>>(a, units);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_step(const ScanArgs& a, bool blend, bool grad, cudaStream_t s) {
    // what is not there has a null pointer, which any access allows
    const uintptr_t rows = (uintptr_t)a.x | (uintptr_t)a.a | (uintptr_t)a.h | (uintptr_t)a.g | (uintptr_t)a.gx | (uintptr_t)a.ga,
                    states = (uintptr_t)a.state | (uintptr_t)a.last | (uintptr_t)a.states | (uintptr_t)a.grad_last | (uintptr_t)a.gs;
    if (a.lines * a.c % 4 == 0 && rows % (4 * sizeof(T)) == 0 && states % 16 == 0) return launch_step<T, 4>(a, blend, grad, s);
    return launch_step<T, 1>(a, blend, grad, s);
}

static int run(const plattice_scan_args* q, bool grad, cudaStream_t s, const char* call) {
    const ScanPlan p = scan_plan(q, grad);
    if (p.bytes && (!q->workspace || ((uintptr_t)q->workspace & 255) || q->workspace_bytes < (size_t)p.bytes))
        return PLATTICE_ERR_WORKSPACE;
    Map *sums = static_cast<Map*>(q->workspace), *tile_sums = sums + p.cells * p.pieces;
    float2 *plain_sums = reinterpret_cast<float2*>(tile_sums + p.cells), *plain_tiles = plain_sums + p.cells * p.pieces;
    const ScanArgs a{q->x, q->gate, q->state, q->h, q->last, q->states, q->grad_h, q->grad_last, q->grad_x, q->grad_gate,
                     q->grad_state, sums, tile_sums, plain_sums, plain_tiles, q->lines, q->steps,
                     ceil_div(q->steps, kSteps), p.tiles, q->c, q->reverse, p.lanes, p.pieces, p.piece_blocks};
    if (q->steps == 1) {
        // pointers of the other direction are not used
        ScanArgs b = a;
        if (grad) b.state = nullptr, b.h = nullptr, b.last = nullptr;
        else b.g = nullptr, b.grad_last = nullptr, b.gx = b.ga = nullptr, b.gs = nullptr;
        const cudaError_t e = q->dtype == PLATTICE_F32    ? launch_step<float>(b, q->blend, grad, s)
                              : q->dtype == PLATTICE_BF16 ? launch_step<__nv_bfloat16>(b, q->blend, grad, s)
                                                          : launch_step<__half>(b, q->blend, grad, s);
        return rows_status(e, call);
    }
    const cudaError_t e = q->dtype == PLATTICE_F32    ? launch<float>(a, p, q->blend, grad, s)
                          : q->dtype == PLATTICE_BF16 ? launch<__nv_bfloat16>(a, p, q->blend, grad, s)
                                                      : launch<__half>(a, p, q->blend, grad, s);
    return rows_status(e, call);
}

static bool shape_ok(const plattice_scan_args* q) {
    return q && dtype_ok(q->dtype) && q->lines >= 0 && q->steps >= 0 && q->c >= 1 && q->c <= (1 << 30) &&
           fits(q->lines, q->c) && fits(q->steps, q->c) && fits(q->lines, q->steps * q->c);
}

}  // namespace plr

using namespace plr;

extern "C" {

int plattice_scan_workspace_size(const plattice_scan_args* q, size_t* bytes) {
    if (!bytes || !shape_ok(q)) return PLATTICE_ERR_INVALID;
    *bytes = q->lines && q->steps ? (size_t)scan_plan(q, false).bytes : 0;
    return PLATTICE_OK;
}

int plattice_scan(const plattice_scan_args* q, void* stream) {
    if (!shape_ok(q)) return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (q->lines == 0) return PLATTICE_OK;
    if (q->steps == 0) {   // the state as it came
        if (!q->last) return PLATTICE_OK;
        const size_t b = (size_t)q->lines * q->c * sizeof(float);
        return rows_status(q->state ? cudaMemcpyAsync(q->last, q->state, b, cudaMemcpyDeviceToDevice, s)
                                    : cudaMemsetAsync(q->last, 0, b, s),
                           "plattice_scan");
    }
    if (!q->x || !q->gate || !q->h || !on_elements(dtype_size(q->dtype), q->x, q->gate, q->h) ||
        !on_elements(sizeof(float), q->state, q->last, q->states))
        return PLATTICE_ERR_INVALID;
    return run(q, false, s, "plattice_scan");
}

int plattice_scan_backward_workspace_size(const plattice_scan_args* q, size_t* bytes) {
    if (!bytes || !shape_ok(q)) return PLATTICE_ERR_INVALID;
    *bytes = q->lines && q->steps ? (size_t)scan_plan(q, true).bytes : 0;
    return PLATTICE_OK;
}

int plattice_scan_backward(const plattice_scan_args* q, void* stream) {
    if (!shape_ok(q)) return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (q->lines == 0) return PLATTICE_OK;
    if (q->steps == 0) {
        if (!q->grad_state) return PLATTICE_OK;
        const size_t b = (size_t)q->lines * q->c * sizeof(float);
        return rows_status(q->grad_last ? cudaMemcpyAsync(q->grad_state, q->grad_last, b, cudaMemcpyDeviceToDevice, s)
                                        : cudaMemsetAsync(q->grad_state, 0, b, s),
                           "plattice_scan_backward");
    }
    if (!q->x || !q->gate || !q->states || !q->grad_h || !q->grad_x || !q->grad_gate ||
        !on_elements(dtype_size(q->dtype), q->x, q->gate, q->grad_h, q->grad_x, q->grad_gate) ||
        !on_elements(sizeof(float), q->states, q->grad_last, q->grad_state))
        return PLATTICE_ERR_INVALID;
    return run(q, true, s, "plattice_scan_backward");
}

}  // extern "C"
