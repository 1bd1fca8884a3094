// rows_embed.cu -- rows from labels and the gradient of their table.
//
//   y[i] = scale table[id_i]            (0 for an id outside the table)
//   grad_table[v] = scale sum_{i: id_i = v} grad_y[i]
//
// The gradient of a small table (up to kSmallTable labels) is added up in shared
// memory as the rows come: every warp has a copy of some of the table's channels of
// its own, CTAs' sums are added by a second kernel.  For a larger table, or fewer
// labels, the positions are sorted by label: by counting smaller ones, or by a stable
// radix sort, 8 to 10 bits of the label a pass, in one launch of a cluster or in two or
// three launches a pass.  The sorted list is cut into chunks of equal length and each
// chunk's runs of equal labels are added in registers.  A run inside one chunk is
// written at once; the parts of a run that crosses chunks go to the workspace and are
// added in order by another kernel.  The order of the sums depends on the sizes alone:
// no atomics but counts.
#include <cooperative_groups.h>

#include <cmath>

#include "plattice_runtime.h"
#include "rows_host.h"
#include "rows_vec.cuh"

namespace plr {

namespace cg = cooperative_groups;

// `lanes` (a power of two) threads a row side by side, four rows a thread, so that
// labels, table rows and stores of four are under way together.
constexpr int kEmbedRows = 4;

template <typename T, int V>
__global__ void __launch_bounds__(256) k_embed(T* __restrict__ y, Labels ids, const T* __restrict__ table, float scale, int64_t count,
                                               int64_t n, int units, int shift) {
    const int lane = threadIdx.x & ((1 << shift) - 1), step = 256 >> shift;
    const int64_t row0 = (int64_t)blockIdx.x * (step * kEmbedRows) + (threadIdx.x >> shift);
    int id[kEmbedRows];
#pragma unroll
    for (int u = 0; u < kEmbedRows; ++u) id[u] = row0 + u * step < count ? ids.at(row0 + u * step, n) : -1;
    for (int col = lane; col < units; col += 1 << shift) {
        Vec<T, V> v[kEmbedRows];
#pragma unroll
        for (int u = 0; u < kEmbedRows; ++u) {
            v[u].zero();
            if (id[u] >= 0) v[u].load(table + ((int64_t)id[u] * units + col) * V);
        }
        T* to = y + (row0 * units + col) * V;
        const int64_t next = (int64_t)step * units * V;
#pragma unroll
        for (int u = 0; u < kEmbedRows; ++u, to += next)
            if (row0 + u * step < count) {
                float f[V];
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = id[u] >= 0 ? v[u].at(i) * scale : 0.f;
                v[u].from(f);
                v[u].store(to);
            }
    }
}

// Rows that allow no whole accesses: a thread writes 16 bytes of the result, which lies
// in one stretch, whatever rows they belong to, from table elements one by one
// (1039280 x 55 bfloat16: 124 us with an element a thread).
template <typename T>
__global__ void __launch_bounds__(256) k_embed_flat(T* __restrict__ y, Labels ids, const T* __restrict__ table, float scale, int64_t all,
                                                    int64_t n, unsigned c) {
    constexpr int kN = 16 / (int)sizeof(T);
    const int64_t base = (int64_t)blockIdx.x * (256 * kN);
    const GroupAt where(base, c);
    const unsigned o = threadIdx.x * kN;
    if (base + o >= all) return;
    int64_t row;
    unsigned col;
    where.at(o, row, col);
    int id = ids.at(row, n);
    float f[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        f[i] = id >= 0 && base + o + i < all ? to_f32(table[(int64_t)id * c + col]) * scale : 0.f;
        if (++col == c && base + o + i + 1 < all) {
            col = 0;
            id = ids.at(++row, n);
        }
    }
    T* to = y + base + o;
    if (base + o + kN <= all) {
        Vec<T, kN> v;
        v.from(f);
        v.store(to);
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (base + o + i < all) to[i] = from_f32<T>(f[i]);
    }
}

// Stores V values as T, or as `dtype` says where that is another type.
template <typename T, int V>
__device__ __forceinline__ void store_out(void* out, int dtype, bool vec, int64_t at, const float (&v)[V]) {
    if (vec) {
        Vec<T, V> o;
        o.from(v);
        o.store(static_cast<T*>(out) + at);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) store_param(out, dtype, at + j, v[j]);
    }
}

// ----------------------------------------------------------------- small tables
//
// A warp goes through rows 32 at a time; a lane adds V channels to the label's place
// in the warp's copy, which is its own place: nothing else reads or writes it.
// Where a row has fewer than 32 V channels, several rows go side by side, each
// group of lanes with a copy.  Warps of a CTA take slabs of 32 V channels first,
// then rows.  The rows come by asynchronous copies, two blocks of 32 under way
// (1048576 rows of 64 bfloat16 channels into 21 labels: 55 us, bound by the few warps
// that the copies of the table leave an SM; from loads to registers 63, sorted 210).
// Rows on no 16-byte boundaries are loaded a block at a time.  kWideTable: labels up to
// which a lane takes 8 bytes of 16-bit rows.

constexpr int kSmallTable = 96, kWideTable = 24, kTableBytes = 200 * 1024;

struct TableArgs {
    void* out;                // where one CTA has all rows, else null
    int out_dtype;
    float* part;              // [row CTAs][n][c]
    Labels ids;
    const void* g;
    float scale;
    int64_t count, n;
    int c, lane_bits, slabs;  // 2^lane_bits lanes of a row (2..32); slabs of a CTA's warps (blockIdx.y has others)
    int copies;               // warps a slab
};

__device__ __forceinline__ void copy_async16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

template <typename T, int V, bool kWhole>
__global__ void __launch_bounds__(1024) k_small_table(const __grid_constant__ TableArgs a) {
    // tables [warp][group][n + 1][lanes V], the last row for rows without a label and what
    // lies behind the rows or channels; then rows [warp][2][32][lanes V] as T
    extern __shared__ float4 memory[];
    float* tables = reinterpret_cast<float*>(memory);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int n = (int)a.n, groups = 32 >> a.lane_bits, bits = a.lane_bits + (V == 4 ? 2 : 1), width = 1 << bits,
              each = (n + 1) * 32 * V;
    T* rows = reinterpret_cast<T*>(tables + warps * each) + warp * 2 * 32 * width;
    for (int i = threadIdx.x; i < warps * each; i += blockDim.x) tables[i] = 0.f;
    __syncthreads();
    const int group = lane >> a.lane_bits, own = lane & ((1 << a.lane_bits) - 1);
    const int slab = blockIdx.y * a.slabs + warp % a.slabs, copy = warp / a.slabs;
    float* table = tables + warp * each + group * (n + 1) * width + own * V;
    const T* g = static_cast<const T*>(a.g) + slab * width;
    const int wide = a.c - slab * width;   // channels from the slab's first on
    const int64_t blocks = (a.count + 31) / 32, step = (int64_t)gridDim.x * a.copies, c = a.c;
    // The rows of block b on their way to a stage; a lane's label of them is the result.
    const auto bring = [&](int64_t b, T* stage) {
        const int64_t row0 = b * 32, left = a.count - row0;
        if (left > 0) {
            constexpr int kN = kWhole ? 16 / (int)sizeof(T) : 1, kBits = kWhole ? (sizeof(T) == 2 ? 3 : 2) : 0;
            // a pass of the warp: 32 accesses of kN elements of neighbouring rows (or a part of one)
            const int per_row = bits - kBits, at = (lane & ((1 << per_row) - 1)) * kN;
            for (int first = 0; first < (1 << per_row); first += 32) {
                const int col = at + first * kN;
                int row = per_row >= 5 ? 0 : lane >> per_row;
                const int next = per_row >= 5 ? 1 : 32 >> per_row;
                const T* from = g + (row0 + row) * c + (per_row >= 5 ? (lane + first) * kN : col);
                T* to = stage + (row << bits) + (per_row >= 5 ? (lane + first) * kN : col);
                const bool inside = (per_row >= 5 ? (lane + first) * kN : col) < wide;
                const int most = left < 32 ? (int)left : 32;
                for (; row < most; row += next, from += next * c, to += next << bits)
                    if (inside) {
                        if constexpr (kWhole) copy_async16(to, from);
                        else *to = *from;
                    }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return lane < left ? a.ids.raw(row0 + lane) : -1ll;   // not looked at yet: it is on its way, too
    };
    const auto add = [&](const T* stage, long long label) {
        const int id = label >= 0 && label < n ? (int)label : n;
        const T* from = stage + (group << bits) + own * V;
        int at = group;
#pragma unroll 4
        for (int r = 0; r < 32; r += 2 * groups, at += 2 * groups, from += (2 * groups) << bits) {
            // two rows of the group together: of the same label they are added first
            const int l0 = __shfl_sync(0xffffffffu, id, at), l1 = __shfl_sync(0xffffffffu, id, at + groups);
            Vec<T, V> v0, v1;
            v0.load(from);
            v1.load(from + (groups << bits));
            Vec<float, V>*p0 = reinterpret_cast<Vec<float, V>*>(table + (l0 << bits)),
            *p1 = reinterpret_cast<Vec<float, V>*>(table + (l1 << bits));
            const Vec<float, V> t0 = *p0, t1 = *p1;
            const bool same = l0 == l1;
            float f0[V], f1[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float x = v1.at(j);
                f0[j] = t0.at(j) + (v0.at(j) + (same ? x : 0.f));
                f1[j] = t1.at(j) + x;
            }
            Vec<float, V> o0, o1;
            o0.from(f0);
            o1.from(f1);
            *p0 = o0;
            if (!same) *p1 = o1;
        }
    };
    T *even = rows, *odd = rows + 32 * width;
    int64_t b = (int64_t)blockIdx.x * a.copies + copy;
    long long id0 = bring(b, even), id1 = bring(b + step, odd);
    for (; b < blocks; b += 2 * step) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        add(even, id0);
        __syncwarp();
        id0 = bring(b + 2 * step, even);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        add(odd, id1);
        __syncwarp();
        id1 = bring(b + 3 * step, odd);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    // The copies of a slab together, in order, for the CTA's channels.
    const int64_t first = (int64_t)blockIdx.y * a.slabs * width;
    const int span = a.c - first < (int64_t)a.slabs * width ? (int)(a.c - first) : a.slabs * width;
    for (int i = threadIdx.x; i < n * span; i += blockDim.x) {
        const int label = i / span, at = i - label * span, w = at / width, j = at - w * width;
        float sum = 0.f;
        for (int k = 0; k < a.copies; ++k)
            for (int q = 0; q < groups; ++q) sum += tables[(k * a.slabs + w) * each + (q * (n + 1) + label) * width + j];
        const int64_t to = (int64_t)label * a.c + first + at;
        if (a.out) store_param(a.out, a.out_dtype, to, sum * a.scale);
        else a.part[(int64_t)blockIdx.x * n * a.c + to] = sum;
    }
}

// out[i] = scale times the sum of part[k][i]: 8 groups of 32 threads, each every 8th part.
__global__ void __launch_bounds__(256) k_small_join(void* out, int dtype, const float* __restrict__ part, int parts, int64_t cells,
                                                    float scale) {
    __shared__ float sums[8][32];
    const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float s = 0.f;
    if (i < cells) {
#pragma unroll 8
        for (int k = threadIdx.y; k < parts; k += 8) s += part[k * cells + i];
    }
    sums[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && i < cells) {
#pragma unroll
        for (int k = 1; k < 8; ++k) s += sums[k][threadIdx.x];
        store_param(out, dtype, i, s * scale);
    }
}

// --------------------------------------------------------------- sorting labels

constexpr int kMostBits = 10;       // of a label, a pass
constexpr int kRankSorted = 2048;      // as many are sorted by counting
constexpr int kClusterSorted = 32768;  // as many by one cluster

struct Entry { unsigned label, at; };   // at: the position in ids

// The table's rows that no label has are 0: all of it is written first, in shares
// by CTAs that the sort's launches have behind their own (a memory-bound write
// beside launches that wait for latencies; 16384 labels of a 50000 x 1024 table).
struct Zeros {
    uint4* p;
    int64_t begin, end;   // of this launch, in 16 bytes
    int ctas;
    __device__ __forceinline__ void share(int cta) const {
        const int64_t each = (end - begin + ctas - 1) / ctas, from = begin + cta * each, to = from + each < end ? from + each : end;
#pragma unroll 4
        for (int64_t i = from + threadIdx.x; i < to; i += blockDim.x) p[i] = make_uint4(0, 0, 0, 0);
    }
};

// A label's place: the labels below it and the equal ones before it.  A CTA has all
// labels in shared memory and places 64; sixteen threads share a label's comparisons.
__global__ void __launch_bounds__(1024) k_rank_sort(Entry* __restrict__ out, unsigned* __restrict__ valid, unsigned* __restrict__ starts, Labels ids, int64_t n,
                                                   int count, Zeros zeros) {
    if ((int)blockIdx.x * 64 >= count) return zeros.share(blockIdx.x - (count + 63) / 64);
    __shared__ uint4 labels[kRankSorted / 4];
    __shared__ unsigned places[16][64], sums[32];
    unsigned* flat = reinterpret_cast<unsigned*>(labels);
    const int padded = (count + 63) / 64 * 64;
    unsigned all = 0;
#pragma unroll 8
    for (int k = threadIdx.x; k < padded; k += 1024) {
        const unsigned v = k < count ? (unsigned)ids.at(k, n) : 0xffffffffu;   // none: behind all
        flat[k] = v;
        all += v != 0xffffffffu;
    }
    __syncthreads();
    const int e = threadIdx.x & 63, i0 = blockIdx.x * 64, i = i0 + e, share = padded / 64;   // fours of a thread
    const unsigned mine = i < count ? flat[i] : 0xffffffffu;
    unsigned place = 0;
    const int from = (threadIdx.x >> 6) * share, to = from + share;
    // the fours before the CTA's own labels, those around them, those behind
    const int low = i0 / 4 < from ? from : i0 / 4 < to ? i0 / 4 : to, high = i0 / 4 + 16 < low ? low : i0 / 4 + 16 < to ? i0 / 4 + 16 : to;
    const unsigned next = mine + 1u;   // equal ones before count
#pragma unroll 4
    for (int k = from; k < low; ++k) {
        const uint4 o = labels[k];
        place += (o.x < next) + (o.y < next) + (o.z < next) + (o.w < next);
    }
    for (int k = low; k < high; ++k) {
        const uint4 o = labels[k];
        place += (o.x < mine + (4 * k < i)) + (o.y < mine + (4 * k + 1 < i)) + (o.z < mine + (4 * k + 2 < i)) +
                 (o.w < mine + (4 * k + 3 < i));
    }
#pragma unroll 4
    for (int k = high; k < to; ++k) {
        const uint4 o = labels[k];
        place += (o.x < mine) + (o.y < mine) + (o.z < mine) + (o.w < mine);
    }
    places[threadIdx.x >> 6][e] = place;
    all = __reduce_add_sync(0xffffffffu, all);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = all;
    __syncthreads();
    if (threadIdx.x < 64 && mine != 0xffffffffu)
    {
        place = 0;
#pragma unroll
        for (int q = 0; q < 16; ++q) place += places[q][e];
        out[place] = Entry{mine, (unsigned)i};
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        all = 0;
#pragma unroll
        for (int w = 0; w < 32; ++w) all += sums[w];
        *valid = all;
        *starts = 0;
    }
}

// Entries of pass 0 come from the labels themselves (those outside the table
// are left out), later ones from the pass before.
struct Source {
    Labels ids;
    int64_t n, count;
    const Entry* from;        // null: the labels
    const unsigned* valid;    // entries in `from`
    __device__ __forceinline__ int64_t size() const { return from ? (int64_t)*valid : count; }
    // digit of entry i (kDigits: none) and the entry
    template <int kDigits> __device__ __forceinline__ int get(int64_t i, int64_t size, int shift, Entry& e) const {
        if (i >= size) return kDigits;
        if (from) {
            e = from[i];
        } else {
            const int id = ids.at(i, n);
            if (id < 0) return kDigits;
            e.label = (unsigned)id;
            e.at = (unsigned)i;
        }
        return (e.label >> shift) & (kDigits - 1);
    }
};

// counts [tile][digit]; a tile is kItems entries a thread.
template <int kItems, int kDigits>
__global__ void __launch_bounds__(256) k_sort_count(unsigned* __restrict__ counts, Source src, int shift, int tiles, Zeros zeros) {
    if ((int)blockIdx.x >= tiles) return zeros.share(blockIdx.x - tiles);
    __shared__ unsigned h[kDigits + 1];
    for (int i = threadIdx.x; i <= kDigits; i += 256) h[i] = 0;
    __syncthreads();
    const int64_t size = src.size(), base = (int64_t)blockIdx.x * (256 * kItems);
    Entry e[kItems];
    int digit[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) digit[k] = src.get<kDigits>(base + k * 256 + threadIdx.x, size, shift, e[k]);
#pragma unroll
    for (int k = 0; k < kItems; ++k) atomicAdd(&h[digit[k]], 1u);   // counts: any order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kDigits; i += 256) counts[(int64_t)blockIdx.x * kDigits + i + threadIdx.x] = h[i + threadIdx.x];
}

// Exclusive sum over the CTA's 256 threads.
__device__ __forceinline__ unsigned before_me(unsigned v, unsigned& all) {
    __shared__ unsigned warps[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned s = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned t = __shfl_up_sync(0xffffffffu, s, d);
        if (lane >= d) s += t;
    }
    if (lane == 31) warps[warp] = s;
    __syncthreads();
    unsigned o = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        if (w < warp) o += warps[w];
        all += warps[w];
    }
    return o + s - v;
}

// counts become the number of entries of the digit in the tiles before (many
// tiles: a CTA a digit); totals [digit].
__global__ void __launch_bounds__(256) k_sort_sums(unsigned* __restrict__ counts, unsigned* __restrict__ totals, int64_t tiles) {
    unsigned carry = 0;
    for (int64_t base = 0; base < tiles; base += 256) {
        const int64_t t = base + threadIdx.x;
        unsigned* at = counts + t * gridDim.x + blockIdx.x;
        unsigned all;
        const unsigned o = before_me(t < tiles ? *at : 0u, all);
        if (t < tiles) *at = carry + o;
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Stable: a warp takes neighbouring entries of the tile, 32 at a time, and counts
// equal digits before its own by a match.  totals null: the tile adds up the
// counts of all tiles itself.  A thread has kEach neighbouring digits.
template <int kItems, int kDigits>
__global__ void __launch_bounds__(256) k_sort_place(Entry* __restrict__ out, const unsigned* __restrict__ counts,
                                                    const unsigned* __restrict__ totals, unsigned* __restrict__ valid,
                                                    unsigned* __restrict__ starts, Source src, int shift, int tiles, Zeros zeros) {
    if ((int)blockIdx.x >= tiles) return zeros.share(blockIdx.x - tiles);
    constexpr int kEach = kDigits / 256;
    __shared__ unsigned h[8][kDigits + 1];
    for (int i = threadIdx.x; i < 8 * (kDigits + 1); i += 256) (&h[0][0])[i] = 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t size = src.size(), base = (int64_t)blockIdx.x * (256 * kItems) + warp * (32 * kItems);
    Entry e[kItems];
    int digit[kItems];
    unsigned rank[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) digit[k] = src.get<kDigits>(base + k * 32 + lane, size, shift, e[k]);
    unsigned o[kEach], total[kEach], sum = 0, all;   // of the thread's digits: in the tiles before, in all
#pragma unroll
    for (int j = 0; j < kEach; ++j) o[j] = total[j] = 0;
    if (totals) {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            o[j] = counts[(int64_t)blockIdx.x * kDigits + threadIdx.x * kEach + j];
            total[j] = totals[threadIdx.x * kEach + j];
        }
    } else {
#pragma unroll 8
        for (int t = 0; t < tiles; ++t) {
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const unsigned v = counts[t * kDigits + threadIdx.x * kEach + j];
                total[j] += v;
                if (t < (int)blockIdx.x) o[j] += v;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) sum += total[j];
    unsigned before = before_me(sum, all);   // all threads: h has been cleared behind it
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        o[j] += before;
        before += total[j];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *valid = all, *starts = 0;
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const unsigned same = __match_any_sync(0xffffffffu, digit[k]);
        const unsigned had = h[warp][digit[k]];
        rank[k] = had + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if ((same & ((1u << lane) - 1)) == 0) h[warp][digit[k]] = had + __popc(same);
        __syncwarp();
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int d = threadIdx.x * kEach + j;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            const unsigned had = h[w][d];
            h[w][d] = o[j];
            o[j] += had;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kItems; ++k)
        if (digit[k] < kDigits) out[h[warp][digit[k]] + rank[k]] = e[k];
}

// All passes in one launch, by a cluster: CTA r has entries 4096 r.. of each pass.  The
// CTAs read each other's counts out of shared memory; the entries go through memory
// (16384 labels of 50000: 27 us as launches of the kernels above).
constexpr int kSortCtas = 8, kSortItems = 4;

__global__ void __cluster_dims__(kSortCtas) __launch_bounds__(1024) k_cluster_sort(Entry* first, Entry* second, unsigned* valid,
                                                                                unsigned* starts, Labels ids, int64_t n, int count,
                                                                                int passes, int bits, Zeros zeros) {
    if (blockIdx.x >= kSortCtas) return zeros.share(blockIdx.x - kSortCtas);   // whole clusters
    extern __shared__ unsigned h[];   // [32][digits + 1], then of the CTA [digits], then where they begin [digits]
    __shared__ unsigned warps[32];
    const cg::cluster_group cluster = cg::this_cluster();
    const int digits = 1 << bits, rank_of = (int)cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5,
              d = threadIdx.x;
    unsigned *own = h + warp * (digits + 1), *totals = h + 32 * (digits + 1), *begins = totals + digits;
    int size = count;
    Entry *from = nullptr, *to = first;
    for (int pass = 0; pass < passes; ++pass) {
        for (int i = threadIdx.x; i < 32 * (digits + 1); i += 1024) h[i] = 0;
        Entry e[kSortItems];
        int digit[kSortItems];
        unsigned rank[kSortItems];
        const int base = rank_of * (1024 * kSortItems) + warp * (32 * kSortItems) + lane;
#pragma unroll
        for (int k = 0; k < kSortItems; ++k) {
            const int i = base + k * 32;
            digit[k] = digits;
            if (i < size) {
                if (from) {   // written by the cluster's other CTAs: not from this SM's cache
                    const uint2 q = __ldcg(reinterpret_cast<const uint2*>(from) + i);
                    e[k] = Entry{q.x, q.y};
                    digit[k] = (e[k].label >> (bits * pass)) & (digits - 1);
                } else if (const int id = ids.at(i, n); id >= 0) {
                    e[k] = Entry{(unsigned)id, (unsigned)i};
                    digit[k] = id & (digits - 1);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSortItems; ++k) {
            const unsigned same = __match_any_sync(0xffffffffu, digit[k]);
            const unsigned had = own[digit[k]];
            rank[k] = had + __popc(same & ((1u << lane) - 1));
            __syncwarp();
            if ((same & ((1u << lane) - 1)) == 0) own[digit[k]] = had + __popc(same);
            __syncwarp();
        }
        __syncthreads();
        if (d < digits) {   // counts of the warps before, and of the CTA
            unsigned o = 0;
#pragma unroll 8
            for (int w = 0; w < 32; ++w) {
                const unsigned had = h[w * (digits + 1) + d];
                h[w * (digits + 1) + d] = o;
                o += had;
            }
            totals[d] = o;
        }
        cluster.sync();
        unsigned before = 0, all = 0;
        if (d < digits)
#pragma unroll
            for (int c = 0; c < kSortCtas; ++c) {
                const unsigned v = *cluster.map_shared_rank(totals + d, c);
                all += v;
                if (c < rank_of) before += v;
            }
        unsigned s = all;   // exclusive sum over the digits
#pragma unroll
        for (int q = 1; q < 32; q <<= 1) {
            const unsigned t = __shfl_up_sync(0xffffffffu, s, q);
            if (lane >= q) s += t;
        }
        if (lane == 31) warps[warp] = s;
        __syncthreads();
        unsigned w = warps[lane];
#pragma unroll
        for (int q = 1; q < 32; q <<= 1) {
            const unsigned t = __shfl_up_sync(0xffffffffu, w, q);
            if (lane >= q) w += t;
        }
        size = (int)__shfl_sync(0xffffffffu, w, 31);
        const unsigned front = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
        if (d < digits) begins[d] = (warp ? front : 0u) + s - all + before;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSortItems; ++k)
            if (digit[k] < digits) to[begins[digit[k]] + own[digit[k]] + rank[k]] = e[k];
        cluster.sync();   // the entries are there, and the counts have been read
        from = to;
        to = to == first ? second : first;
    }
    if (rank_of == 0 && threadIdx.x == 0) *valid = (unsigned)size, *starts = 0;
}

// ------------------------------------------------------------------ sums of runs

struct RunArgs {
    void* out;
    int out_dtype;
    float* part;              // [chunks][2][c]: of a run that came from before; that goes on behind
    const Entry* sorted;
    const unsigned* valid;
    unsigned* starts;         // their number, then the chunks in which a run begins that goes on behind
    const void* g;
    float scale;
    int64_t count;            // entries that `sorted` has room for
    int c, length;            // length: entries of a chunk
    bool vec, vec4;           // rows of out, of part: whole accesses
};

// A thread's V channels of the entries of one chunk.  blockDim: (lanes of a row, chunks of a CTA).
template <typename T, int V>
__global__ void __launch_bounds__(256) k_runs(const __grid_constant__ RunArgs a) {
    const int64_t chunk = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int64_t begin = chunk * a.length;
    const int64_t col = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V;
    if (begin >= a.count || col >= a.c) return;
    Entry e[8];   // read ahead of what `valid` allows (there is room for all), used as far as it does
    const auto entries = [&](int64_t i) {
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = a.sorted[i + k < a.count ? i + k : a.count - 1];
    };
    entries(begin);
    const unsigned before = a.sorted[begin > 0 ? begin - 1 : 0].label;
    const int64_t valid = *a.valid;
    if (begin >= valid) return;
    const int64_t end = begin + a.length < valid ? begin + a.length : valid;
    const T* g = static_cast<const T*>(a.g) + col;
    unsigned label = e[0].label;
    bool head = begin > 0 && before == label;
    const bool tail_at_end = end < valid && a.sorted[end].label == a.sorted[end - 1].label;
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
    const auto out = [&](bool tail) {
        if (head || tail) {
            store_out<float, V>(a.part, PLATTICE_F32, a.vec4, (chunk * 2 + (head ? 0 : 1)) * a.c + col, acc);
        } else {
            float v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = acc[j] * a.scale;
            store_out<T, V>(a.out, a.out_dtype, a.vec, (int64_t)label * a.c + col, v);
        }
    };
    for (int64_t i = begin; i < end; i += 8) {
        Vec<T, V> v[8];
        unsigned of[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (i + k < end) {
                of[k] = e[k].label;
                v[k].load(g + (int64_t)e[k].at * a.c);
            } else {
                v[k].zero();
                of[k] = of[k - 1 < 0 ? 0 : k - 1];   // i < end: k is above 0
            }
        }
        entries(i + 8);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (of[k] != label) {
                out(false);
                label = of[k];
                head = false;
#pragma unroll
                for (int j = 0; j < V; ++j) acc[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += v[k].at(j);
        }
    }
    out(tail_at_end);
    if (col == 0 && tail_at_end && !head) a.starts[1 + atomicAdd(a.starts, 1u)] = (unsigned)chunk;   // in any order: runs are apart
}

// The runs that begin in a chunk and go on behind it: its part and those of the
// chunks up to the run's end, in order.  A warp 32 V channels of a run; runs of more
// than kLongRun parts by the CTA: `lanes` threads of V channels side by side, each such
// group takes every groups-th part, and theirs are added in pairs.
constexpr int kLongRun = 24, kJoinWarps = 16;

template <int V>
__device__ __forceinline__ void add_parts(float (&s)[V], const RunArgs& a, int64_t chunk, int64_t col, int64_t first, int64_t last,
                                          int64_t step) {
    for (int64_t k = first; k <= last; k += 8 * step) {
        Vec<float, V> v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            v[u].zero();
            if (k + u * step <= last) v[u].load(a.part + (chunk + k + u * step) * 2 * a.c + col);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] += v[u].at(j);
    }
}

template <int V>
__global__ void __launch_bounds__(32 * kJoinWarps, 2) k_join_runs(const __grid_constant__ RunArgs a, int lanes) {
    __shared__ float sums[kJoinWarps * 32 * V];
    __shared__ int64_t long_chunk[kJoinWarps], long_parts[kJoinWarps], long_first[kJoinWarps];
    const unsigned starts = a.starts[0];
    const int64_t valid = *a.valid;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned strips = (unsigned)((a.c + 32 * V - 1) / (32 * V));
    const uint64_t items = (uint64_t)starts * strips;
    const auto tail = [&](float (&s)[V], int64_t chunk, int64_t col) {   // the run's first part
        Vec<float, V> v;
        v.load(a.part + (chunk * 2 + 1) * a.c + col);
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = v.at(j);
    };
    const auto write = [&](float (&s)[V], int64_t chunk, int64_t col) {
        const int64_t at = (int64_t)a.sorted[(chunk + 1) * a.length].label * a.c + col;
#pragma unroll
        for (int j = 0; j < V; ++j) store_param(a.out, a.out_dtype, at + j, s[j] * a.scale);
    };
    // Neighbouring items, such as the strips of a long run, go to different CTAs (side by
    // side in one: 285886 x 97 of 1289 labels, the most frequent one 37000 times, 58 us;
    // so 30).
    for (uint64_t i0 = blockIdx.x; i0 < items; i0 += (uint64_t)gridDim.x * kJoinWarps) {
        const uint64_t i = i0 + (uint64_t)warp * gridDim.x;
        int64_t chunk = 0, parts = 0;   // chunks behind this one that the run reaches: those that begin with its label
        if (i < items) {
            const unsigned run = (unsigned)(i / strips), strip = (unsigned)(i - (uint64_t)run * strips);
            chunk = a.starts[1 + run];
            const unsigned label = a.sorted[(chunk + 1) * a.length].label;
            parts = 1;
            for (int count = 128; count == 128; parts += count) {
                bool same[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int64_t at = (chunk + 1 + parts + 32 * u + lane) * a.length;
                    same[u] = at < valid && a.sorted[at < valid ? at : 0].label == label;
                }
                count = 0;
#pragma unroll
                for (int u = 0; u < 4; ++u) count += __popc(__ballot_sync(0xffffffffu, same[u]));
            }
            const int64_t col = ((int64_t)strip * 32 + lane) * V;
            if (parts <= kLongRun && col < a.c) {
                float s[V];
                tail(s, chunk, col);
                add_parts(s, a, chunk, col, 1, parts, 1);
                write(s, chunk, col);
            }
            if (lane == 0) long_first[warp] = (int64_t)strip * 32 * V;
        }
        if (lane == 0) {
            long_chunk[warp] = chunk;
            long_parts[warp] = parts;
        }
        __syncthreads();
        for (int w = 0; w < kJoinWarps; ++w) {
            if (long_parts[w] <= kLongRun) continue;
            const int group = threadIdx.x / lanes, groups = 32 * kJoinWarps / lanes, at = threadIdx.x % lanes * V;
            const int64_t col = long_first[w] + at;
            float s[V];
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] = 0.f;
            if (col < a.c) {
                if (group == 0) tail(s, long_chunk[w], col);
                add_parts(s, a, long_chunk[w], col, 1 + group, long_parts[w], groups);
            }
            for (int d = groups / 2; d; d >>= 1) {
#pragma unroll
                for (int j = 0; j < V; ++j) sums[threadIdx.x * V + j] = s[j];
                __syncthreads();
                if (group < d)
#pragma unroll
                    for (int j = 0; j < V; ++j) s[j] += sums[(threadIdx.x + d * lanes) * V + j];
                __syncthreads();
            }
            if (group == 0 && col < a.c) write(s, long_chunk[w], col);
        }
        __syncthreads();
    }
}

// The same for up to 8 V channels: `lanes` threads of V channels a run (a warp a run uses few
// of its threads: 510952 x 8 of 107924 labels 31 us, so 5).  The longer runs of a round are
// listed, in any order, and added by a warp or, above kWarpRun parts, by the CTA.
constexpr int kJoinNarrow = 8, kWarpRun = 512;

template <int V>
__global__ void __launch_bounds__(32 * kJoinWarps, 2) k_join_narrow(const __grid_constant__ RunArgs a, int bits) {
    __shared__ float sums[kJoinWarps * 32 * V];
    __shared__ unsigned long_chunk[kJoinWarps * 32], far_chunk[kJoinWarps * 32], far_parts[kJoinWarps * 32], longs, fars;
    const unsigned starts = a.starts[0];
    const int64_t valid = *a.valid;
    const int lanes = 1 << bits, groups = 32 * kJoinWarps >> bits, group = threadIdx.x >> bits, at = (threadIdx.x & (lanes - 1)) * V;
    const auto same_label = [&](int64_t chunk, unsigned label) {
        const int64_t i = chunk * a.length;
        return i < valid && a.sorted[i < valid ? i : 0].label == label;
    };
    const auto tail = [&](float (&s)[V], int64_t chunk) {
        Vec<float, V> v;
        v.load(a.part + (chunk * 2 + 1) * a.c + at);
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = v.at(j);
    };
    const auto write = [&](float (&s)[V], int64_t chunk) {
        const int64_t to = (int64_t)a.sorted[(chunk + 1) * a.length].label * a.c + at;
#pragma unroll
        for (int j = 0; j < V; ++j) store_param(a.out, a.out_dtype, to + j, s[j] * a.scale);
    };
    for (uint64_t r0 = blockIdx.x; r0 < starts; r0 += (uint64_t)gridDim.x * groups) {
        const uint64_t run = r0 + (uint64_t)group * gridDim.x;
        if (threadIdx.x == 0) longs = fars = 0;
        __syncthreads();
        if (run < starts) {
            const int64_t chunk = a.starts[1 + run];
            const unsigned label = a.sorted[(chunk + 1) * a.length].label;
            int parts = 1;
            for (int count = 8; count == 8 && parts <= kLongRun; parts += count) {
                bool same[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) same[u] = same_label(chunk + 1 + parts + u, label);
                count = 0;
#pragma unroll
                for (int u = 0; u < 8; ++u) count += same[u];
            }
            if (parts > kLongRun) {
                if (at == 0) long_chunk[atomicAdd(&longs, 1u)] = (unsigned)chunk;
            } else if (at < a.c) {
                float s[V];
                tail(s, chunk);
                add_parts(s, a, chunk, at, 1, parts, 1);
                write(s, chunk);
            }
        }
        __syncthreads();
        for (unsigned k = threadIdx.x >> 5; k < longs; k += kJoinWarps) {   // a warp a run
            const int64_t chunk = long_chunk[k];
            const unsigned label = a.sorted[(chunk + 1) * a.length].label;
            const int lane = threadIdx.x & 31;
            int64_t parts = 1;
            for (int count = 128; count == 128; parts += count) {
                bool same[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) same[u] = same_label(chunk + 1 + parts + 32 * u + lane, label);
                count = 0;
#pragma unroll
                for (int u = 0; u < 4; ++u) count += __popc(__ballot_sync(0xffffffffu, same[u]));
            }
            if (parts > kWarpRun) {
                if (lane == 0) {
                    const unsigned i = atomicAdd(&fars, 1u);
                    far_chunk[i] = (unsigned)chunk;
                    far_parts[i] = (unsigned)parts;
                }
                continue;
            }
            float s[V];
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] = 0.f;
            if (at < a.c) {
                if (lane < lanes) tail(s, chunk);
                add_parts(s, a, chunk, at, 1 + (lane >> bits), parts, 32 >> bits);
            }
            for (int d = 16; d >= lanes; d >>= 1)
#pragma unroll
                for (int j = 0; j < V; ++j) s[j] += __shfl_down_sync(0xffffffffu, s[j], d);
            if (lane < lanes && at < a.c) write(s, chunk);
        }
        __syncthreads();
        for (unsigned k = 0; k < fars; ++k) {   // the CTA a run
            const int64_t chunk = far_chunk[k];
            float s[V];
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] = 0.f;
            if (at < a.c) {
                if (group == 0) tail(s, chunk);
                add_parts(s, a, chunk, at, 1 + group, far_parts[k], groups);
            }
            for (int d = groups / 2; d; d >>= 1) {
#pragma unroll
                for (int j = 0; j < V; ++j) sums[threadIdx.x * V + j] = s[j];
                __syncthreads();
                if (group < d)
#pragma unroll
                    for (int j = 0; j < V; ++j) s[j] += sums[(threadIdx.x + d * lanes) * V + j];
                __syncthreads();
            }
            if (group == 0 && at < a.c) write(s, chunk);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ host side

static int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }

struct EmbedPlan {
    bool small;
    int v, lane_bits, slabs, warps, warp_bytes, ctas, ctas_y;   // small table
    int passes, bits, items, tiles, length;      // sorted; passes 0: by counting
    int64_t chunks;
    int64_t totals, starts, counts, first, second, part, bytes;   // offsets in the workspace
};

constexpr int kOwnSums = 48;   // tiles up to which the tiles add up the counts themselves

static EmbedPlan embed_plan(int64_t count, int64_t n, int c, int element) {
    EmbedPlan p = {};
    // Worth the tables' way in and out (620 labels of 95 x 98: 85 us, sorted 21), and of rows
    // that come in whole accesses (118781 x 333 element by element: 275 us).
    p.small = n <= kSmallTable && count >= 512 * n && c * element % 16 == 0;
    if (p.small) {
        // 8 bytes a lane (half the instructions a row) where many warps' copies of that fit
        p.v = element == 4 || n <= kWideTable ? 8 / element : 4 / element;
        const int units = c / p.v;
        p.lane_bits = 1;
        while (p.lane_bits < 5 && 1 << p.lane_bits < units) ++p.lane_bits;
        p.warp_bytes = (int)(n + 1) * 32 * p.v * 4 + 64 * (p.v << p.lane_bits) * element;
        const int all = (int)ceil_div(units, 1 << p.lane_bits), fit = kTableBytes / p.warp_bytes;
        p.warps = fit < 32 ? fit : 32;
        p.slabs = all < p.warps ? all : p.warps;
        p.warps = p.warps / p.slabs * p.slabs;
        p.ctas_y = (int)ceil_div(all, p.slabs);
        const int copies = p.warps / p.slabs;
        // each warp has some blocks of 32 rows, so that its table's way in and out is worth it
        const int64_t need = ceil_div(count, 32 * 4 * (int64_t)copies), most = p.ctas_y < kPlanSms ? kPlanSms / p.ctas_y : 1;
        p.ctas = (int)(need < most ? need : most);
        p.bytes = p.ctas > 1 ? (int64_t)p.ctas * n * c * 4 : 0;
        return p;
    }
    if (count > kRankSorted) {
        int bits = 1;
        while ((n - 1) >> bits) ++bits;
        p.passes = (bits + kMostBits - 1) / kMostBits;
        p.bits = (bits + p.passes - 1) / p.passes < 8 ? 8 : (bits + p.passes - 1) / p.passes;
        // (510952 labels of 5489: 31, 32 and 39 us a sort with 4, 8 and 16; 1000000 of
        // 500000: 88, 67 and 69; above, half as many counts to keep)
        p.items = count <= 262144 ? 4 : count <= 1 << 22 ? 8 : 16;
        p.tiles = count <= kClusterSorted ? 0 : (int)ceil_div(count, 256 * p.items);   // 0: by one cluster
    }
    // chunks long enough that few runs cross them, short enough that they fill the device
    const int64_t want = count * ceil_div(c, 8) / (kPlanSms * 2048);
    const int64_t fit = want < 1 ? 8 : want < 16 ? 16 : want > 256 ? 256 : (want + 7) / 8 * 8;
    // (labels with many entries each: longer ones, so that their runs have fewer parts)
    const int64_t run = count / n / 16;
    p.length = (int)(run > fit ? (run < 128 ? run / 8 * 8 : fit > 128 ? fit : 128) : fit);
    p.chunks = ceil_div(count, p.length);
    p.totals = 256;   // the number of valid entries is in front
    int64_t at = p.totals + (4 << kMostBits);
    p.starts = at;
    at += align256((p.chunks + 1) * 4);
    p.counts = at;
    at += align256(((int64_t)4 << p.bits) * p.tiles);
    p.first = at;
    at += align256(count * (int64_t)sizeof(Entry));
    p.second = at;
    at += p.passes > 1 ? align256(count * (int64_t)sizeof(Entry)) : 0;
    p.part = at;
    at += align256(p.chunks * 2 * (int64_t)c * 4);
    p.bytes = at;
    return p;
}

template <typename T, int V, bool kWhole>
static cudaError_t launch_small(const TableArgs& a, const EmbedPlan& p, cudaStream_t s) {
    int unused = 0;
    const cudaError_t e = pl::kernel_once(
        reinterpret_cast<const void*>(k_small_table<T, V, kWhole>),
        [](int*) {
            return cudaFuncSetAttribute(k_small_table<T, V, kWhole>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTableBytes);
        },
        &unused);
    if (e != cudaSuccess) return e;
    k_small_table<T, V, kWhole><<<dim3(p.ctas, p.ctas_y), p.warps * 32, (size_t)p.warps * p.warp_bytes, s>>>(a);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t small_table(const TableArgs& a, const EmbedPlan& p, cudaStream_t s) {
    const bool whole = aligned16(a.g);   // all rows, then: c is in whole 16 bytes
    if (p.v == 2) return whole ? launch_small<T, 2, true>(a, p, s) : launch_small<T, 2, false>(a, p, s);
    if constexpr (sizeof(T) == 2) return whole ? launch_small<T, 4, true>(a, p, s) : launch_small<T, 4, false>(a, p, s);
    return cudaErrorInvalidValue;
}

// The i-th of `launches` shares of the zeros.
static Zeros zeros_of(void* table, int64_t bytes, int i, int launches) {
    const int64_t all = bytes / 16;
    Zeros z{static_cast<uint4*>(table), all * i / launches, all * (i + 1) / launches, 0};
    const int64_t need = ceil_div(z.end - z.begin, 256 * 4), most = 2 * (int64_t)sm_count();
    z.ctas = (int)(need < most ? need : most);
    return z;
}

template <int kItems, int kDigits>
static void sort_pass(Entry* to, unsigned* counts, unsigned* totals, unsigned* valid, unsigned* starts, const Source& src, int shift,
                      int tiles, const Zeros& first, const Zeros& second, cudaStream_t s) {
    k_sort_count<kItems, kDigits><<<tiles + first.ctas, 256, 0, s>>>(counts, src, shift, tiles, first);
    const bool own = tiles <= kOwnSums;
    if (!own) k_sort_sums<<<kDigits, 256, 0, s>>>(counts, totals, tiles);
    k_sort_place<kItems, kDigits>
        <<<tiles + second.ctas, 256, 0, s>>>(to, counts, own ? nullptr : totals, valid, starts, src, shift, tiles, second);
}

// The labels in order with their positions; `bytes` of the table (a multiple of
// 16) are zeroed on the way.
static const Entry* sort_labels(const EmbedPlan& p, uint8_t* ws, const Labels& ids, int64_t count, int64_t n, void* table, int64_t bytes,
                                cudaError_t* error, cudaStream_t s) {
    unsigned *valid = reinterpret_cast<unsigned*>(ws), *totals = reinterpret_cast<unsigned*>(ws + p.totals),
             *starts = reinterpret_cast<unsigned*>(ws + p.starts), *counts = reinterpret_cast<unsigned*>(ws + p.counts);
    Entry *to = reinterpret_cast<Entry*>(ws + p.first), *other = reinterpret_cast<Entry*>(ws + p.second), *from = nullptr;
    if (p.passes == 0) {
        const Zeros z = zeros_of(table, bytes, 0, 1);
        k_rank_sort<<<(unsigned)ceil_div(count, 64) + z.ctas, 1024, 0, s>>>(to, valid, starts, ids, n, (int)count, z);
        return to;
    }
    if (p.tiles == 0) {
        Zeros z = zeros_of(table, bytes, 0, 1);
        z.ctas = (z.ctas + kSortCtas - 1) / kSortCtas * kSortCtas;
        int unused = 0;
        *error = pl::kernel_once(
            reinterpret_cast<const void*>(k_cluster_sort),
            [](int*) {
                return cudaFuncSetAttribute(k_cluster_sort, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            (32 * ((1 << kMostBits) + 1) + (2 << kMostBits)) * 4);
            },
            &unused);
        const size_t smem = (32 * ((1 << p.bits) + 1) + (2 << p.bits)) * sizeof(unsigned);
        if (*error == cudaSuccess)
            k_cluster_sort<<<kSortCtas + z.ctas, 1024, smem, s>>>(to, other, valid, starts, ids, n, (int)count, p.passes, p.bits, z);
        return p.passes % 2 ? to : other;
    }
    for (int pass = 0; pass < p.passes; ++pass) {
        const Source src{ids, n, count, from, valid};
        const Zeros first = zeros_of(table, bytes, 2 * pass, 2 * p.passes), second = zeros_of(table, bytes, 2 * pass + 1, 2 * p.passes);
        const auto run = p.items == 4   ? (p.bits == 8 ? sort_pass<4, 256> : p.bits == 9 ? sort_pass<4, 512> : sort_pass<4, 1024>)
                         : p.items == 8 ? (p.bits == 8 ? sort_pass<8, 256> : p.bits == 9 ? sort_pass<8, 512> : sort_pass<8, 1024>)
                                        : (p.bits == 8 ? sort_pass<16, 256> : p.bits == 9 ? sort_pass<16, 512> : sort_pass<16, 1024>);
        run(to, counts, totals, valid, starts, src, p.bits * pass, p.tiles, first, second, s);
        from = to;
        to = other;
        other = from;
    }
    return from;
}

template <typename T, int V>
static cudaError_t launch_embed(void* y, const Labels& ids, const void* table, float scale, int64_t count, int64_t n,
                                int c, cudaStream_t s) {
    const int units = c / V;
    int shift = 0;
    while (shift < 8 && 1 << shift < units) ++shift;
    const int64_t ctas = ceil_div(count, (256 >> shift) * kEmbedRows);
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    k_embed<T, V><<<(unsigned)ctas, 256, 0, s>>>(static_cast<T*>(y), ids, static_cast<const T*>(table), scale, count, n, units, shift);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_embed(int v, void* y, const Labels& ids, const void* table, float scale, int64_t count,
                                int64_t n, int c, cudaStream_t s) {
    if (v * sizeof(T) < 8 && aligned16(y)) {
        const int64_t all = count * c, ctas = ceil_div(all, 256 * (16 / (int)sizeof(T)));
        if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
        k_embed_flat<T><<<(unsigned)ctas, 256, 0, s>>>(static_cast<T*>(y), ids, static_cast<const T*>(table), scale, all, n, (unsigned)c);
        return cudaGetLastError();
    }
    if (v * sizeof(T) == 16) return launch_embed<T, 16 / sizeof(T)>(y, ids, table, scale, count, n, c, s);
    if (v == 4) return launch_embed<T, 4>(y, ids, table, scale, count, n, c, s);
    if (v == 2) return launch_embed<T, 2>(y, ids, table, scale, count, n, c, s);
    return launch_embed<T, 1>(y, ids, table, scale, count, n, c, s);
}

template <typename T, int V>
static cudaError_t launch_runs(const RunArgs& a, int64_t chunks, cudaStream_t s) {
    const int units = a.c / V, x = units < 256 ? units : 256;
    // chunks of a CTA: fewer where they are few, so that all SMs have some
    const int64_t spread = ceil_div(chunks, 2 * (int64_t)sm_count());
    const int y = spread < 256 / x ? (int)spread : 256 / x;
    const dim3 grid((unsigned)ceil_div(chunks, y), (unsigned)ceil_div(units, x));
    if (grid.y > 65535) return cudaErrorInvalidValue;
    k_runs<T, V><<<grid, dim3(x, y), 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_runs(int v, const RunArgs& a, int64_t chunks, cudaStream_t s) {
    if (v * sizeof(T) == 16) return launch_runs<T, 16 / sizeof(T)>(a, chunks, s);
    if (v == 4) return launch_runs<T, 4>(a, chunks, s);
    if (v == 2) return launch_runs<T, 2>(a, chunks, s);
    return launch_runs<T, 1>(a, chunks, s);
}

static cudaError_t join_runs(const RunArgs& a, int64_t chunks, cudaStream_t s) {
    const int v = a.c % 4 == 0 ? 4 : 1;
    const bool narrow = a.c <= kJoinNarrow * v;
    int bits = 0;   // lanes of a run
    while (bits < 5 && v << bits < a.c) ++bits;
    const int64_t items = (chunks - 1) * ceil_div(a.c, 32 * v), need = narrow ? ceil_div(items << bits, 32 * kJoinWarps) : items;
    const unsigned grid = (unsigned)(need < 296 ? need : 296);   // one round
    if (v == 4 && narrow) k_join_narrow<4><<<grid, 32 * kJoinWarps, 0, s>>>(a, bits);
    else if (narrow) k_join_narrow<1><<<grid, 32 * kJoinWarps, 0, s>>>(a, bits);
    else if (v == 4) k_join_runs<4><<<grid, 32 * kJoinWarps, 0, s>>>(a, 1 << bits);
    else k_join_runs<1><<<grid, 32 * kJoinWarps, 0, s>>>(a, 1 << bits);
    return cudaGetLastError();
}

static bool embed_ok(long long count, long long n, int c) {
    return count >= 0 && n >= 1 && n <= 0x7fffffff && c >= 1 && c <= (1 << 21) && fits(count, c) && fits(n, c);
}

}  // namespace plr

using namespace plr;

extern "C" {

int plattice_embed(void* y, const void* ids, int ids_wide, const void* table, int dtype, float scale, long long count,
                   long long n, int c, void* stream) {
    if (!dtype_ok(dtype) || !embed_ok(count, n, c) || !std::isfinite(scale)) return PLATTICE_ERR_INVALID;
    if (count == 0) return PLATTICE_OK;
    if (!y || !ids || !table || !on_elements(ids_wide ? 8 : 4, ids) || !on_elements(dtype_size(dtype), y, table))
        return PLATTICE_ERR_INVALID;
    const int v = widest(c, dtype_size(dtype), (uintptr_t)y | (uintptr_t)table);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const Labels l{ids, ids_wide};
    const cudaError_t e = dtype == PLATTICE_F32    ? launch_embed<float>(v, y, l, table, scale, count, n, c, s)
                          : dtype == PLATTICE_BF16 ? launch_embed<__nv_bfloat16>(v, y, l, table, scale, count, n, c, s)
                                                   : launch_embed<__half>(v, y, l, table, scale, count, n, c, s);
    return rows_status(e, "plattice_embed");
}

int plattice_embed_backward_workspace_size(long long count, long long n, int c, size_t* bytes) {
    if (!bytes || !embed_ok(count, n, c) || count > 0x7fffffff) return PLATTICE_ERR_INVALID;
    *bytes = 0;
    for (int element = 2; count && element <= 4; element += 2) {   // of gradients of either size
        const size_t b = (size_t)embed_plan(count, n, c, element).bytes;
        *bytes = b > *bytes ? b : *bytes;
    }
    return PLATTICE_OK;
}

int plattice_embed_backward(void* grad_table, int table_dtype, const void* grad_y, int dtype, const void* ids,
                            int ids_wide, float scale, void* workspace, size_t workspace_bytes, long long count,
                            long long n, int c, void* stream) {
    if (!dtype_ok(dtype) || !dtype_ok(table_dtype) || !std::isfinite(scale) || !embed_ok(count, n, c) || count > 0x7fffffff || !grad_table ||
        !on_elements(dtype_size(table_dtype), grad_table))
        return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (count && (!grad_y || !ids || !on_elements(ids_wide ? 8 : 4, ids) || !on_elements(dtype_size(dtype), grad_y)))
        return PLATTICE_ERR_INVALID;
    const EmbedPlan p = embed_plan(count, n, c, (int)dtype_size(dtype));
    if (count && p.bytes && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < (size_t)p.bytes))
        return PLATTICE_ERR_WORKSPACE;
    const Labels labels{ids, ids_wide};
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    cudaError_t e = cudaSuccess;
    if (count && p.small) {
        const TableArgs a{p.ctas > 1 ? nullptr : grad_table, table_dtype, reinterpret_cast<float*>(ws), labels, grad_y, scale, count, n, c,
                          p.lane_bits, p.slabs, p.warps / p.slabs};
        e = dtype == PLATTICE_F32    ? small_table<float>(a, p, s)
            : dtype == PLATTICE_BF16 ? small_table<__nv_bfloat16>(a, p, s)
                                     : small_table<__half>(a, p, s);
        if (e == cudaSuccess && p.ctas > 1) {
            k_small_join<<<(unsigned)ceil_div(n * c, 32), dim3(32, 8), 0, s>>>(grad_table, table_dtype, a.part, p.ctas, n * c, scale);
            e = cudaGetLastError();
        }
        return rows_status(e, "plattice_embed_backward");
    }
    const size_t bytes = (size_t)n * c * dtype_size(table_dtype), whole = count && aligned16(grad_table) ? bytes / 16 * 16 : 0;
    if (whole < bytes) e = cudaMemsetAsync(static_cast<uint8_t*>(grad_table) + whole, 0, bytes - whole, s);
    if (count == 0 || e != cudaSuccess) return rows_status(e, "plattice_embed_backward");
    unsigned* starts = reinterpret_cast<unsigned*>(ws + p.starts);
    const Entry* sorted = sort_labels(p, ws, labels, count, n, grad_table, (int64_t)whole, &e, s);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) return rows_status(e, "plattice_embed_backward");
    const int v = widest(c, dtype_size(dtype), (uintptr_t)grad_y);
    const RunArgs a{grad_table, table_dtype, reinterpret_cast<float*>(ws + p.part), sorted, reinterpret_cast<unsigned*>(ws), starts, grad_y, scale,
                    count, c, p.length, table_dtype == dtype && widest(c, dtype_size(dtype), (uintptr_t)grad_table) >= v,
                    v * (int)sizeof(float) <= 16 ? c % v == 0 : c % 4 == 0};
    e = dtype == PLATTICE_F32    ? launch_runs<float>(v, a, p.chunks, s)
        : dtype == PLATTICE_BF16 ? launch_runs<__nv_bfloat16>(v, a, p.chunks, s)
                                 : launch_runs<__half>(v, a, p.chunks, s);
    if (e == cudaSuccess && p.chunks > 1) e = join_runs(a, p.chunks, s);
    return rows_status(e, "plattice_embed_backward");
}

}  // extern "C"
