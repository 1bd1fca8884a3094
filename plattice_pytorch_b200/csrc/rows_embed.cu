// rows_embed.cu -- rows from labels and the gradient of their table.
//
//   y[i] = scale table[id_i]            (0 for an id outside the table)
//   grad_table[v] = scale sum_{i: id_i = v} grad_y[i]
//
// The gradient sorts the positions by label (a stable radix sort, 8 bits of the
// label a pass), cuts the sorted list into chunks of equal length and adds each
// chunk's runs of equal labels in registers.  A run inside one chunk is written
// at once; the parts of a run that crosses chunks go to the workspace and are
// added in order by a second kernel.  No atomics: the order of the sums depends
// on the sizes alone.
#include "plattice_runtime.h"
#include "rows_host.h"
#include "rows_vec.cuh"

namespace plr {

constexpr int kEmbedUnits = 4;   // accesses a thread makes

template <typename T, int V>
__global__ void __launch_bounds__(256) k_embed(T* __restrict__ y, Labels ids, const T* __restrict__ table, float scale,
                                               int64_t all, int64_t n, unsigned units) {
    const int64_t base = (int64_t)blockIdx.x * (256 * kEmbedUnits);
    const GroupAt where(base, units);
    Vec<T, V> v[kEmbedUnits];
#pragma unroll
    for (int u = 0; u < kEmbedUnits; ++u) {
        const unsigned o = u * 256 + threadIdx.x;
        v[u].zero();
        if (base + o < all) {
            int64_t row;
            unsigned g;
            where.at(o, row, g);
            const int id = ids.at(row, n);
            if (id >= 0) v[u].load(table + ((int64_t)id * units + g) * V);
        }
    }
#pragma unroll
    for (int u = 0; u < kEmbedUnits; ++u) {
        const unsigned o = u * 256 + threadIdx.x;
        float f[V];
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = v[u].at(i) * scale;
        v[u].from(f);
        if (base + o < all) v[u].store(y + (base + o) * V);
    }
}

// --------------------------------------------------------------- sorting labels

constexpr int kTile = 4096;        // entries that a CTA of the sort takes
constexpr int kDigits = 256;

struct Entry { unsigned label, at; };   // at: the position in ids

// Entries of pass 0 come from the labels themselves (those outside the table
// are left out), later ones from the pass before.
struct Source {
    Labels ids;
    int64_t n, count;
    const Entry* from;        // null: the labels
    const unsigned* valid;    // entries in `from`
    __device__ __forceinline__ int64_t size() const { return from ? (int64_t)*valid : count; }
    // digit of entry i (kDigits: none) and the entry
    __device__ __forceinline__ int get(int64_t i, int64_t size, int shift, Entry& e) const {
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

// counts [digit][tile]
__global__ void __launch_bounds__(256) k_sort_count(unsigned* __restrict__ counts, Source src, int shift, int tiles) {
    __shared__ unsigned h[kDigits + 1];
    h[threadIdx.x] = 0;
    if (threadIdx.x == 0) h[kDigits] = 0;
    __syncthreads();
    const int64_t size = src.size(), base = (int64_t)blockIdx.x * kTile;
    for (int k = 0; k < kTile; k += 256) {
        Entry e;
        atomicAdd(&h[src.get(base + k + threadIdx.x, size, shift, e)], 1u);   // counts: any order
    }
    __syncthreads();
    counts[(int64_t)threadIdx.x * tiles + blockIdx.x] = h[threadIdx.x];
}

// Exclusive sums of m counts by one CTA; the total goes to *valid.
__global__ void __launch_bounds__(1024) k_sort_sums(unsigned* __restrict__ counts, int64_t m, unsigned* valid) {
    __shared__ unsigned warps[32];
    unsigned carry = 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t base = 0; base < m; base += 1024 * 8) {
        const int64_t at = base + (int64_t)threadIdx.x * 8;
        unsigned v[8], sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = at + i < m ? counts[at + i] : 0;
            sum += v[i];
        }
        unsigned s = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const unsigned t = __shfl_up_sync(0xffffffffu, s, d);
            if (lane >= d) s += t;
        }
        if (lane == 31) warps[warp] = s;
        __syncthreads();
        unsigned w = warps[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const unsigned t = __shfl_up_sync(0xffffffffu, w, d);
            if (lane >= d) w += t;
        }
        const unsigned all = __shfl_sync(0xffffffffu, w, 31);
        const unsigned before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);   // the lanes all take part
        unsigned o = carry + (warp ? before : 0) + s - sum;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (at + i < m) counts[at + i] = o;
            o += v[i];
        }
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) *valid = carry;
}

// Stable: a warp takes 512 neighbouring entries of the tile, 32 at a time, and
// counts equal digits before its own by a match.
__global__ void __launch_bounds__(256) k_sort_place(Entry* __restrict__ out, const unsigned* __restrict__ offsets,
                                                    Source src, int shift, int tiles) {
    __shared__ unsigned h[8][kDigits + 1];
    for (int i = threadIdx.x; i < 8 * (kDigits + 1); i += 256) (&h[0][0])[i] = 0;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t size = src.size(), base = (int64_t)blockIdx.x * kTile + warp * 512;
    Entry e[16];
    int digit[16];
    unsigned rank[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) digit[k] = src.get(base + k * 32 + lane, size, shift, e[k]);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const unsigned same = __match_any_sync(0xffffffffu, digit[k]);
        const unsigned had = h[warp][digit[k]];
        rank[k] = had + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if ((same & ((1u << lane) - 1)) == 0) h[warp][digit[k]] = had + __popc(same);
        __syncwarp();
    }
    __syncthreads();
    unsigned o = offsets[(int64_t)threadIdx.x * tiles + blockIdx.x];
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        const unsigned had = h[w][threadIdx.x];
        h[w][threadIdx.x] = o;
        o += had;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
        if (digit[k] < kDigits) out[h[warp][digit[k]] + rank[k]] = e[k];
}

// ------------------------------------------------------------------ sums of runs

struct RunArgs {
    void* out;
    int out_dtype;
    float* part;              // [chunks][2][c]: of a run that came from before; that goes on behind
    const Entry* sorted;
    const unsigned* valid;
    const void* g;
    float scale;
    int c, length;            // length: entries of a chunk
};

// A thread's V channels of the entries of one chunk.  blockDim: (lanes of a row, chunks of a CTA).
template <typename T, int V>
__global__ void __launch_bounds__(256) k_runs(RunArgs a) {
    const int64_t valid = *a.valid;
    const int64_t chunk = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int64_t begin = chunk * a.length;
    const int64_t col = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V;
    if (begin >= valid || col >= a.c) return;
    const int64_t end = begin + a.length < valid ? begin + a.length : valid;
    const T* g = static_cast<const T*>(a.g) + col;
    unsigned label = a.sorted[begin].label;
    bool head = begin > 0 && a.sorted[begin - 1].label == label;
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
    const auto out = [&](bool tail) {
        if (head || tail) {
            float* p = a.part + (chunk * 2 + (head ? 0 : 1)) * a.c + col;
#pragma unroll
            for (int j = 0; j < V; ++j) p[j] = acc[j];
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                store_param(a.out, a.out_dtype, (int64_t)label * a.c + col + j, acc[j] * a.scale);
        }
    };
    for (int64_t i = begin; i < end; i += 8) {
        Entry e[8];
        Vec<T, V> v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            e[k].label = label;
            if (i + k < end) {
                e[k] = a.sorted[i + k];
                v[k].load(g + (int64_t)e[k].at * a.c);
            } else {
                v[k].zero();
                if (k) e[k].label = e[k - 1].label;
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (e[k].label != label) {
                out(false);
                label = e[k].label;
                head = false;
#pragma unroll
                for (int j = 0; j < V; ++j) acc[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += v[k].at(j);
        }
    }
    out(end < valid && a.sorted[end].label == label);
}

// The runs that begin in a chunk and go on behind it: its part and those of the
// chunks up to the run's end, which a search of the sorted list finds.
// blockDim (32 channels, 8): each of the 8 adds every 8th part, then they are
// added in order.
__global__ void __launch_bounds__(256) k_join_runs(RunArgs a) {
    __shared__ float sums[8][32];
    const int64_t valid = *a.valid, chunk = blockIdx.x, end = (chunk + 1) * a.length;
    if (end >= valid) return;
    const unsigned label = a.sorted[end].label;
    if (a.sorted[end - 1].label != label) return;
    const int64_t begin = chunk * a.length;
    if (a.sorted[begin].label == label && begin > 0 && a.sorted[begin - 1].label == label) return;   // began earlier
    int64_t lo = end, hi = valid;   // the run ends at the first entry of another label: lo < it <= hi
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (a.sorted[mid].label == label) lo = mid;
        else hi = mid;
    }
    const int64_t parts = (lo / a.length) - chunk;   // chunks behind this one
    const int64_t col = (int64_t)blockIdx.y * 32 + threadIdx.x;
    float s = 0.f;
    if (col < a.c) {
        if (threadIdx.y == 0) s = a.part[(chunk * 2 + 1) * a.c + col];
        for (int64_t j = 1 + threadIdx.y; j <= parts; j += 8) s += a.part[(chunk + j) * 2 * a.c + col];
    }
    sums[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && col < a.c) {
#pragma unroll
        for (int k = 1; k < 8; ++k) s += sums[k][threadIdx.x];
        store_param(a.out, a.out_dtype, (int64_t)label * a.c + col, s * a.scale);
    }
}

// ------------------------------------------------------------------ host side

static int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }

struct EmbedPlan {
    int passes, tiles, length;
    int64_t chunks;
    int64_t valid, counts, first, second, part, bytes;   // offsets in the workspace
};

static EmbedPlan embed_plan(int64_t count, int64_t n, int c) {
    EmbedPlan p = {};
    while (p.passes < 4 && (n - 1) >> (8 * p.passes)) ++p.passes;
    if (p.passes == 0) p.passes = 1;
    p.tiles = (int)ceil_div(count, kTile);
    // chunks long enough that few runs cross them, short enough that they fill the device
    const int64_t want = count * ceil_div(c, 8) / (148 * 2048);
    p.length = (int)(want < 16 ? 16 : want > 256 ? 256 : (want + 7) / 8 * 8);
    p.chunks = ceil_div(count, p.length);
    int64_t at = 256;   // the number of valid entries is in front
    p.counts = at;
    at += align256((int64_t)kDigits * p.tiles * 4);
    p.first = at;
    at += align256(count * (int64_t)sizeof(Entry));
    p.second = at;
    at += p.passes > 1 ? align256(count * (int64_t)sizeof(Entry)) : 0;
    p.part = at;
    at += align256(p.chunks * 2 * (int64_t)c * 4);
    p.bytes = at;
    return p;
}

template <typename T, int V>
static cudaError_t launch_embed(void* y, const Labels& ids, const void* table, float scale, int64_t count, int64_t n,
                                int c, cudaStream_t s) {
    const int64_t all = count * (c / V), ctas = ceil_div(all, 256 * kEmbedUnits);
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    k_embed<T, V><<<(unsigned)ctas, 256, 0, s>>>(static_cast<T*>(y), ids, static_cast<const T*>(table), scale, all, n,
                                                 (unsigned)(c / V));
    return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_embed(int v, void* y, const Labels& ids, const void* table, float scale, int64_t count,
                                int64_t n, int c, cudaStream_t s) {
    if (v * sizeof(T) == 16) return launch_embed<T, 16 / sizeof(T)>(y, ids, table, scale, count, n, c, s);
    if (v == 4) return launch_embed<T, 4>(y, ids, table, scale, count, n, c, s);
    if (v == 2) return launch_embed<T, 2>(y, ids, table, scale, count, n, c, s);
    return launch_embed<T, 1>(y, ids, table, scale, count, n, c, s);
}

template <typename T, int V>
static cudaError_t launch_runs(const RunArgs& a, int64_t chunks, cudaStream_t s) {
    const int units = a.c / V;
    int x = 1;
    while (x < units && x < 256) x <<= 1;
    const int y = 256 / x;
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

static bool embed_ok(long long count, long long n, int c) {
    return count >= 0 && n >= 1 && n <= 0x7fffffff && c >= 1 && c <= (1 << 21) && fits(count, c) && fits(n, c);
}

}  // namespace plr

using namespace plr;

extern "C" {

int plattice_embed(void* y, const void* ids, int ids_wide, const void* table, int dtype, float scale, long long count,
                   long long n, int c, void* stream) {
    if (!dtype_ok(dtype) || !embed_ok(count, n, c)) return PLATTICE_ERR_INVALID;
    if (count == 0) return PLATTICE_OK;
    if (!y || !ids || !table || (uintptr_t)ids % (ids_wide ? 8 : 4)) return PLATTICE_ERR_INVALID;
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
    *bytes = count ? (size_t)embed_plan(count, n, c).bytes : 0;
    return PLATTICE_OK;
}

int plattice_embed_backward(void* grad_table, int table_dtype, const void* grad_y, int dtype, const void* ids,
                            int ids_wide, float scale, void* workspace, size_t workspace_bytes, long long count,
                            long long n, int c, void* stream) {
    if (!dtype_ok(dtype) || !dtype_ok(table_dtype) || !embed_ok(count, n, c) || count > 0x7fffffff || !grad_table)
        return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (count && (!grad_y || !ids || (uintptr_t)ids % (ids_wide ? 8 : 4))) return PLATTICE_ERR_INVALID;
    const EmbedPlan p = embed_plan(count, n, c);
    if (count && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < (size_t)p.bytes))
        return PLATTICE_ERR_WORKSPACE;
    cudaError_t e = cudaMemsetAsync(grad_table, 0, (size_t)n * c * dtype_size(table_dtype), s);
    if (count == 0 || e != cudaSuccess) return rows_status(e, "plattice_embed_backward");
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    unsigned* valid = reinterpret_cast<unsigned*>(ws);
    unsigned* counts = reinterpret_cast<unsigned*>(ws + p.counts);
    Entry *from = nullptr, *to = reinterpret_cast<Entry*>(ws + p.first),
          *other = reinterpret_cast<Entry*>(ws + p.second);
    for (int pass = 0; pass < p.passes; ++pass) {
        const Source src{{ids, ids_wide}, n, count, from, valid};
        k_sort_count<<<p.tiles, 256, 0, s>>>(counts, src, 8 * pass, p.tiles);
        k_sort_sums<<<1, 1024, 0, s>>>(counts, (int64_t)kDigits * p.tiles, valid);
        k_sort_place<<<p.tiles, 256, 0, s>>>(to, counts, src, 8 * pass, p.tiles);
        from = to;
        to = other;
        other = from;
    }
    e = cudaGetLastError();
    if (e != cudaSuccess) return rows_status(e, "plattice_embed_backward");
    const RunArgs a{grad_table, table_dtype, reinterpret_cast<float*>(ws + p.part), from, valid, grad_y, scale, c, p.length};
    const int v = widest(c, dtype_size(dtype), (uintptr_t)grad_y);
    e = dtype == PLATTICE_F32    ? launch_runs<float>(v, a, p.chunks, s)
        : dtype == PLATTICE_BF16 ? launch_runs<__nv_bfloat16>(v, a, p.chunks, s)
                                 : launch_runs<__half>(v, a, p.chunks, s);
    if (e == cudaSuccess && p.chunks > 1) {
        k_join_runs<<<dim3((unsigned)(p.chunks - 1), (unsigned)ceil_div(c, 32)), dim3(32, 8), 0, s>>>(a);
        e = cudaGetLastError();
    }
    return rows_status(e, "plattice_embed_backward");
}

}  // extern "C"
