// rows_mma.cuh -- the products of the linear map on the tensor cores
// (tcgen05, operands by TMA, accumulators in tensor memory).
//
//   D[i][j] = sum over r of A(i, r) B(j, r)
//
// in three kinds, by what i, j, r are and along which index each operand is
// contiguous ("K-major": along the sum; "MN-major": along the result):
//   kForward   i row, j output channel, r input channel   A = x   K   B = w   K
//   kGradX     i row, j input channel,  r output channel  A = gz  K   B = w   MN
//   kGradW     i input channel, j output channel, r row   A = x   MN  B = gz  MN
// so no operand is ever transposed in memory.
//
// Operands are 16-bit.  float32 operands come as three bfloat16 parts whose
// sum is the value (8 + 8 + 8 significant bits); the six products of parts
// down to 2^-16 of the largest are added, the small ones first.  8-bit rows
// come unpacked to bfloat16 (exact).
//
// One CTA per SM walks over 128 x kBN tiles of D (times parts of the sum for
// kGradW): one thread issues TMA copies of 64-deep slices into a ring of
// stages, one issues the MMAs, the epilogue's warps empty the other of two
// accumulators (activation, residual, stores) meanwhile.  Bound by the tensor
// cores where the sum is deep (8192 x 8192 x 8192 in bfloat16: 832 us, 1321
// TFLOP/s; the input gradient of 32768 x 1024 -> 4096: 177 us, 1553), by the
// epilogue where it is not (its forward with gelu, residual and kept z: 302 us,
// plain 215), by HBM where K and n are small (262144 x 64 -> 64: 17 us, 67 MB).  Every wait is
// bounded: a wait that gives up ends all roles, copies and MMAs in flight are
// waited for, tensor memory is freed and the call's failure is reported.
#pragma once
#include <cuda.h>
#include <limits.h>

#include "plattice_runtime.h"
#include "rows_common.cuh"
#include "rows_host.h"

namespace plr {

constexpr int kStageA = kBM * kBK * 2;

// What an epilogue is compiled for: rows of any alignment, everything looked
// up at run time; rows on 16-byte boundaries; those without activation,
// residual, split and kept pre-activation.  (Control flow that asks for each of
// these at every 16 columns cost a third of a plain forward's time.)
enum Mode { kAny = 0, kAligned = 1, kPlain = 2 };

// Warps that empty accumulators.  The forward's work per output (activation,
// residual, 8-bit codes) waits more than it issues: 16 warps hide what 8 do
// not (422 against 353 us at 32768 x 1024 -> 4096, gelu, residual, kept z).
// For the plain stores of the gradients 8 do.
__host__ __device__ constexpr int epilogue_warps(int kind, bool chunked) { return kind == 0 || chunked ? 16 : 8; }
__host__ __device__ constexpr int role_threads(int kind, bool chunked) { return 64 + 32 * epilogue_warps(kind, chunked); }

// A float32 result of a deep sum, and a 16-bit one of a far deeper (deepest_sum):
// kChunked.  The MMA cuts where an addition rounds, so that an accumulator drifts
// by about 2^-26 of itself with each of them, terms of both signs (1.1e-6 of the
// result at a depth of 1024, 4.5e-6 at 4096; float16 terms of one sign: 2^-23).
// The sum then goes in chunks of kChunk slices through the two accumulators, and
// the epilogue adds those in registers, rounding; a warp holds one 32-column
// piece, so tiles are at most 128 wide.
constexpr int kChunk = 8;

__host__ __device__ constexpr bool a_mn(int kind) { return kind == kGradW; }
__host__ __device__ constexpr bool b_mn(int kind) { return kind != kForward; }
// MN-major slices come in groups of 64 columns
__host__ __device__ constexpr int b_columns(int kind, int bn) { return b_mn(kind) && bn < 64 ? 64 : bn; }
__host__ __device__ constexpr int stage_bytes(int kind, int bn) { return kStageA + b_columns(kind, bn) * kBK * 2; }
constexpr int kWarpStaging = 32 * 16 * 4 + 32 * 4;   // a 32 x 16 float tile and 32 biases
__host__ __device__ constexpr int fixed_smem(int kind, bool chunked) {
    return 1024 + epilogue_warps(kind, chunked) * kWarpStaging + 256;
}
__host__ __device__ constexpr int stages(int kind, int bn, bool chunked) {
    const int n = (kMaxSmem - 16 - fixed_smem(kind, chunked)) / stage_bytes(kind, bn);
    return n > 8 ? 8 : n;
}
__host__ __device__ constexpr int smem_bytes(int kind, int bn, bool chunked) {
    return fixed_smem(kind, chunked) + stages(kind, bn, chunked) * stage_bytes(kind, bn);
}

// ------------------------------------------------------------- PTX wrappers

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, int bytes) {
    asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, int parity) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}

// Waits for the phase; false when another role has given up or the wait itself
// does, after `patience` clock cycles: about two seconds, and more than a sum takes
// as a whole (an accumulator is full when all of its slices are in: 2^24 of them
// take three seconds).
__device__ __forceinline__ bool bar_wait(uint32_t bar, int parity, long long patience, volatile int* dead) {
    if (bar_try(bar, parity)) return true;
    const long long begin = clock64();
    for (long long i = 0; i < patience; ++i) {   // a try takes a cycle at least
        if (bar_try(bar, parity)) return true;
        if ((i & 15) == 15 && (*dead || clock64() - begin > patience)) break;
    }
    *dead = 1;
    return false;
}

// The same for all lanes of a warp, with one answer.
__device__ __forceinline__ bool warp_wait(uint32_t bar, int parity, long long patience, volatile int* dead) {
    return __all_sync(0xffffffffu, bar_wait(bar, parity, patience, dead));
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_load16(float (&v)[16], uint32_t addr) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_load32(float (&v)[32], uint32_t addr) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Shared-memory operand descriptor of a slice in the 128-byte swizzle: 8-row
// groups of 128 bytes lie 1024 bytes apart (along i for K-major, along r for
// MN-major slices); MN-major groups of 64 columns lie 64 rows = 8192 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool mn) {
    const uint64_t lead = mn ? 8192 >> 4 : 1;
    return (uint64_t)((addr & 0x3ffff) >> 4) | (lead << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// ------------------------------------------------------------------- tiles

struct Tile {
    int64_t i0, j0;
    int part, begin, end;   // slices [begin, end) of the sum
};

// Tiles of a part are numbered in bands of kBand columns of tiles, along j
// first: the tiles that run at a time then form a block about as high as it is
// wide (148 SMs: 12 x 12 of 128 x 256), which shares most of the slices it
// reads.  Parts of the sum come one after the other.
constexpr unsigned kBand = 12;

template <int kBN>
__device__ __forceinline__ Tile tile_at(const MmaArgs& p, unsigned t) {
    const unsigned nj = (unsigned)((p.nj + kBN - 1) / kBN), ni = (unsigned)((p.ni + kBM - 1) / kBM);
    Tile r;
    r.part = 0;
    if (p.parts > 1) {
        r.part = (int)(t / (ni * nj));
        t -= r.part * (ni * nj);
    }
    unsigned first = 0, width = nj;
    if (nj > kBand + kBand / 2) {   // up to there one band
        first = t / (ni * kBand) * kBand;
        t -= first * ni;
        width = min(kBand, nj - first);
    }
    const unsigned i = t / width;
    r.i0 = (int64_t)i * kBM;
    r.j0 = (int64_t)(first + t - i * width) * kBN;
    r.begin = r.part * p.part_steps;
    r.end = min(p.steps, r.begin + p.part_steps);
    return r;
}

// ---------------------------------------------------------------- epilogue

template <int kOut> struct OutType { typedef float type; };
template <> struct OutType<PLATTICE_BF16> { typedef __nv_bfloat16 type; };
template <> struct OutType<PLATTICE_F16> { typedef __half type; };

// Half a warp's 32 x 32 tile in shared memory, 16 columns: float4 c of row r at
// slot c ^ ((r >> 1) & 3), free of bank conflicts both a row per lane and two
// lanes a row.
__device__ __forceinline__ float4* staged(float* s, int row, int c4) {
    return reinterpret_cast<float4*>(s) + row * 4 + (c4 ^ ((row >> 1) & 3));
}
__device__ __forceinline__ float staged_at(const float* s, int row, int c) {
    return s[row * 16 + (((c >> 2) ^ ((row >> 1) & 3)) << 2) + (c & 3)];
}

__device__ __forceinline__ void stage_rows(float* s, const float* v, int lane) {
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; ++c) *staged(s, lane, c) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
    __syncwarp();
}

// 32 x 32 of the residual as store_aligned's lanes take them, loaded a piece
// ahead: a load waited for at each store would cost a trip to HBM four times a
// piece (652 us against 422 at 32768 x 1024 -> 4096, gelu, residual, kept z).
struct Ahead {
    uint4 r[4];   // twice 8 columns of each half, of a 16-bit type (float32 is loaded at the store)
    bool have;
};

template <int kOut>
__device__ __forceinline__ void load_ahead(Ahead& a, const MmaArgs& p, int64_t row0, int64_t col0, int lane) {
    a.have = kOut != PLATTICE_F32 && p.residual && col0 + 32 <= p.nj && row0 + 32 <= p.ni;
    if (!a.have) return;
    const uint16_t* src = static_cast<const uint16_t*>(p.residual) + (row0 + (lane >> 1)) * p.nj + col0 + (lane & 1) * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) a.r[i] = *reinterpret_cast<const uint4*>(src + (i & 1) * 16 * p.nj + (i >> 1) * 16);
}

// 16 columns of 32 rows (a row per lane) to (row0, col0) of an [ni][nj] tensor,
// `add` (the residual, same layout) added: through the staging to two lanes a
// row, 8 columns each.  nj is a multiple of 8: a lane's columns all exist or
// none does.
template <int kOut, int kHalf = 0>
__device__ __forceinline__ void store_aligned(float* s, const float* v, void* dst, const MmaArgs& p, int64_t row0,
                                              int64_t col0, const void* add, const Ahead& ahead, int lane) {
    typedef typename OutType<kOut>::type T;
    const int rows = (int)min((int64_t)32, p.ni - row0), c = (lane & 1) * 8;
    const bool have = col0 + c < p.nj;
    T* out = static_cast<T*>(dst) + (row0 + (lane >> 1)) * p.nj + col0 + c;
    if constexpr (sizeof(T) == 2) {
        if (!add) {   // rounded before the staging: half its traffic.  Row r's two
                      // 16-byte slots change places with r >> 2: no bank conflicts
            uint4* q = reinterpret_cast<uint4*>(s);
            union { uint4 u[2]; typename Pair<T>::type h[8]; } o;
#pragma unroll
            for (int i = 0; i < 8; ++i) pair_from(o.h[i], v[2 * i], v[2 * i + 1]);
            __syncwarp();
            q[lane * 2 + ((lane >> 2) & 1)] = o.u[0];
            q[lane * 2 + (((lane >> 2) & 1) ^ 1)] = o.u[1];
            __syncwarp();
#pragma unroll
            for (int it = 0; it < 2; ++it) {
                const int r = it * 16 + (lane >> 1);
                if (r < rows && have)
                    *reinterpret_cast<uint4*>(out + (int64_t)it * 16 * p.nj) = q[r * 2 + ((lane & 1) ^ ((r >> 2) & 1))];
            }
            return;
        }
    }
    stage_rows(s, v, lane);
#pragma unroll
    for (int it = 0; it < 2; ++it) {
        const int r = it * 16 + (lane >> 1);
        if (r >= rows || !have) continue;
        const float4 a = *staged(s, r, c >> 2), b = *staged(s, r, (c >> 2) + 1);
        float o[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        if (add) {
            Raw8<T> q;
            float t[8];
            if constexpr (sizeof(T) == 2) {
                if (ahead.have) q.u = ahead.r[kHalf * 2 + it];
                else q.load(static_cast<const T*>(add) + (out - static_cast<T*>(dst)) + (int64_t)it * 16 * p.nj, true, 8);
            } else {
                q.load(static_cast<const T*>(add) + (out - static_cast<T*>(dst)) + (int64_t)it * 16 * p.nj, true, 8);
            }
            q.widen(t);
#pragma unroll
            for (int i = 0; i < 8; i += 2) add2(o[i], o[i + 1], t[i], t[i + 1]);
        }
        store8(out + (int64_t)it * 16 * p.nj, o, true, 8);
    }
}

// The same where rows lie on no 16-byte boundaries: a lane per column, two
// rows at a time, all of the residual's loads before the first store.
template <typename T>
__device__ __forceinline__ void store_any_as(const float* s, T* dst, const MmaArgs& p, int64_t row0, int64_t col0,
                                             const T* add, int lane) {
    const int rows = (int)min((int64_t)32, p.ni - row0) - (lane >> 4);   // of this lane, every second
    const int64_t col = col0 + (lane & 15), at = (row0 + (lane >> 4)) * p.nj + col;
    if (col >= p.nj) return;
    T* out = dst + at;
    const int64_t step = 2 * p.nj;
    float x[16];
    if (add) {
        const T* in = add + at;
#pragma unroll
        for (int i = 0; i < 16; ++i, in += step) x[i] = 2 * i < rows ? to_f32(*in) : 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i, out += step)
        if (2 * i < rows) *out = from_f32<T>(x[i] + staged_at(s, (lane >> 4) + 2 * i, lane & 15));
}

__device__ __forceinline__ void store_any(float* s, const float* v, void* dst, const MmaArgs& p, int64_t row0,
                                          int64_t col0, const void* add, int lane) {
    stage_rows(s, v, lane);
    if (p.out_dtype == PLATTICE_F32)
        store_any_as(s, static_cast<float*>(dst), p, row0, col0, static_cast<const float*>(add), lane);
    else if (p.out_dtype == PLATTICE_BF16)
        store_any_as(s, static_cast<__nv_bfloat16*>(dst), p, row0, col0, static_cast<const __nv_bfloat16*>(add), lane);
    else
        store_any_as(s, static_cast<__half*>(dst), p, row0, col0, static_cast<const __half*>(add), lane);
}

// Two tensors of a split: columns below `split` and the others.
__device__ __forceinline__ void store_split(float* s, const float* v, const MmaArgs& p, int64_t row0,
                                            int64_t col0, int lane) {
    stage_rows(s, v, lane);
    const int rows = (int)min((int64_t)32, p.ni - row0), c = lane & 15;
    const int64_t col = col0 + c;
    if (col >= p.nj) return;
    for (int r = lane >> 4; r < rows; r += 2) {
        const float x = staged_at(s, r, c);
        if (col < p.split) store_param(p.y0, p.out_dtype, (row0 + r) * p.split + col, x);
        else store_param(p.y1, p.out_dtype, (row0 + r) * (p.nj - p.split) + col - p.split, x);
    }
}

__device__ __forceinline__ void add_bias(float* v, const float* sb) {
#pragma unroll
    for (int c = 0; c < 16; c += 4) {
        const float4 b = *reinterpret_cast<const float4*>(sb + c);
        add2(v[c], v[c + 1], b.x, b.y);
        add2(v[c + 2], v[c + 3], b.z, b.w);
    }
}

// A row's 32 columns, one block of the kept 8-bit rows: its codes and scale, a
// lane's 32 bytes in one store (whole sectors).
__device__ __forceinline__ void keep_codes(const float (&v)[32], const MmaArgs& p, int64_t row, int64_t col0) {
    bool infinite;
    const int e = block_exponent(finite_amax_of(v, infinite));
    if (row >= p.ni) return;
    const float inv = pow2(-e);
    uint2 q[4];
    codes_of(q, v, inv, infinite);
    const int64_t at = row * ((p.nj + 31) / 32) + (col0 >> 5);
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(static_cast<uint8_t*>(p.z) + at * 32),
                 "r"(q[0].x), "r"(q[0].y), "r"(q[1].x), "r"(q[1].y), "r"(q[2].x), "r"(q[2].y), "r"(q[3].x), "r"(q[3].y)
                 : "memory");
    p.z_scale[at] = (uint8_t)(e + 127);
}

// A 32-column piece of the forward, a row per lane, with whatever is asked for.
template <int kOut, int kMode>
__device__ __forceinline__ void finish32(float (&v)[32], const MmaArgs& p, int64_t row0, int64_t col0, float* s,
                                         const Ahead& ahead, int lane) {
    if (p.bias) {
        add_bias(v, s + 32 * 16);
        add_bias(v + 16, s + 32 * 16 + 16);
    }
    const bool second = col0 + 16 < p.nj;
    if (p.z_scale) {
        if (col0 + 32 > p.nj) {   // zeros behind the last column (a row that is not finite makes NaN there)
            const int left = (int)(p.nj - col0);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = i < left ? v[i] : 0.f;
        }
        keep_codes(v, p, row0 + lane, col0);
    } else if (p.z) {
        if (kMode == kAligned) store_aligned<kOut>(s, v, p.z, p, row0, col0, nullptr, ahead, lane);
        else store_any(s, v, p.z, p, row0, col0, nullptr, lane);
        if (kMode == kAligned && second) store_aligned<kOut>(s, v + 16, p.z, p, row0, col0 + 16, nullptr, ahead, lane);
        else if (second) store_any(s, v + 16, p.z, p, row0, col0 + 16, nullptr, lane);
    }
    activate(v, p.act);
    if (kMode == kAligned) {
        store_aligned<kOut, 0>(s, v, p.y0, p, row0, col0, p.residual, ahead, lane);
        if (second) store_aligned<kOut, 1>(s, v + 16, p.y0, p, row0, col0 + 16, p.residual, ahead, lane);
    } else if (p.split) {
        store_split(s, v, p, row0, col0, lane);
        if (second) store_split(s, v + 16, p, row0, col0 + 16, lane);
    } else {
        store_any(s, v, p.y0, p, row0, col0, p.residual, lane);
        if (second) store_any(s, v + 16, p.y0, p, row0, col0 + 16, p.residual, lane);
    }
}

// Half a 32-column piece (16 columns from col0) of a plain forward or a
// gradient, a row per lane.
template <int kKind, int kOut, int kMode>
__device__ __forceinline__ void finish16(float (&v)[16], const MmaArgs& p, const Tile& t, int64_t row0, int64_t col0,
                                         float* s, int half, int lane) {
    typedef typename OutType<kOut>::type T;
    if (kKind == kGradW) {
        // D is [input channel][output channel], its result [output channel]
        // [input channel]: a lane per input channel stores whole lines
        const int64_t i = row0 + lane;
        if (i >= p.ni) return;
        const int left = (int)min((int64_t)16, p.nj - col0);
        T* out = static_cast<T*>(p.y0) + ((int64_t)t.part * p.nj + col0) * p.ni + i;
#pragma unroll
        for (int c = 0; c < 16; ++c, out += p.ni)
            if (c < left) *out = from_f32<T>(v[c]);
        return;
    }
    if (kKind == kForward && p.bias) add_bias(v, s + 32 * 16 + half * 16);
    if (kMode == kPlain) store_aligned<kOut>(s, v, p.y0, p, row0, col0, nullptr, Ahead{}, lane);
    else store_any(s, v, p.y0, p, row0, col0, nullptr, lane);
}

// -------------------------------------------------------------- the kernel

// kOut: the type of y0 (kAny: looked up).
template <int kKind, int kBN, int kOut, int kMode, bool kChunked>
__global__ void __launch_bounds__(role_threads(kKind, kChunked), 1)
    k_mma(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const MmaArgs p,
          unsigned tiles) {
    constexpr int kStages = stages(kKind, kBN, kChunked), kEpilogueWarps = epilogue_warps(kKind, kChunked);
    constexpr bool kKeeps = kKind == kForward && kMode != kPlain;   // a kept pre-activation, a residual
    constexpr int kGroups = kEpilogueWarps / 4;   // warps that share 32 accumulator rows
    constexpr int kStage = stage_bytes(kKind, kBN);
    constexpr int kColumns = 2 * kBN;   // tensor memory: two accumulators
    extern __shared__ char smem_raw[];
    __shared__ uint32_t tmem_slot;
    __shared__ int dead_flag;
    volatile int* dead = &dead_flag;

    char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    const uint32_t ring = smem_addr(smem);
    float* staging = reinterpret_cast<float*>(smem + kStages * kStage);
    const uint32_t bars = smem_addr(smem + kStages * kStage + kEpilogueWarps * kWarpStaging);
    auto full = [&](int s) { return bars + 8 * s; };
    auto empty = [&](int s) { return bars + 8 * (kStages + s); };
    auto acc_full = [&](int b) { return bars + 8 * (2 * kStages + b); };
    auto acc_empty = [&](int b) { return bars + 8 * (2 * kStages + 2 + b); };
    const uint32_t drained = bars + 8 * (2 * kStages + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        dead_flag = 0;
        for (int s = 0; s < kStages; ++s) {
            bar_init(full(s), 1);
            bar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            bar_init(acc_full(b), 1);
            bar_init(acc_empty(b), kEpilogueWarps);
        }
        bar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)),
                     "r"(kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        // ---- TMA copies
        if (lane == 0) {
            int s = 0, phase = 0, issued = 0;
            for (unsigned t = blockIdx.x; t < tiles && !*dead; t += gridDim.x) {
                const Tile tile = tile_at<kBN>(p, t);
                for (int from = tile.begin; from < tile.end; from += kChunked ? kChunk : tile.end - tile.begin) {
                const int to = kChunked ? min(tile.end, from + kChunk) : tile.end;
                for (int pair = 0; pair < p.pairs; ++pair) {
                    const int za = (p.pairs_a >> (2 * pair)) & 3, zb = (p.pairs_b >> (2 * pair)) & 3;
                    for (int k = from; k < to; ++k) {
                        if (!bar_wait(empty(s), phase ^ 1, p.patience, dead)) goto copies_done;
                        const uint32_t a = ring + s * kStage, b = a + kStageA;
                        bar_expect(full(s), kStageA + b_columns(kKind, kBN) * kBK * 2);
                        if (a_mn(kKind)) {
                            for (int g = 0; g < kBM / 64; ++g)
                                tma_load(a + g * 8192, &map_a, full(s), (int)tile.i0 + g * 64, k * kBK, za);
                        } else {
                            tma_load(a, &map_a, full(s), k * kBK, (int)tile.i0, za);
                        }
                        if (b_mn(kKind)) {
                            for (int g = 0; g < b_columns(kKind, kBN) / 64; ++g)
                                tma_load(b + g * 8192, &map_b, full(s), (int)tile.j0 + g * 64, k * kBK, zb);
                        } else {
                            tma_load(b, &map_b, full(s), k * kBK, (int)tile.j0, zb);
                        }
                        ++issued;
                        if (++s == kStages) s = 0, phase ^= 1;
                    }
                }
                }
            }
        copies_done:
            if (*dead) {   // no thread leaves while a copy may still write here
                for (int b = issued < kStages ? issued : kStages; b > 0; --b) {
                    const int n = issued - b, at = n % kStages, par = (n / kStages) & 1;
                    const long long begin = clock64();
                    while (!bar_try(full(at), par) && clock64() - begin < 200000000ll) {}
                }
            }
        }
    } else if (warp == 1) {
        // ---- MMAs.  All lanes walk the loop, so that what the instructions take
        // stays in uniform registers, and one lane issues them: a slice of a
        // narrow tile costs 360 cycles instead of 495 (2560 x 4096 -> 64: 20.4 ->
        // 15.6 us).  The copies' warp is the faster with one lane alone (16.5).
        const bool leader = elect_one();
        const uint32_t fmt = p.half ? 0u : 1u;
        const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)a_mn(kKind) << 15) |
                               ((uint32_t)b_mn(kKind) << 16) | ((uint32_t)(kBN >> 3) << 17) |
                               ((uint32_t)(kBM >> 4) << 24);
        constexpr int kStepA = (a_mn(kKind) ? 2048 : 32) >> 4, kStepB = (b_mn(kKind) ? 2048 : 32) >> 4;
        int s = 0, phase = 0, n = 0;
        bool going = true;
        for (unsigned t = blockIdx.x; t < tiles && going; t += gridDim.x) {
            const Tile tile = tile_at<kBN>(p, t);
            for (int from = tile.begin; from < tile.end && going; ++n) {
                const int to = kChunked ? min(tile.end, from + kChunk) : tile.end, buf = n & 1;
                if (!warp_wait(acc_empty(buf), ((n >> 1) & 1) ^ 1, p.patience, dead)) {
                    going = false;
                    break;
                }
                fence_after();
                const uint32_t d = tmem + buf * kBN;
                const int count = p.pairs * (to - from);
                from = to;
                for (int k = 0; k < count; ++k) {
                    if (!warp_wait(full(s), phase, p.patience, dead)) {
                        going = false;
                        break;
                    }
                    fence_after();
                    if (leader) {
                        const uint64_t a = operand_desc(ring + s * kStage, a_mn(kKind));
                        const uint64_t b = operand_desc(ring + s * kStage + kStageA, b_mn(kKind));
#pragma unroll
                        for (int u = 0; u < kBK / 16; ++u)
                            mma_f16(d, a + u * kStepA, b + u * kStepB, idesc, k > 0 || u > 0);
                        mma_commit(empty(s));
                    }
                    __syncwarp();
                    if (++s == kStages) s = 0, phase ^= 1;
                }
                if (going && leader) mma_commit(acc_full(buf));
                __syncwarp();
            }
        }
        if (leader && *dead) {   // MMAs in flight end before the shared memory they read goes
            mma_commit(drained);
            const long long begin = clock64();
            while (!bar_try(drained, 0) && clock64() - begin < 200000000ll) {}
        }
    } else {
        // ---- epilogue: warp w reads the 32 accumulator rows 32 (w % 4)..,
        // the warps of a quarter take turns over its 32-column pieces
        const int quarter = warp & 3, group = (warp - 2) >> 2;
        float* s = staging + (warp - 2) * (kWarpStaging / 4);
        int n = 0;
        if constexpr (kChunked) {
            static_assert(kBN / 32 <= kGroups, "a piece a warp");
            for (unsigned t = blockIdx.x; t < tiles; t += gridDim.x) {
                const Tile tile = tile_at<kBN>(p, t);
                const bool mine = group < kBN / 32;
                const int64_t row0 = tile.i0 + quarter * 32, col0 = tile.j0 + group * 32;
                const bool live = mine && col0 < p.nj && row0 < p.ni;
                float sum[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) sum[i] = 0.f;
                bool given_up = false;
                for (int from = tile.begin; from < tile.end; from += kChunk, ++n) {
                    const int buf = n & 1;
                    if (!warp_wait(acc_full(buf), (n >> 1) & 1, p.patience, dead)) {
                        given_up = true;
                        break;
                    }
                    fence_after();
                    if (mine) {
                        float v[16];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            tmem_load16(v, tmem + buf * kBN + ((uint32_t)(quarter * 32) << 16) + group * 32 + h * 16);
#pragma unroll
                            for (int i = 0; i < 16; i += 2) add2(sum[h * 16 + i], sum[h * 16 + i + 1], v[i], v[i + 1]);
                        }
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(acc_empty(buf));
                }
                if (given_up) break;
                if (!live) continue;
                if (kKind == kForward && p.bias) {
                    __syncwarp();
                    s[32 * 16 + lane] = col0 + lane < p.nj ? load_param(p.bias, p.bias_dtype, col0 + lane) : 0.f;
                    __syncwarp();
                }
                if constexpr (kKeeps) {
                    Ahead ahead;
                    ahead.have = false;
                    finish32<kOut, kMode>(sum, p, row0, col0, s, ahead, lane);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float v[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = sum[h * 16 + i];
                        if (col0 + h * 16 < p.nj) finish16<kKind, kOut, kMode>(v, p, tile, row0, col0 + h * 16, s, h, lane);
                    }
                }
            }
        } else
        for (unsigned t = blockIdx.x; t < tiles; t += gridDim.x, ++n) {
            const Tile tile = tile_at<kBN>(p, t);
            constexpr int kPieces = kBN / 32;
            const int buf = n & 1;
            const int64_t row0 = tile.i0 + quarter * 32;
            Ahead ahead;
            float bias = 0.f;
            auto bias_ahead = [&](int c) {
                const int64_t col = tile.j0 + c * 32 + lane;
                bias = kKind == kForward && p.bias && c < kPieces && col < p.nj ? load_param(p.bias, p.bias_dtype, col) : 0.f;
            };
            auto release = [&] {
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(acc_empty(buf));
            };
            ahead.have = false;
            bias_ahead(group);
            if (kKeeps && kMode == kAligned && group < kPieces) load_ahead<kOut>(ahead, p, row0, tile.j0 + group * 32, lane);
            if (!warp_wait(acc_full(buf), (n >> 1) & 1, p.patience, dead)) break;
            fence_after();
            const uint32_t base = tmem + buf * kBN + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
            for (int c = group; c < kPieces; c += kGroups) {
                const int64_t col0 = tile.j0 + c * 32;
                const bool live = col0 < p.nj && row0 < p.ni;
                const bool last = c + kGroups >= kPieces;
                __syncwarp();
                if (kKind == kForward && live && p.bias) {
                    s[32 * 16 + lane] = bias;
                    __syncwarp();
                }
                bias_ahead(c + kGroups);
                if constexpr (kKeeps) {
                    float v[32];
                    tmem_load32(v, base + c * 32);
                    if (last) release();   // the accumulator is free before any of the work on its values
                    if (live) finish32<kOut, kMode>(v, p, row0, col0, s, ahead, lane);
                    if (kMode == kAligned && !last) load_ahead<kOut>(ahead, p, row0, col0 + kGroups * 32, lane);
                } else {
                    float v[16];
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        __syncwarp();
                        tmem_load16(v, base + c * 32 + h * 16);
                        if (h == 1 && last) release();
                        if (live && col0 + h * 16 < p.nj)
                            finish16<kKind, kOut, kMode>(v, p, tile, row0, col0 + h * 16, s, h, lane);
                    }
                }
            }
            if (group >= kPieces && lane == 0) bar_arrive(acc_empty(buf));
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
    if (threadIdx.x == 0 && dead_flag && p.fault) *reinterpret_cast<volatile unsigned*>(p.fault) = 1;
}

// ------------------------------------------------------------------ launch

template <int kKind, int kBN, int kOut, int kMode, bool kChunked>
cudaError_t launch_mma(const Operand& a, const Operand& b, const MmaArgs& p, cudaStream_t s) {
    int unused = 0;
    cudaError_t e = pl::kernel_once(
        reinterpret_cast<const void*>(k_mma<kKind, kBN, kOut, kMode, kChunked>),
        [](int*) {
            return cudaFuncSetAttribute(k_mma<kKind, kBN, kOut, kMode, kChunked>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(kKind, kBN, kChunked));
        },
        &unused);
    if (e != cudaSuccess) return e;
    CUtensorMap ma, mb;
    if ((e = make_map(&ma, a, a_mn(kKind) ? kBK : kBM)) != cudaSuccess) return e;
    if ((e = make_map(&mb, b, b_mn(kKind) ? kBK : kBN)) != cudaSuccess) return e;
    const int64_t tiles = mma_tiles(p.ni, p.nj, kBN) * p.parts;
    if (tiles > INT_MAX) return cudaErrorInvalidValue;
    const int ctas = (int)(tiles < sm_count() ? tiles : sm_count());
    k_mma<kKind, kBN, kOut, kMode, kChunked>
        <<<ctas, role_threads(kKind, kChunked), smem_bytes(kKind, kBN, kChunked), s>>>(ma, mb, p, (unsigned)tiles);
    return cudaGetLastError();
}

// kDeep: results whose deep sums go in chunks.
template <int kKind, int kOut, int kMode, bool kDeep>
cudaError_t launch_bn(int bn, const Operand& a, const Operand& b, const MmaArgs& p, cudaStream_t s) {
    if constexpr (kDeep) {
        if (chunked(p.part_steps, p.out_dtype, p.precise)) {
            if (bn > 64) return launch_mma<kKind, 128, kOut, kMode, true>(a, b, p, s);
            if constexpr (kKind == kForward)
                if (bn == 32) return launch_mma<kKind, 32, kOut, kMode, true>(a, b, p, s);
            return launch_mma<kKind, 64, kOut, kMode, true>(a, b, p, s);
        }
    }
    if (bn == 256) return launch_mma<kKind, 256, kOut, kMode, false>(a, b, p, s);
    if (bn == 128) return launch_mma<kKind, 128, kOut, kMode, false>(a, b, p, s);
    if (bn == 64) return launch_mma<kKind, 64, kOut, kMode, false>(a, b, p, s);
    if constexpr (kKind == kForward) return launch_mma<kKind, 32, kOut, kMode, false>(a, b, p, s);
    return cudaErrorInvalidValue;
}

template <int kKind, int kMode>
cudaError_t launch_out(int bn, const Operand& a, const Operand& b, const MmaArgs& p, cudaStream_t s) {
    if (p.out_dtype == PLATTICE_F32) return launch_bn<kKind, PLATTICE_F32, kMode, true>(bn, a, b, p, s);
    if (p.out_dtype == PLATTICE_BF16) return launch_bn<kKind, PLATTICE_BF16, kMode, false>(bn, a, b, p, s);
    return launch_bn<kKind, PLATTICE_F16, kMode, false>(bn, a, b, p, s);
}

}  // namespace plr
