// rows_narrow.cu -- launches of the linear map with at most 32 output channels
// and with few rows.
#include "rows_narrow.cuh"

namespace plr {

template <int kXT, int kNF, bool kW3, bool kSplit, bool kPlain>
static cudaError_t launch_narrow(const SmallArgs& a, int64_t blocks, cudaStream_t s) {
    const int64_t smem = narrow_fragments(a.k, kNF, kW3 ? 3 : 1) + narrow_staging(NarrowShape<kXT>::kM);
    int unused = 0;
    const cudaError_t e = pl::kernel_once(
        reinterpret_cast<const void*>(k_narrow<kXT, kNF, kW3, kSplit, kPlain>),
        [](int*) {
            return cudaFuncSetAttribute(k_narrow<kXT, kNF, kW3, kSplit, kPlain>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)(kNarrowMost + narrow_staging(2)));
        },
        &unused);
    if (e != cudaSuccess) return e;
    // one round of CTAs: as many as are resident at a time
    const int64_t need = kSplit ? blocks : ceil_div(blocks, kNarrowWarps);
    const int64_t fit = kMaxSmem / (smem + 1024), ctas = narrow_ctas(kXT, kNF);
    const int64_t most = (fit < ctas ? fit : ctas) * sm_count();
    k_narrow<kXT, kNF, kW3, kSplit, kPlain><<<(unsigned)(need < most ? need : most), 32 * kNarrowWarps, smem, s>>>(a);
    return cudaGetLastError();
}

template <int kXT, bool kW3, int kNF>
static cudaError_t run_narrow_as(const SmallArgs& a, cudaStream_t s) {
    const int64_t blocks = ceil_div(a.rows, 16 * NarrowShape<kXT>::kM);
    if constexpr (kW3)
        if (narrow_shares(blocks, a.k)) return launch_narrow<kXT, kNF, kW3, true, false>(a, blocks, s);
    if (a.out_dtype == PLATTICE_F32 && a.act == PLATTICE_ACT_NONE && !a.residual && !a.z)
        return launch_narrow<kXT, kNF, kW3, false, true>(a, blocks, s);
    return launch_narrow<kXT, kNF, kW3, false, false>(a, blocks, s);
}

template <int kXT, bool kW3>
static cudaError_t run_narrow_nf(const SmallArgs& a, cudaStream_t s) {
    switch ((a.n + 7) / 8) {
        case 1: return run_narrow_as<kXT, kW3, 1>(a, s);
        case 2: return run_narrow_as<kXT, kW3, 2>(a, s);
        case 3: return run_narrow_as<kXT, kW3, 3>(a, s);
        default: return run_narrow_as<kXT, kW3, 4>(a, s);
    }
}

cudaError_t run_narrow(const SmallArgs& a, int dtype, cudaStream_t s) {
    if (a.x_scale) return dtype == PLATTICE_F32 ? run_narrow_nf<kX8, true>(a, s) : run_narrow_nf<kX8, false>(a, s);
    return dtype == PLATTICE_F32    ? run_narrow_nf<kXFloat, true>(a, s)
           : dtype == PLATTICE_BF16 ? run_narrow_nf<kXBf16, false>(a, s)
                                    : run_narrow_nf<kXHalf, false>(a, s);
}

template <int kWT, bool kX8In>
static cudaError_t run_few(const SmallArgs& a, cudaStream_t s) {
    const dim3 ctas((unsigned)ceil_div(a.n, 32), (unsigned)ceil_div(a.rows, 16));
    if (a.rows <= 8) k_few<kWT, kX8In, 1><<<ctas, 64 * few_splits(kWT), 0, s>>>(a);
    else k_few<kWT, kX8In, 2><<<ctas, 64 * few_splits(kWT), 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t run_few_rows(const SmallArgs& a, int dtype, cudaStream_t s) {
    if (a.x_scale) return dtype == PLATTICE_F32 ? run_few<kXFloat, true>(a, s) : run_few<kXBf16, true>(a, s);
    return dtype == PLATTICE_F32    ? run_few<kXFloat, false>(a, s)
           : dtype == PLATTICE_BF16 ? run_few<kXBf16, false>(a, s)
                                    : run_few<kXHalf, false>(a, s);
}

}  // namespace plr
