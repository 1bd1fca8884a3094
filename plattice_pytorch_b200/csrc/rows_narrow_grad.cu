// rows_narrow_grad.cu -- launches of the linear map's backward with at most 32
// output channels.
#include "rows_narrow.cuh"

namespace plr {

template <int kXT, int kParts, int kNF, bool kG32>
static cudaError_t launch_narrow_grad(const SmallGradArgs& a, int lines, cudaStream_t s) {
    int unused = 0;
    const cudaError_t e = pl::kernel_once(
        reinterpret_cast<const void*>(k_narrow_grad<kXT, kParts, kNF, kG32>),
        [](int*) {
            return cudaFuncSetAttribute(k_narrow_grad<kXT, kParts, kNF, kG32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        NarrowGradShape<kXT, kParts>::kBytes);
        },
        &unused);
    if (e != cudaSuccess) return e;
    k_narrow_grad<kXT, kParts, kNF, kG32><<<dim3(lines, (unsigned)ceil_div(a.s.k, 64)), 32 * kGradWarps,
                                            NarrowGradShape<kXT, kParts>::kBytes, s>>>(a);
    return cudaGetLastError();
}

template <int kXT, int kParts, bool kG32>
static cudaError_t run_narrow_grad_as(const SmallGradArgs& a, int lines, cudaStream_t s) {
    switch ((a.s.n + 7) / 8) {
        case 1: return launch_narrow_grad<kXT, kParts, 1, kG32>(a, lines, s);
        case 2: return launch_narrow_grad<kXT, kParts, 2, kG32>(a, lines, s);
        case 3: return launch_narrow_grad<kXT, kParts, 3, kG32>(a, lines, s);
        default: return launch_narrow_grad<kXT, kParts, 4, kG32>(a, lines, s);
    }
}

template <int kXT, int kParts>
static cudaError_t run_narrow_grad_nf(const SmallGradArgs& a, int lines, cudaStream_t s) {
    if constexpr (kParts == 1)
        if (a.s.out_dtype != PLATTICE_F32) return run_narrow_grad_as<kXT, kParts, false>(a, lines, s);
    return run_narrow_grad_as<kXT, kParts, true>(a, lines, s);
}

cudaError_t run_narrow_grad(const SmallGradArgs& a, int dtype, int parts, int lines, cudaStream_t s) {
    if (dtype == PLATTICE_F16)
        return parts == 2 ? run_narrow_grad_as<kXHalf, 2, true>(a, lines, s) : run_narrow_grad_as<kXHalf, 1, false>(a, lines, s);
    if (a.s.x_scale || !a.s.x)   // without x (no weight gradient) its type does not matter
        return dtype == PLATTICE_F32 ? run_narrow_grad_nf<kX8, 3>(a, lines, s) : run_narrow_grad_nf<kX8, 1>(a, lines, s);
    return dtype == PLATTICE_F32 ? run_narrow_grad_nf<kXFloat, 3>(a, lines, s) : run_narrow_grad_nf<kXBf16, 1>(a, lines, s);
}

}  // namespace plr
