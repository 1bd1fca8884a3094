// rows_mma_forward.cu -- the tiled product of the linear map's forward.
#include "rows_mma.cuh"

namespace plr {

cudaError_t mma_forward(int bn, bool aligned, const Operand& x, const Operand& w, const MmaArgs& p, cudaStream_t s) {
    const bool deep16 = p.out_dtype != PLATTICE_F32 && chunked(p.part_steps, p.out_dtype, p.precise);
    if (!aligned || p.split || deep16) return launch_bn<kForward, PLATTICE_F32, kAny, true>(bn, x, w, p, s);
    if (p.act == PLATTICE_ACT_NONE && !p.residual && !p.z) return launch_out<kForward, kPlain>(bn, x, w, p, s);
    return launch_out<kForward, kAligned>(bn, x, w, p, s);
}

}  // namespace plr
