// rows_mma_grad.cu -- the tiled products of the linear map's gradients.
#include "rows_mma.cuh"

namespace plr {

cudaError_t mma_grad_x(int bn, bool aligned, const Operand& gz, const Operand& w, const MmaArgs& p, cudaStream_t s) {
    const bool deep16 = p.out_dtype != PLATTICE_F32 && chunked(p.part_steps, p.out_dtype, p.precise);
    if (!aligned || deep16) return launch_bn<kGradX, PLATTICE_F32, kAny, true>(bn, gz, w, p, s);
    return launch_out<kGradX, kPlain>(bn, gz, w, p, s);
}

cudaError_t mma_grad_w(int bn, const Operand& x, const Operand& gz, const MmaArgs& p, cudaStream_t s) {
    return launch_out<kGradW, kAny>(bn, x, gz, p, s);
}

}  // namespace plr
