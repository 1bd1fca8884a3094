// rows_logp_bf16.cu -- log probabilities of bfloat16 scores.
#include "rows_logp.cuh"

namespace plr {

template cudaError_t logp_forward<__nv_bfloat16>(const LogpArgs& a, cudaStream_t s);
template cudaError_t logp_backward<__nv_bfloat16>(const LogpArgs& a, cudaStream_t s);

}  // namespace plr
