// rows_logp_f32.cu -- log probabilities of float32 scores.
#include "rows_logp.cuh"

namespace plr {

template cudaError_t logp_forward<float>(const LogpArgs& a, cudaStream_t s);
template cudaError_t logp_backward<float>(const LogpArgs& a, cudaStream_t s);

}  // namespace plr
