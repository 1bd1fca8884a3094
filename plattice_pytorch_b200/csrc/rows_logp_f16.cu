// rows_logp_f16.cu -- log probabilities of float16 scores.
#include "rows_logp.cuh"

namespace plr {

template cudaError_t logp_forward<__half>(const LogpArgs& a, cudaStream_t s);
template cudaError_t logp_backward<__half>(const LogpArgs& a, cudaStream_t s);

}  // namespace plr
