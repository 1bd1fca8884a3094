// rows_logp.cu -- C entry points of the log probabilities; the kernels are
// rows_logp.cuh, made for a type each by rows_logp_f32.cu and its siblings.
#include "rows_host.h"
#include "rows_logp.h"

using namespace plr;

extern "C" {

static bool logp_ok(const plattice_log_probs_args* q) {
    return q && dtype_ok(q->dtype) && q->rows >= 0 && q->n >= 1 && q->n <= (1 << 30) && q->top >= 0 &&
           q->top <= PLATTICE_MAX_TOP && q->top <= q->n && fits(q->rows, q->n) &&
           on_elements(q->labels_wide ? 8 : 4, q->labels);
}

static LogpArgs logp_args(const plattice_log_probs_args* q) {
    return {q->logits, q->labels, q->labels_wide, q->logp, q->entropy, reinterpret_cast<float2*>(q->stats), q->lse, q->top_logp,
            q->top_ids, q->grad_logp, q->grad_entropy, q->grad_lse, q->grad_logits, q->rows, q->n, q->top};
}

int plattice_log_probs(const plattice_log_probs_args* q, void* stream) {
    if (!logp_ok(q)) return PLATTICE_ERR_INVALID;
    if (q->rows == 0) return PLATTICE_OK;
    if (!q->logits || !on_elements(dtype_size(q->dtype), q->logits) || !q->stats || !on_elements(2 * sizeof(float), q->stats) ||
        !on_elements(sizeof(float), q->logp, q->entropy, q->lse) || (q->logp && !q->labels) ||
        (q->top && (!q->top_logp || !q->top_ids || !on_elements(sizeof(float), q->top_logp) || !on_elements(8, q->top_ids))))
        return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const LogpArgs a = logp_args(q);
    const cudaError_t e = q->dtype == PLATTICE_F32    ? logp_forward<float>(a, s)
                          : q->dtype == PLATTICE_BF16 ? logp_forward<__nv_bfloat16>(a, s)
                                                      : logp_forward<__half>(a, s);
    return rows_status(e, "plattice_log_probs");
}

int plattice_log_probs_backward(const plattice_log_probs_args* q, void* stream) {
    if (!logp_ok(q)) return PLATTICE_ERR_INVALID;
    if (q->rows == 0) return PLATTICE_OK;
    if (!q->logits || !q->stats || !on_elements(2 * sizeof(float), q->stats) || !q->grad_logits ||
        !on_elements(dtype_size(q->dtype), q->logits, q->grad_logits) ||
        !on_elements(sizeof(float), q->grad_logp, q->grad_entropy, q->grad_lse) || (q->grad_logp && !q->labels) ||
        (q->grad_entropy && (!q->entropy || !on_elements(sizeof(float), q->entropy))))
        return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const LogpArgs a = logp_args(q);
    const cudaError_t e = q->dtype == PLATTICE_F32    ? logp_backward<float>(a, s)
                          : q->dtype == PLATTICE_BF16 ? logp_backward<__nv_bfloat16>(a, s)
                                                      : logp_backward<__half>(a, s);
    return rows_status(e, "plattice_log_probs_backward");
}

}  // extern "C"
