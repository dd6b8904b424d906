// Gradients of the masked attention of f16.
#include "masked_attention_bwd.h"

namespace vgo {
namespace masked {

template int run_grad<f16_t>(const vgo_masked_attn*, const vgo_masked_attn_grads*, const GradPlan&, char*, hipStream_t);

}  // namespace masked
}  // namespace vgo
