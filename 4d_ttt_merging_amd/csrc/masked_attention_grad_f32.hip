// Gradients of the masked attention of fp32.
#include "masked_attention_bwd.h"

namespace vgo {
namespace masked {

template int run_grad<float>(const vgo_masked_attn*, const vgo_masked_attn_grads*, const GradPlan&, char*, hipStream_t);

}  // namespace masked
}  // namespace vgo
