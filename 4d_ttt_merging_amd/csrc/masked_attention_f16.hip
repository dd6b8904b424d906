// Masked attention, forward, of f16.
#include "masked_attention_fwd.h"

namespace vgo {
namespace masked {

template int run_forward<f16_t>(const vgo_masked_attn*, const ForwardPlan&, void*, const int64_t[3], float*, void*,
                                 char*, hipStream_t);

}  // namespace masked
}  // namespace vgo
