// Attention over the paged cache for many queries of one type.
#include "cached_attention_many.h"

namespace vgo {
namespace paged {

template <>
int launch_many<f16_t>(const Attend& a, int64_t pieces, int head_dim, hipStream_t s) {
  return head_dim == 64 ? run_many<f16_t, 64>(a, pieces, s) : run_many<f16_t, 128>(a, pieces, s);
}
template <>
ManyShape many_shape<f16_t>(int head_dim, bool causal, int64_t group) {
  return head_dim == 64 ? shape_of<f16_t, 64>(causal, group) : shape_of<f16_t, 128>(causal, group);
}

}  // namespace paged
}  // namespace vgo
