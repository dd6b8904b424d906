// Attention over the paged cache for many queries of one type.
#include "cached_attention_many.h"

namespace vgo {
namespace paged {

template <>
int launch_many<f16_t>(const Attend& a, int64_t pieces, int head_dim, hipStream_t s) {
  return head_dim == 64 ? run_many<f16_t, 64>(a, pieces, s) : run_many<f16_t, 128>(a, pieces, s);
}
template <>
ManyShape many_shape<f16_t>(int head_dim) {
  return head_dim == 64 ? ManyShape{32 * Many<f16_t, 64>::kTiles * Many<f16_t, 64>::kWaves, 4 * Many<f16_t, 64>::kResident / Many<f16_t, 64>::kWaves}
                        : ManyShape{32 * Many<f16_t, 128>::kTiles * Many<f16_t, 128>::kWaves, 4 * Many<f16_t, 128>::kResident / Many<f16_t, 128>::kWaves};
}

}  // namespace paged
}  // namespace vgo
