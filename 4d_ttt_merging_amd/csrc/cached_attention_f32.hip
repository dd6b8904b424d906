// Attention over the paged cache for many queries of one type.
#include "cached_attention_many.h"

namespace vgo {
namespace paged {

template <>
int launch_many<float>(const Attend& a, int64_t pieces, int head_dim, hipStream_t s) {
  return head_dim == 64 ? run_many<float, 64>(a, pieces, s) : run_many<float, 128>(a, pieces, s);
}
template <>
ManyShape many_shape<float>(int head_dim) {
  return head_dim == 64 ? ManyShape{32 * Many<float, 64>::kTiles * Many<float, 64>::kWaves, 4 * Many<float, 64>::kResident / Many<float, 64>::kWaves}
                        : ManyShape{32 * Many<float, 128>::kTiles * Many<float, 128>::kWaves, 4 * Many<float, 128>::kResident / Many<float, 128>::kWaves};
}

}  // namespace paged
}  // namespace vgo
