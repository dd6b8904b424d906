// Attention over the paged cache for many queries of one type.
#include "cached_attention_many.h"

namespace vgo {
namespace paged {

template <>
int launch_many<bf16_t>(const Attend& a, int64_t pieces, int head_dim, hipStream_t s) {
  return head_dim == 64 ? run_many<bf16_t, 64>(a, pieces, s) : run_many<bf16_t, 128>(a, pieces, s);
}
template <>
ManyShape many_shape<bf16_t>(int head_dim) {
  return head_dim == 64 ? ManyShape{32 * Many<bf16_t, 64>::kTiles * Many<bf16_t, 64>::kWaves, 4 * Many<bf16_t, 64>::kResident / Many<bf16_t, 64>::kWaves}
                        : ManyShape{32 * Many<bf16_t, 128>::kTiles * Many<bf16_t, 128>::kWaves, 4 * Many<bf16_t, 128>::kResident / Many<bf16_t, 128>::kWaves};
}

}  // namespace paged
}  // namespace vgo
