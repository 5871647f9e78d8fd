// attn_step.hpp for F16 caches and F16 rows.
#include "attn_step.hpp"

namespace ember_attn_impl {
int launch_step_f16(const AttnArgs& a, const Parts& p, int part0, int splits, int chunk, int begin, hipStream_t st) {
  return launch_step_type<EMBER_TYPE_F16, EMBER_TYPE_F16>(a, p, part0, splits, chunk, begin, st);
}
}  // namespace ember_attn_impl
