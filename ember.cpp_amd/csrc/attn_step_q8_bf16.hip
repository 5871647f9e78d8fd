// attn_step.hpp for Q8_0 caches and BF16 rows.
#include "attn_step.hpp"

namespace ember_attn_impl {
int launch_step_q8_bf16(const AttnArgs& a, const Parts& p, int part0, int splits, int chunk, int begin, hipStream_t st) {
  return launch_step_type<EMBER_TYPE_Q8_0, EMBER_TYPE_BF16>(a, p, part0, splits, chunk, begin, st);
}
}  // namespace ember_attn_impl
