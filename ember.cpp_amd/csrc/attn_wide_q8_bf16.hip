// attn_wide.hpp for Q8_0 caches and BF16 rows.
#include "attn_wide.hpp"

namespace ember_attn_impl {
int launch_wide_q8_bf16(const AttnArgs& a, const Parts& p, const WideCall& w, hipStream_t st) {
  return launch_wide_type<EMBER_TYPE_Q8_0, EMBER_TYPE_BF16>(a, p, w, st);
}
}  // namespace ember_attn_impl
