// attn_wide.hpp for BF16 caches and BF16 rows.
#include "attn_wide.hpp"

namespace ember_attn_impl {
int launch_wide_bf16(const AttnArgs& a, const Parts& p, const WideCall& w, hipStream_t st) {
  return launch_wide_type<EMBER_TYPE_BF16, EMBER_TYPE_BF16>(a, p, w, st);
}
}  // namespace ember_attn_impl
