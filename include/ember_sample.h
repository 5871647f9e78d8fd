/* C ABI of the pick of the next token (libember_moe.so, HIP / gfx950): temperature, top-k, top-p and min-p over rows of
 * logits, drawn by random numbers that the caller gives. Contract as of ember_attn.h: one stream, no allocation, no host
 * synchronisation, an ember_status as the result and nothing launched on an error. */
#ifndef EMBER_SAMPLE_H
#define EMBER_SAMPLE_H
#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>
#include "ember_moe_host.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Per row, over the logits z: weights w_i = exp((z_i - max z) / temperature), then three filters, each on the
 * distribution of the tokens that top-k leaves:
 *   top_k  (> 0, < V) the k largest logits, of equal ones those of lower index;
 *   top_p  (< 1)      in descending order (equal ones by index) the tokens before which less than top_p of the
 *                     top-k tokens' whole weight lies: at least the first;
 *   min_p  (> 0)      the tokens with w_i >= min_p, that is min_p times the most likely one's (over 1: as 1).
 * The token drawn is the first index at which the kept tokens' weights, added by index, are more than u times their sum.
 * temperature <= 0 or top_k = 1: the largest logit's (lowest) index. NaN and -inf are never drawn; with +inf
 * among the logits only those are. A row in which no token can be drawn gives -1 and probability 0. The sums are of
 * fixed-point weights (in steps of 2^-51 of the largest, coarser only where the row's sum would pass 61 bits), so neither order nor grid
 * has an effect on the result.
 * A row's setting is the array's where that is not NULL ([n] device), the field's otherwise; NaN settings count as off
 * (temperature: as 1). */
typedef struct ember_sampler {
  float temperature;
  int top_k;              /* <= 0: off */
  float top_p;            /* >= 1: off; <= 0: the most likely token alone */
  float min_p;            /* <= 0: off */
  const float* temperatures;
  const int32_t* top_ks;
  const float* top_ps;
  const float* min_ps;
} ember_sampler;

/* ids[r], probs[r] (probs may be NULL) for the n rows (n < 1 << 23) of V logits (V <= 1 << 24), `stride` elements apart, of `type` F32,
 * F16 or BF16 (aligned as that type); u [n] device, in [0, 1) (others count as the nearest). probs: the drawn token's
 * share of the kept tokens' weight (1 for the largest logit's pick). */
int ember_sample(const ember_sampler* s, const void* logits, int type, int n, int V, int64_t stride, const float* u,
                 int32_t* ids, float* probs, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
