/* C ABI of the cache and the attention of a decoder layer around the MoE FFN (libember_moe.so, HIP / gfx950):
 * K and V rows stored into a paged cache, as halves or quantised, and read back; attention of a batch's new
 * tokens over the cache, for prompts and single tokens, with or without first pages that the batch shares.
 *
 * The reference keeps these in its engine (attention, KV cache, kv_quant.cu), outside the MoE operator that this
 * library replaces; there is no entry of its own to mirror, and layouts and names here are this library's.
 *
 * Contract of every entry, as of ember_moe_ffn: caller-owned device memory, one stream, no allocation and no host
 * synchronisation (so calls can be captured in a HIP graph), an ember_status as the result, and nothing launched on
 * an error. The current device has to be the one that holds the memory. Calls that overlap may share a cache that
 * none of them writes, and never a scratch buffer.
 *
 * Device arrays are not checked by the host. The kernels keep every access inside the buffers that the descriptors
 * state: a sequence's length counts as at most max_kv and what its pages hold, a token whose place is in no page
 * (a page id outside [0, n_pages), a negative position) is not stored and reads as zeros in ember_kv_load, and
 * attention rows that see such a key are NaN.
 */
#ifndef EMBER_ATTN_H
#define EMBER_ATTN_H
#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>
#include "ember_moe_host.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The cache of one layer: n_pages pages of `page` tokens each, for every KV head.
 *   F16, BF16  k, v [n_pages][n_kv][page][head_dim] halves; k_scale, v_scale NULL
 *   Q8_0       k, v [n_pages][n_kv][page][head_dim] int8 codes, and per 32 of them one fp16 scale in k_scale, v_scale
 *              [n_pages][n_kv][page][head_dim / 32]: the numbers of ggml's Q8_0 blocks in two planes, so that rows
 *              stay 16-byte aligned
 * head_dim: a multiple of 32 from 32 to 256. n_kv <= 256, n_pages * n_kv * page < 2^32 - 1. All pointers 16-byte aligned. */
typedef struct ember_kv_cache {
  int type;
  int n_kv, head_dim, page, n_pages;
  void* k;
  void* v;
  void* k_scale;
  void* v_scale;
} ember_kv_cache;

/* What a call works on: the new tokens of n_seqs sequences, as rows of q, k, v and out. Sequence b has the rows
 * q_start[b] .. q_start[b + 1] - 1 (q_start NULL: the row b alone), and kv_len[b] tokens in the cache, the new ones
 * its last: row i is at position p = kv_len[b] - (q_start[b + 1] - q_start[b]) + (i - q_start[b]), and position p
 * lies in row p % page of page pages[b * max_pages + p / page] (pages NULL: of page b, which then holds all of
 * sequence b). Rows behind the last sequence's (n_tokens may be larger than q_start[n_seqs]) are left as they are.
 * No two rows of a call may have the same place in the cache where the call stores them. */
typedef struct ember_kv_batch {
  int n_seqs;               /* up to 65535 */
  int n_tokens;             /* rows of q, k, v and out. A call too large for a launch (2^24 blocks: of 128 rows of a KV head in the
                             * attention, of 8192 values in store and load) is refused with EMBER_ERR_SHAPE */
  int max_q;                /* no sequence has more new tokens (those past max_q get no attention output) */
  int max_kv;               /* no sequence has more tokens in the cache; up to 1 << 29 */
  const int32_t* q_start;   /* [n_seqs + 1] device, ascending, or NULL: one token each, n_tokens >= n_seqs */
  const int32_t* kv_len;    /* [n_seqs] device */
  const int32_t* pages;     /* [n_seqs][max_pages] device, or NULL */
  int max_pages;
  /* Attention: the first `shared` tokens of every sequence lie in the same pages, those of sequence 0 (as when
   * many answers continue one prompt): a multiple of page, 0 if there are none. Where that saves enough,
   * their keys and values are read once for the whole batch; results are those of the same call with shared = 0, but for
   * the order of its sums. Sequences shorter than `shared` attend to what they have of it. Needs pages. */
  int shared;
} ember_kv_batch;

/* Stores the batch's rows k, v [n_tokens][n_kv][head_dim] (rows k_stride, v_stride elements apart, `type` F32, F16 or
 * BF16) at their places. Halves are rounded to nearest even. Q8_0, per 32 values: d = fp16(min(max|x| / 127, 515.5)),
 * code = the integer nearest to x / d (ties to even, at most 127 in magnitude), so magnitudes over 127 * 515.5 saturate;
 * a NaN makes its 32 values NaN. Base pointers and row strides: multiples of 16 bytes; strides >= n_kv * head_dim. */
int ember_kv_store(const ember_kv_cache* c, const ember_kv_batch* b, const void* k, int64_t k_stride, const void* v,
                   int64_t v_stride, int type, hipStream_t stream);

/* The reverse: the values at the batch's places into the rows k, v, rounded once to `type` (F32: exact). */
int ember_kv_load(const ember_kv_cache* c, const ember_kv_batch* b, void* k, int64_t k_stride, void* v, int64_t v_stride,
                  int type, hipStream_t stream);

/* Options of the attention. Head h of the n_heads reads KV head h / (n_heads / n_kv). For the row at position p, key j
 * (< kv_len[b]) is visible if j <= p or j < prefix[b], and, where window > 0, p - j < window. Its score is
 *   s = scale * (q . k_j);  softcap > 0: s = softcap * tanh(s / softcap);  slopes: s -= slopes[h] * |p - j|
 * and the output row the softmax-weighted sum of the visible keys' values, zeros if no key is visible. Keys and
 * values that a row does not see have no effect on it, whatever they hold; a row that sees one that is infinite or NaN is
 * not finite in the columns that hold it, or in all. Scores are f32 and have to stay within +-1e29. */
typedef struct ember_attn_opts {
  int n_heads;           /* a multiple of n_kv, up to 128 per KV head */
  float scale;           /* > 0 */
  float softcap;         /* 0: none; else over scale * 1e-30 */
  int window;            /* 0: none */
  const float* slopes;   /* [n_heads] device, or NULL */
  const int32_t* prefix; /* [n_seqs] device, or NULL */
} ember_attn_opts;

/* Scratch bytes ember_attn needs for these sizes (device arrays are not read), 0 for invalid arguments and for calls
 * that need none. A batch with smaller max_q, max_kv, n_seqs or n_tokens may need more: size for each. */
size_t ember_attn_scratch_bytes(const ember_attn_opts* a, const ember_kv_cache* c, const ember_kv_batch* b);

/* out = attention of the rows q [n_tokens][n_heads][head_dim] over the cache (which already holds the new tokens: call
 * ember_kv_store first). q and out are of `type`: that of an F16 or BF16 cache, either of them for Q8_0. Rows q_stride,
 * out_stride elements apart; base pointers and row strides multiples of 16 bytes, strides >= n_heads * head_dim.
 * scratch: ember_attn_scratch_bytes, 256-byte aligned (NULL where that is 0). out may be q itself. */
int ember_attn(const ember_attn_opts* a, const ember_kv_cache* c, const ember_kv_batch* b, const void* q, int64_t q_stride,
               void* out, int64_t out_stride, int type, void* scratch, size_t scratch_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
