// Internal declarations shared by the cache and attention translation units (not part of the C ABI).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ember_attn.h"

namespace ember_attn_impl {

// n / d for 0 <= n < 2^31 by a multiplication and a shift (Granlund and Montgomery, 1994): a page may hold any
// number of tokens, and every lane divides.
struct FastDiv {
  uint32_t d, mul, shift;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {d, (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}
__host__ __device__ inline uint32_t div_by(uint32_t n, const FastDiv& f) {
  return ((uint32_t)((uint64_t)n * f.mul >> 32) + n) >> f.shift;
}

// A call's cache and batch as the kernels take them.
struct CacheArgs {
  void *k, *v;
  _Float16 *ks, *vs;       // Q8_0 scales
  int type, n_kv, D, n_pages;
  FastDiv page;            // tokens per page
  // the batch
  int n_seqs, n_tokens, max_q;
  int cap;                 // tokens that a sequence can have: max_kv, and what its pages hold
  int max_pages;           // row width of `pages`
  const int32_t* q_start;  // or null
  const int32_t* kv_len;
  const int32_t* pages;    // or null
};

// Where the device arrays point, kept inside the buffers whatever they hold (host code too, for its test on the CPU).

// Index of the cache row (page, KV head 0, row in the page) in units of [page] rows of one head: the page's first row
// is pid * n_kv * page. -1: no such page.
__host__ __device__ inline int64_t cache_row(const CacheArgs& c, int b, int pos) {
  const uint32_t pg = div_by((uint32_t)pos, c.page);
  const int pid = c.pages ? c.pages[(int64_t)b * c.max_pages + pg] : b;
  if ((uint32_t)pid >= (uint32_t)c.n_pages) return -1;
  return (int64_t)pid * c.n_kv * c.page.d + (pos - (int)(pg * c.page.d));
}
__host__ __device__ inline int length(const CacheArgs& c, int len) { return len < 0 ? 0 : len < c.cap ? len : c.cap; }
__device__ inline int seq_len(const CacheArgs& c, int b) { return length(c, c.kv_len[b]); }

constexpr int64_t kNoSeq = -1, kNoPage = -2;
// Cache row of token i, which is of sequence b, whose rows are first .. end - 1 and whose length is len;
// kNoSeq: the row belongs to no sequence; kNoPage: its place is in no page.
__host__ __device__ inline int64_t place_of(const CacheArgs& c, int b, int first, int end, int len, int i) {
  if (b >= c.n_seqs || i < first || first < 0 || i >= c.n_tokens) return kNoSeq;
  const int64_t pos = (int64_t)length(c, len) - ((int64_t)end - first) + (i - first);
  if (pos < 0 || pos >= c.cap) return kNoPage;
  const int64_t row = cache_row(c, b, (int)pos);
  return row < 0 ? kNoPage : row;
}

// Rows of sequence b: first row and count, kept inside [0, n_tokens).
__host__ __device__ inline void seq_rows(const CacheArgs& c, int b, int& first, int& count) {
  if (!c.q_start) {
    first = b;
    count = 1;
    return;
  }
  first = c.q_start[b];
  const int last = c.q_start[b + 1], end = last < c.n_tokens ? last : c.n_tokens;
  count = first < 0 || end < first ? 0 : end - first;
}

// Blocks of 256 threads that a launch can have in x: the runtime counts threads in 32 bits.
constexpr int64_t kMaxBlocks = (1 << 24) - 1;

int make_cache_args(const ember_kv_cache* c, const ember_kv_batch* b, CacheArgs* out);

int launch_kv_store(const CacheArgs& c, const void* k, int64_t ks, const void* v, int64_t vs, int type, hipStream_t st);
int launch_kv_load(const CacheArgs& c, void* k, int64_t ks, void* v, int64_t vs, int type, hipStream_t st);

struct AttnArgs {
  CacheArgs c;
  int H, G;                // heads, heads per KV head
  float scale, softcap;
  int window;              // 0: none
  const float* slopes;     // or null
  const int32_t* prefix;   // or null
  int shared;
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  int type;                // of q and out
};
// How a call runs, by its sizes alone. Every sequence's keys from `begin` on: attn_step_kernel for up to 64 rows per KV head and
// sequence, attn_wide_kernel for more, in `splits` parts of `chunk` keys; before that the shared pages (begin > 0), the batch's
// rows together, in shared_splits of shared_chunk.
struct AttnPlan {
  bool step;
  int splits, chunk;
  int begin, shared_splits, shared_chunk;
  int parts;  // parts in the scratch, 0 where the kernel writes the output itself
};
AttnPlan attn_plan(const AttnArgs& a);
size_t attn_scratch(const AttnArgs& a);
int launch_attn(const AttnArgs& a, void* scratch, hipStream_t st);

struct Parts;
// `part0`: the first of the parts that a launch writes
int launch_step_bf16(const AttnArgs& a, const Parts& p, int part0, int splits, int chunk, int begin, hipStream_t st);
int launch_step_f16(const AttnArgs& a, const Parts& p, int part0, int splits, int chunk, int begin, hipStream_t st);
int launch_step_q8_bf16(const AttnArgs& a, const Parts& p, int part0, int splits, int chunk, int begin, hipStream_t st);
int launch_step_q8_f16(const AttnArgs& a, const Parts& p, int part0, int splits, int chunk, int begin, hipStream_t st);
// A launch of attn_wide_kernel: its parts begin with part0; end > 0: the shared pages, up to there.
struct WideCall {
  int part0, splits, chunk, begin, end;
};
int launch_wide_bf16(const AttnArgs& a, const Parts& p, const WideCall& w, hipStream_t st);
int launch_wide_f16(const AttnArgs& a, const Parts& p, const WideCall& w, hipStream_t st);
int launch_wide_q8_bf16(const AttnArgs& a, const Parts& p, const WideCall& w, hipStream_t st);
int launch_wide_q8_f16(const AttnArgs& a, const Parts& p, const WideCall& w, hipStream_t st);

}  // namespace ember_attn_impl
