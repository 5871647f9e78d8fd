// Attention over the paged cache (ember_attn): which kernels a call takes, and the join of its parts.
#include <algorithm>

#include "attn_dev.hpp"

namespace ember_attn_impl {
namespace {

// Rows of parts (Parts) as output rows: a wave per row. Its lanes first hold one part's maximum and sum each, then the row's columns.
template <int IO>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, Parts parts) {
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63, at = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int tok = at / a.H, h = at - tok * a.H;
  int first, count;
  seq_rows(c, blockIdx.y, first, count);
  if (tok >= min(count, c.max_q)) return;
  const int64_t row = (int64_t)(first + tok) * a.H + h;
  float M = kNoScore;
  for (int p = lane; p < parts.n; p += 64) M = fmaxf(M, parts.ml[(p * parts.rows + row) * 2]);
  for (int k = 32; k; k >>= 1) M = fmaxf(M, __shfl_xor(M, k));
  float sum = 0.0f;
  f4 x = {0, 0, 0, 0};
  const int d = lane * 4;
  for (int p0 = 0; p0 < parts.n; p0 += 64) {
    float w = 0.0f, l = 0.0f;
    if (p0 + lane < parts.n) {
      const float* ml = parts.ml + ((p0 + lane) * parts.rows + row) * 2;
      l = ml[1];
      w = exp2_fast(ml[0] - M);
    }
    sum += l * w;
    for (uint64_t todo = __ballot(l != 0.0f); todo; todo &= todo - 1) {  // (parts without a visible key hold nothing)
      const int p = __ffsll((unsigned long long)todo) - 1;
      const float wp = __shfl(w, p);
      if (d < c.D) {
        f4 y = *reinterpret_cast<const f4*>(parts.o + ((p0 + p) * parts.rows + row) * c.D + d);
        y *= wp;
        x += y;
      }
    }
  }
  for (int k = 32; k; k >>= 1) sum += __shfl_xor(sum, k);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  x *= inv;
  const u2 y = {pack2<IO == EMBER_TYPE_BF16>(x[0], x[1]), pack2<IO == EMBER_TYPE_BF16>(x[2], x[3])};
  if (d < c.D) *reinterpret_cast<u2*>(static_cast<uint16_t*>(a.out) + (int64_t)(first + tok) * a.out_stride + (int64_t)h * c.D + d) = y;
}

}  // namespace

AttnPlan attn_plan(const AttnArgs& a) {
  AttnPlan p{};
  const CacheArgs& c = a.c;
  const int64_t rows = (int64_t)c.max_q * a.G;
  p.step = rows <= 64;
  p.begin = std::min(a.shared, c.cap);
  auto split = [](int64_t keys, int64_t blocks, int64_t want, int unit, int& splits, int& chunk) {
    const int64_t n = std::max<int64_t>(1, std::min<int64_t>({keys / unit, 256, (want + blocks - 1) / blocks}));
    chunk = (int)((keys + n * unit - 1) / (n * unit)) * unit;
    splits = (int)((keys + chunk - 1) / chunk);
  };
  // keys that the rows of a sequence can see at most, and one tile for where they begin within one
  int64_t range = c.cap - p.begin;
  if (a.window > 0 && !a.prefix) range = std::min<int64_t>(range, (int64_t)a.window + c.max_q - 1);
  range = std::max<int64_t>(range, 1) + 63;
  const int64_t groups = (int64_t)c.n_seqs * c.n_kv;
  if (p.step) split(range, groups * ((rows + 15) / 16), 2048, 128, p.splits, p.chunk);
  else split(range, groups * ((rows + 127) / 128), 512, 256, p.splits, p.chunk);
  if (p.begin) split(p.begin, c.n_kv * (((int64_t)c.n_tokens * a.G + 127) / 128), 512, 256, p.shared_splits, p.shared_chunk);
  p.parts = p.splits + p.shared_splits > 1 ? p.splits + p.shared_splits : 0;
  return p;
}

size_t attn_scratch(const AttnArgs& a) {
  const AttnPlan p = attn_plan(a);
  return (size_t)p.parts * a.c.n_tokens * a.H * (a.c.D + 2) * 4;
}

int launch_attn(const AttnArgs& a, void* scratch, hipStream_t st) {
  const AttnPlan p = attn_plan(a);
  Parts parts{nullptr, nullptr, (int64_t)a.c.n_tokens * a.H, std::max(p.parts, 1)};
  if (p.parts) {
    parts.o = static_cast<float*>(scratch);
    parts.ml = parts.o + p.parts * parts.rows * a.c.D;
  }
  const int kind = a.c.type == EMBER_TYPE_BF16 ? 0 : a.c.type == EMBER_TYPE_F16 ? 1 : a.type == EMBER_TYPE_BF16 ? 2 : 3;
  decltype(&launch_step_bf16) const steps[4] = {launch_step_bf16, launch_step_f16, launch_step_q8_bf16, launch_step_q8_f16};
  decltype(&launch_wide_bf16) const wides[4] = {launch_wide_bf16, launch_wide_f16, launch_wide_q8_bf16, launch_wide_q8_f16};
  int s = EMBER_OK;
  if (p.begin) s = wides[kind](a, parts, WideCall{0, p.shared_splits, p.shared_chunk, 0, p.begin}, st);
  if (s) return s;
  if (p.step) s = steps[kind](a, parts, p.shared_splits, p.splits, p.chunk, p.begin, st);
  else s = wides[kind](a, parts, WideCall{p.shared_splits, p.splits, p.chunk, p.begin, 0}, st);
  if (s || !p.parts) return s;
  const dim3 grid((unsigned)(((int64_t)a.c.max_q * a.H + 3) / 4), a.c.n_seqs);
  if (a.type == EMBER_TYPE_BF16) attn_join_kernel<EMBER_TYPE_BF16><<<grid, 256, 0, st>>>(a, parts);
  else attn_join_kernel<EMBER_TYPE_F16><<<grid, 256, 0, st>>>(a, parts);
  return hipGetLastError() == hipSuccess ? EMBER_OK : EMBER_ERR_LAUNCH;
}

}  // namespace ember_attn_impl
