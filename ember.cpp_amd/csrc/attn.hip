// Attention over the paged cache (ember_attn): which kernels a call takes, and the join of its parts.
#include <algorithm>

#include "attn_dev.hpp"

namespace ember_attn_impl {
namespace {

// Rows of parts (Parts) as output rows: W waves of a block per row, each on a share of the parts, four rows or one per block. A wave's
// lanes first hold one part's maximum and sum each, then the row's columns. W = 4 where parts are many (a wave alone took 126 us for 32
// rows of 256 parts: one load after another), 1 where they are few, and rows may be many.
constexpr int kFewParts = 16;
template <int IO, int W>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, Parts parts) {
  __shared__ f4 xs[W][64];
  __shared__ float ms[W], sums[W];
  constexpr int U = W > 1 ? 2 : 1;  // (at most 512 parts)
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = W > 1 ? blockIdx.x : blockIdx.x * 4 + wave, tok = at / a.H, h = at - tok * a.H;
  int first, count;
  seq_rows(c, blockIdx.y, first, count);
  if (tok >= min(count, c.max_q)) return;
  const int64_t row = (int64_t)(first + tok) * a.H + h;
  const int per = (parts.n + W - 1) / W, from = W > 1 ? wave * per : 0, n = min(per, parts.n - from);
  const int d = min(lane * 4, c.D - 4);
  float m[U], l[U], M = kNoScore;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    m[u] = kNoScore;
    l[u] = 0.0f;
    if (u * 64 + lane < n) {
      const float* ml = parts.ml + ((from + u * 64 + lane) * parts.rows + row) * 2;
      m[u] = ml[0];
      l[u] = ml[1];
    }
    M = fmaxf(M, m[u]);
  }
  for (int k = W > 1 ? 32 : kFewParts / 2; k; k >>= 1) M = fmaxf(M, __shfl_xor(M, k));
  if (W == 1) M = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, M)));
  float sum = 0.0f;
  f4 x = {0, 0, 0, 0};
  const float* const o = parts.o + (from * parts.rows + row) * c.D + d;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float w = exp2_fast(m[u] - M);
    sum += l[u] * w;
    const float live = l[u] != 0.0f ? w : -1.0f;  // (parts without a visible key hold nothing; NaN is not 0)
    const int end = min(64, n - u * 64);
    for (int p0 = 0; p0 < end; p0 += 8) {
      f4 y[8];
      float wp[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        wp[i] = __shfl(live, (p0 + i) & 63);
        y[i] = f4{0, 0, 0, 0};
        if (p0 + i < end && wp[i] != -1.0f) y[i] = *reinterpret_cast<const f4*>(o + (u * 64 + p0 + i) * parts.rows * c.D);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (p0 + i < end && wp[i] != -1.0f) {
          y[i] *= wp[i];
          x += y[i];
        }
    }
  }
  for (int k = 32; k; k >>= 1) sum += __shfl_xor(sum, k);
  if constexpr (W > 1) {
    xs[wave][lane] = x;
    if (lane == 0) {
      ms[wave] = M;
      sums[wave] = sum;
    }
    __syncthreads();
    if (wave) return;
    M = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
    sum = 0.0f;
    x = f4{0, 0, 0, 0};
    for (int w = 0; w < W; ++w) {
      const float al = exp2_fast(ms[w] - M);
      sum += sums[w] * al;
      f4 y = xs[w][lane];
      y *= al;
      x += y;
    }
  }
  if (lane * 4 >= c.D) return;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  x *= inv;
  const u2 y = {pack2<IO == EMBER_TYPE_BF16>(x[0], x[1]), pack2<IO == EMBER_TYPE_BF16>(x[2], x[3])};
  *reinterpret_cast<u2*>(static_cast<uint16_t*>(a.out) + (int64_t)(first + tok) * a.out_stride + (int64_t)h * c.D + d) = y;
}

int64_t join_blocks(const AttnArgs& a, int parts) {
  const int64_t rows = (int64_t)a.c.max_q * a.H;
  return parts <= kFewParts ? (rows + 3) / 4 : rows;
}
template <int IO>
int launch_join(const AttnArgs& a, const Parts& parts, hipStream_t st) {
  const dim3 grid((unsigned)join_blocks(a, parts.n), a.c.n_seqs);
  if (parts.n <= kFewParts) attn_join_kernel<IO, 1><<<grid, 256, 0, st>>>(a, parts);
  else attn_join_kernel<IO, 4><<<grid, 256, 0, st>>>(a, parts);
  return hipGetLastError() == hipSuccess ? EMBER_OK : EMBER_ERR_LAUNCH;
}

}  // namespace

AttnPlan attn_plan(const AttnArgs& a) {
  AttnPlan p{};
  const CacheArgs& c = a.c;
  const bool q8 = c.type == EMBER_TYPE_Q8_0;
  const int64_t rows = (int64_t)c.max_q * a.G, row_bytes = q8 ? c.D + c.D / 16 : 2 * c.D;
  p.step = rows <= 64;
  // Shared pages cost a launch and a part more per row, and what they save are reads of the same memory again, which the caches serve
  // in part: from some 128 MB on (Q8_0, 8 KV heads of 128, shared / not: 32 sequences x 1024 tokens, 71 MB, 30 / 22 us; 4 x 16384, 107 MB,
  // 35 / 34; 32 x 4096, 276 MB, 33 / 50; 96 x 8192, 1.7 GB, 83 / 221).
  p.begin = std::min(a.shared, c.cap);
  if ((int64_t)(c.n_seqs - 1) * p.begin * c.n_kv * 2 * row_bytes < (int64_t)1 << 27) p.begin = 0;
  // `keys` in parts of whole `unit`s, so many that there are about `want` blocks
  auto split = [](int64_t keys, int64_t blocks, int64_t want, int unit, int& splits, int& chunk) {
    const int64_t n = std::max<int64_t>(1, std::min<int64_t>({keys / unit, 256, (want + blocks - 1) / blocks}));
    chunk = (int)((keys + n * unit - 1) / (n * unit)) * unit;
    splits = (int)((keys + chunk - 1) / chunk);
  };
  // keys that the rows of a sequence can see at most, and a tile's where they may begin within one
  int64_t range = c.cap - p.begin;
  if (a.window > 0 && !a.prefix) range = std::min<int64_t>(range, (int64_t)a.window + c.max_q - 1);
  range = std::max<int64_t>(range, 1) + (a.window > 0 || p.begin % 64 ? 63 : 0);
  const int64_t groups = (int64_t)c.n_seqs * c.n_kv;
  // Step kernel: one block for each place that 256 CUs have (more parts cost more than they level out: 131000 bf16 tokens on 512 / 1024 /
  // 2048 blocks 102 / 108 / 116 us, 8 sequences of up to 20000 Q8_0 tokens on 512 / 768 / 1024 78 / 66 / 77); up to 256 keys in one part,
  // which saves the join (256 keys 9.3 us in one part, 10.7 in two; 512 11.6, 11.0).
  const int places = 256 * (c.D > 128 ? (q8 ? 2 : 1) : q8 ? 3 : 2);
  // Many rows: two blocks per CU, and parts of 512 keys and more while the join's traffic stays under 32 MB (1024 new tokens of 32 heads in one part / two
  // 33 / 45 us, 512 20 / 25; 64 after 8000 in 31 parts / 15 / 7 29 / 37 / 60).
  const int64_t joined = (int64_t)c.n_tokens * a.H * c.D * 8, most = std::max<int64_t>(1, ((int64_t)32 << 20) / std::max<int64_t>(joined, 1));
  const int64_t wide_blocks = groups * ((rows + 127) / 128);
  if (p.step) split(range, groups * ((rows + 15) / 16), range <= 256 ? 1 : places, 128, p.splits, p.chunk);
  else split(range, wide_blocks, std::min<int64_t>(512, most * wide_blocks), 512, p.splits, p.chunk);
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
  auto tiles = [&](int64_t tokens) { return (tokens * a.G + 127) / 128 * a.c.n_kv; };  // of attn_wide_kernel
  if ((p.begin && tiles(a.c.n_tokens) * p.shared_splits > kMaxBlocks) || (!p.step && tiles(a.c.max_q) * p.splits > kMaxBlocks) ||
      (p.parts && join_blocks(a, p.parts) > kMaxBlocks))
    return EMBER_ERR_SHAPE;
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
  return a.type == EMBER_TYPE_BF16 ? launch_join<EMBER_TYPE_BF16>(a, parts, st) : launch_join<EMBER_TYPE_F16>(a, parts, st);
}

}  // namespace ember_attn_impl
