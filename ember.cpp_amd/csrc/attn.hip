// Attention over the paged cache (ember_attn): which kernels a call takes, and the join of its parts.
#include <algorithm>

#include "attn_dev.hpp"

namespace ember_attn_impl {
namespace {

__device__ inline float load_half(const void* p, int64_t at, int type) {
  return type == EMBER_TYPE_F16 ? (float)static_cast<const _Float16*>(p)[at] : ember_moe::bf16_f32(static_cast<const uint16_t*>(p)[at]);
}
__device__ inline float cached(const CacheArgs& c, const void* p, const _Float16* scales, int64_t row, int d) {
  if (c.type == EMBER_TYPE_Q8_0) return (float)static_cast<const int8_t*>(p)[row * c.D + d] * (float)scales[row * (c.D / 32) + d / 32];
  return load_half(p, row * c.D + d, c.type);
}

// One wave per (new token, head): lanes over the keys of a 64-key tile for the scores, over the head's columns for the
// weighted sum; the running maximum and sum of the softmax in f32.
__global__ __launch_bounds__(64) void attn_row_kernel(AttnArgs a) {
  const CacheArgs& c = a.c;
  const int b = blockIdx.z, h = blockIdx.y, i = blockIdx.x, lane = threadIdx.x, D = c.D;
  __shared__ float qs[256], ps[64];
  __shared__ int64_t rows[64];
  int first, count;
  seq_rows(c, b, first, count);
  if (i >= count) return;
  const int len = seq_len(c, b), total = c.q_start ? c.q_start[b + 1] - first : 1;
  const int64_t p = (int64_t)len - total + i;
  const int kvh = h / a.G;
  const int64_t q_at = (int64_t)(first + i) * a.q_stride + (int64_t)h * D;
  for (int d = lane; d < D; d += 64) qs[d] = load_half(a.q, q_at + d, a.type);
  const int prefix = a.prefix ? a.prefix[b] : 0;
  const float slope = a.slopes ? a.slopes[h] : 0.0f;
  const int64_t lo = a.window > 0 ? max((int64_t)0, p - a.window + 1) : 0;
  const int64_t hi = p < 0 ? 0 : min((int64_t)len, max(p + 1, (int64_t)prefix));
  float m = -INFINITY, l = 0.0f, o[4] = {0, 0, 0, 0};
  __syncthreads();
  for (int64_t j0 = lo; j0 < hi; j0 += 64) {
    const int64_t j = j0 + lane;
    const bool seen = j < hi;
    const int64_t row = seen ? cache_row(c, b, (int)j) : -1;
    float s = -INFINITY;
    if (seen) {
      s = __builtin_nanf("");
      if (row >= 0) {
        s = 0.0f;
        for (int d = 0; d < D; ++d) s += qs[d] * cached(c, c.k, c.ks, row + (int64_t)kvh * c.page.d, d);
        s *= a.scale;
        if (a.softcap > 0.0f) s = a.softcap * tanhf(s / a.softcap);
        if (a.slopes) s -= slope * fabsf((float)(p - j));
      }
    }
    float t = s;
    for (int k = 32; k; k >>= 1) t = fmaxf(t, __shfl_xor(t, k));
    const float m2 = fmaxf(m, t), base = m2 == -INFINITY ? 0.0f : m2;
    const float w = expf(s - base), alpha = expf(m - base);
    float sum = w;
    for (int k = 32; k; k >>= 1) sum += __shfl_xor(sum, k);
    l = l * alpha + sum;
    m = m2;
    ps[lane] = w;
    rows[lane] = row;
    __syncthreads();
    const int n = (int)min((int64_t)64, hi - j0);
    for (int u = 0; u * 64 + lane < D; ++u) {
      o[u] *= alpha;
      for (int k = 0; k < n; ++k)
        if (rows[k] >= 0) o[u] += ps[k] * cached(c, c.v, c.vs, rows[k] + (int64_t)kvh * c.page.d, u * 64 + lane);
    }
    __syncthreads();
  }
  const int64_t out_at = (int64_t)(first + i) * a.out_stride + (int64_t)h * D;
  for (int u = 0; u * 64 + lane < D; ++u) {
    const float r = l == 0.0f ? 0.0f : o[u] / l;
    if (a.type == EMBER_TYPE_F16) static_cast<_Float16*>(a.out)[out_at + u * 64 + lane] = (_Float16)r;
    else static_cast<uint16_t*>(a.out)[out_at + u * 64 + lane] = ember_moe::bf16_rne(r);
  }
}

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
  p.step = (int64_t)c.max_q * a.G <= 64;
  if (!p.step) return p;
  // keys that the rows of a sequence can see at most, and one tile for where they begin within one
  int64_t range = c.cap;
  if (a.window > 0 && !a.prefix) range = std::min<int64_t>(range, (int64_t)a.window + c.max_q - 1);
  range = std::max<int64_t>(range, 1) + 31;
  const int64_t blocks = (int64_t)c.n_seqs * c.n_kv * ((c.max_q * a.G + 15) / 16);
  const int64_t most = (range + 127) / 128;
  int64_t splits = std::min<int64_t>({most, 256, (2048 + blocks - 1) / blocks});
  p.chunk = (int)((range + splits - 1) / splits + 127) / 128 * 128;
  p.splits = (int)((range + p.chunk - 1) / p.chunk);
  p.parts = p.splits > 1 ? p.splits : 0;
  return p;
}

size_t attn_scratch(const AttnArgs& a) {
  const AttnPlan p = attn_plan(a);
  return (size_t)p.parts * a.c.n_tokens * a.H * (a.c.D + 2) * 4;
}

int launch_attn(const AttnArgs& a, void* scratch, hipStream_t st) {
  const AttnPlan p = attn_plan(a);
  if (!p.step) {
    attn_row_kernel<<<dim3(a.c.max_q, a.H, a.c.n_seqs), 64, 0, st>>>(a);
    return hipGetLastError() == hipSuccess ? EMBER_OK : EMBER_ERR_LAUNCH;
  }
  Parts parts{nullptr, nullptr, (int64_t)a.c.n_tokens * a.H, std::max(p.parts, 1)};
  if (p.parts) {
    parts.o = static_cast<float*>(scratch);
    parts.ml = parts.o + p.parts * parts.rows * a.c.D;
  }
  auto* step = a.c.type == EMBER_TYPE_BF16 ? launch_step_bf16 : a.c.type == EMBER_TYPE_F16 ? launch_step_f16
               : a.type == EMBER_TYPE_BF16 ? launch_step_q8_bf16 : launch_step_q8_f16;
  if (int s = step(a, parts, p.splits, p.chunk, 0, st)) return s;
  if (!p.parts) return EMBER_OK;
  const dim3 grid(((unsigned)a.c.max_q * a.H + 3) / 4, a.c.n_seqs);
  if (a.type == EMBER_TYPE_BF16) attn_join_kernel<EMBER_TYPE_BF16><<<grid, 256, 0, st>>>(a, parts);
  else attn_join_kernel<EMBER_TYPE_F16><<<grid, 256, 0, st>>>(a, parts);
  return hipGetLastError() == hipSuccess ? EMBER_OK : EMBER_ERR_LAUNCH;
}

}  // namespace ember_attn_impl
