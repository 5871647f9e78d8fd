// Attention over the paged cache (ember_attn).
#include "attn_internal.hpp"
#include "moe_conv.hpp"

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

}  // namespace

int launch_attn(const AttnArgs& a, void*, hipStream_t st) {
  attn_row_kernel<<<dim3(a.c.max_q, a.H, a.c.n_seqs), 64, 0, st>>>(a);
  return hipGetLastError() == hipSuccess ? EMBER_OK : EMBER_ERR_LAUNCH;
}

}  // namespace ember_attn_impl
