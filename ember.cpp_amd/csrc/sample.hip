// The pick of the next token (ember_sample): one block per row.
//
// Everything that decides is exact, so that the result depends on neither the order of the sums nor the grid: logits are
// compared as order-preserving 32-bit keys, and weights are summed as integers, w_i 2^s rounded once, with s such that
// a row's V weights (at most 1 each) stay below 2^62. Both filters are thresholds in the descending order: the key at
// which the count (top-k) or the weight (top-p) of the keys at or above it reaches its share, found digit by digit (11,
// 11, 10 bits) from a histogram in LDS, and how many of the logits equal to the threshold, by index, still belong.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ember_sample.h"
#include "moe_conv.hpp"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;
typedef unsigned long long u64;

struct Args {
  ember_sampler s;
  const void* z;
  int type, V;
  int64_t stride;
  const float* u;
  int32_t* ids;
  float* probs;
  int frac;  // s of the comment above
};

// Ascending in the logit; -0 as +0; 0 for what is never drawn (NaN, -inf), so every other key is larger.
__device__ inline uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.0f);
  if (z != z || b == 0xff800000u) return 0;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

template <int T>
__device__ inline float logit(const Args& a, int64_t row, int i) {
  const int64_t at = row * a.stride + i;
  if constexpr (T == EMBER_TYPE_F32) return static_cast<const float*>(a.z)[at];
  if constexpr (T == EMBER_TYPE_F16) return (float)static_cast<const _Float16*>(a.z)[at];
  return ember_moe::bf16_f32(static_cast<const uint16_t*>(a.z)[at]);
}

struct Shared {
  uint32_t cnt[kBins];
  u64 mass[kBins];
  u64 wave[kWaves];
  u64 got[4];
};

template <class F>
__device__ inline u64 block_sum(Shared& sh, u64 x, F) {
  for (int k = 32; k; k >>= 1) x += __shfl_xor(x, k);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = x;
  __syncthreads();
  u64 t = 0;
  for (int w = 0; w < kWaves; ++w) t += sh.wave[w];
  return t;
}
// Sum of x over the threads before this one; `total` over all.
__device__ inline u64 block_before(Shared& sh, u64 x, u64& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64 inc = x;
  for (int k = 1; k < 64; k <<= 1) {
    const u64 y = __shfl_up(inc, k);
    if (lane >= k) inc += y;
  }
  __syncthreads();
  if (lane == 63) sh.wave[wave] = inc;
  __syncthreads();
  u64 before = 0;
  total = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before += sh.wave[w];
    total += sh.wave[w];
  }
  return before + inc - x;
}

struct Weigh {
  float top;
  double inv_t;
  int frac;
  __device__ double e(uint32_t key) const {
    const float z = value_of(key);
    return z == top ? 1.0 : exp(((double)z - (double)top) * inv_t);
  }
  __device__ u64 fix(double e) const { return (u64)rint(ldexp(e, frac)); }
};

// The largest key t whose keys >= t have together at least `need` (by_mass: weight, else count), over the keys above
// `floor_key`, with `extra` of the floor key itself; `above` gets what the keys > t have.
template <int T, bool MASS>
__device__ uint32_t select(const Args& a, int64_t row, Shared& sh, const Weigh& w, uint32_t floor_key, u64 extra, u64 need, u64& above) {
  const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
  uint32_t prefix = 0;
  above = 0;
  for (int p = 0; p < 3; ++p) {
    const int sh_ = shifts[p], nb = 1 << bits[p];
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.mass[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < a.V; i += kThreads) {
      const uint32_t k = key_of(logit<T>(a, row, i));
      if (k <= floor_key || k == 0) continue;
      if (p && (k >> (sh_ + bits[p])) != prefix) continue;
      atomicAdd(&sh.mass[(k >> sh_) & (nb - 1)], MASS ? w.fix(w.e(k)) : 1ull);
    }
    __syncthreads();
    if (extra && threadIdx.x == 0 && (!p || (floor_key >> (sh_ + bits[p])) == prefix))
      sh.mass[(floor_key >> sh_) & (nb - 1)] += extra;
    __syncthreads();
    // the bin, from the top, at which the running sum reaches `need`: thread t has the bins nb - 1 - 2 t and the one below
    u64 x[2] = {0, 0};
    for (int e = 0; e < 2; ++e) {
      const int bin = nb - 1 - (2 * (int)threadIdx.x + e);
      if (bin >= 0) x[e] = sh.mass[bin];
    }
    u64 total, run = above + block_before(sh, x[0] + x[1], total);
    for (int e = 0; e < 2; ++e) {
      const int bin = nb - 1 - (2 * (int)threadIdx.x + e);
      if (bin >= 0 && run < need && run + x[e] >= need) {
        sh.got[0] = bin;
        sh.got[1] = run;
      }
      run += x[e];
    }
    __syncthreads();
    prefix = (prefix << bits[p]) | (uint32_t)sh.got[0];
    above = sh.got[1];
    __syncthreads();
  }
  return prefix;
}

template <int T>
__global__ __launch_bounds__(kThreads) void sample_kernel(Args a) {
  __shared__ Shared sh;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  float temp = a.s.temperatures ? a.s.temperatures[row] : a.s.temperature;
  int top_k = a.s.top_ks ? a.s.top_ks[row] : a.s.top_k;
  float top_p = a.s.top_ps ? a.s.top_ps[row] : a.s.top_p;
  float min_p = a.s.min_ps ? a.s.min_ps[row] : a.s.min_p;
  if (temp != temp) temp = 1.0f;
  if (top_p != top_p) top_p = 1.0f;
  if (!(min_p > 0.0f)) min_p = 0.0f;
  min_p = fminf(min_p, 1.0f);
  float u = a.u[row];
  u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;

  // the largest key, its lowest index, and how many can be drawn at all
  u64 best = 0;
  u64 n_valid = 0;
  for (int i = tid; i < a.V; i += kThreads) {
    const uint32_t k = key_of(logit<T>(a, row, i));
    n_valid += k != 0;
    const u64 x = (u64)k << 32 | (uint32_t)~i;
    best = x > best ? x : best;
  }
  for (int k = 32; k; k >>= 1) {
    const u64 o = __shfl_xor(best, k);
    best = o > best ? o : best;
  }
  if ((tid & 63) == 0) sh.wave[tid >> 6] = best;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) best = sh.wave[w] > best ? sh.wave[w] : best;
  n_valid = block_sum(sh, n_valid, 0);
  const uint32_t top_key = (uint32_t)(best >> 32);
  if (top_key == 0 || temp <= 0.0f || top_k == 1 || top_p <= 0.0f) {
    if (tid == 0) {
      a.ids[row] = top_key ? (int32_t)~(uint32_t)best : -1;
      if (a.probs) a.probs[row] = top_key ? 1.0f : 0.0f;
    }
    return;
  }
  const Weigh w{value_of(top_key), 1.0 / (double)temp, a.frac};

  // the threshold key and how many of the logits equal to it belong
  uint32_t t = 0;
  u64 ties = ~0ull, above;
  if (top_k > 0 && (u64)top_k < n_valid) {
    t = select<T, false>(a, row, sh, w, 0, 0, (u64)top_k, above);
    ties = (u64)top_k - above;
  }
  if (top_p < 1.0f) {
    const u64 wt = t ? w.fix(w.e(t)) : 0, extra = t ? ties * wt : 0;
    u64 sum = 0;
    for (int i = tid; i < a.V; i += kThreads) {
      const uint32_t k = key_of(logit<T>(a, row, i));
      if (k > t) sum += w.fix(w.e(k));
    }
    sum = block_sum(sh, sum, 0) + extra;
    const u64 need = max(1ull, (u64)ceil((double)top_p * (double)sum));
    const uint32_t t2 = select<T, true>(a, row, sh, w, t, extra, need, above);
    const u64 w2 = w.fix(w.e(t2)), n = (need - above + w2 - 1) / w2;
    ties = t2 == t ? min(ties, n) : n;
    t = t2;
  }

  // the kept tokens' weight, tile by tile of 1024 consecutive indices; then the tile, and the token in it
  auto weight = [&](uint32_t k, u64 rank) -> u64 {  // rank: how many of equal key come before
    if (k == 0 || k < t || (k == t && rank >= ties)) return 0;
    const double e = w.e(k);
    return e >= (double)min_p ? w.fix(e) : 0;
  };
  u64 sum = 0, seen = 0;
  for (int i0 = 0; i0 < a.V; i0 += kThreads) {
    const int i = i0 + tid;
    const uint32_t k = i < a.V ? key_of(logit<T>(a, row, i)) : 0;
    u64 n, rank = seen + block_before(sh, t && k == t, n);
    seen += n;
    sum += weight(k, rank);
  }
  sum = block_sum(sh, sum, 0);
  const u64 target = (u64)((double)u * (double)sum);
  u64 run = 0;
  seen = 0;
  for (int i0 = 0; i0 < a.V; i0 += kThreads) {
    const int i = i0 + tid;
    const uint32_t k = i < a.V ? key_of(logit<T>(a, row, i)) : 0;
    u64 n, rank = seen + block_before(sh, t && k == t, n);
    seen += n;
    const u64 x = weight(k, rank);
    const u64 before = run + block_before(sh, x, n);
    run += n;
    if (before <= target && target < before + x) {
      a.ids[row] = i;
      if (a.probs) a.probs[row] = (float)((double)x / (double)sum);
    }
    if (run > target) break;
  }
}

}  // namespace

extern "C" int ember_sample(const ember_sampler* s, const void* logits, int type, int n, int V, int64_t stride, const float* u,
                            int32_t* ids, float* probs, hipStream_t stream) {
  if (!s) return EMBER_ERR_NULL;
  if (type != EMBER_TYPE_F32 && type != EMBER_TYPE_F16 && type != EMBER_TYPE_BF16) return EMBER_ERR_TYPE;
  if (n < 0 || V < 1 || V > (1 << 24) || stride < V || stride > (int64_t)1 << 40) return EMBER_ERR_SHAPE;
  if (n == 0) return EMBER_OK;
  if (!logits || !u || !ids) return EMBER_ERR_NULL;
  const uintptr_t size = type == EMBER_TYPE_F32 ? 4 : 2;
  auto off = [](const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; };
  if (off(logits, size) || off(u, 4) || off(ids, 4) || off(probs, 4) || off(s->temperatures, 4) || off(s->top_ks, 4) ||
      off(s->top_ps, 4) || off(s->min_ps, 4))
    return EMBER_ERR_ALIGN;
  int bits = 0;
  while ((1 << bits) < V) ++bits;
  const Args a{*s, logits, type, V, stride, u, ids, probs, 61 - bits};
  switch (type) {
    case EMBER_TYPE_F32: sample_kernel<EMBER_TYPE_F32><<<n, kThreads, 0, stream>>>(a); break;
    case EMBER_TYPE_F16: sample_kernel<EMBER_TYPE_F16><<<n, kThreads, 0, stream>>>(a); break;
    default: sample_kernel<EMBER_TYPE_BF16><<<n, kThreads, 0, stream>>>(a); break;
  }
  return hipGetLastError() == hipSuccess ? EMBER_OK : EMBER_ERR_LAUNCH;
}
