// The pick of the next token (ember_sample): one block per row.
//
// Everything that decides is exact, so that the result depends on neither the order of the sums nor the grid: logits are
// compared as order-preserving 32-bit keys, and weights are summed as integers, w_i 2^s rounded once, with s such that
// a row's V weights (at most 1 each) stay below 2^62. Both filters are thresholds in the descending order: the key at
// which the count (top-k) or the weight (top-p) of the keys at or above it reaches its share, and how many of the logits equal
// to it, by index, still belong.
//
// A row takes as few passes as its settings allow; the first finds the largest logit.
//   * Where a bound leaves at most kCap tokens (top-k: the k-th largest of 2048 groups' maxima, four a thread, is no larger than the
//     k-th largest logit; min-p alone: its logit; or a short row), a second pass gathers them into LDS, 16 a thread, and the
//     rest works on these.
//   * Otherwise a filter takes a pass that puts the tokens into 2048 bins of equal width in the logit (by the key's digits, a
//     wave's lanes would meet in a few bins and wait for each other: 187 us for one row of 32000), after which the tokens down to the
//     bin that holds the threshold are gathered as above; or should they be too many those of that bin alone, for the threshold, or
//     should even these be (nearly all logits equal), three passes by the key's digits find it.
//   * Kept tokens that are too many to gather: a pass sums their weights in cells of consecutive tokens.
// 512 threads: what is between two barriers is short, and eight waves meet sooner than sixteen.
//
// One CU has a row, so few rows are bound by its own arithmetic and waits: 38 us for one of 32000 f32 by top-p, 3 of them the first pass, 14 the bins (10
// its weights), 5 the gathering, 10 five levels of selection in LDS (a bin's sum, two barriers and five round trips to LDS each). 128 rows of 131072, 67 MB, by all filters 52 us:
// the first pass 12, as fast as memory gives (5.5 TB/s), 20 the selection of a bound and the pass that gathers, the rest on what it gathered.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "ember_sample.h"
#include "moe_conv.hpp"

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kPer = 16, kCap = kPer * kThreads;  // gathered tokens, kPer * 64 of them by each wave
constexpr int kCell = 256;                       // tokens that a wave takes at once: 4 a lane, side by side
constexpr int kAhead = 16;                       // cells per wave whose loads are on the way at once: 128 KB per block
constexpr int kBinPer = kBins / kThreads;
static_assert(kBinPer == 4, "find_bin");
constexpr int kGroupMaxK = 1600;                 // top-k that the maxima of 2048 groups bound well
typedef unsigned long long u64;

struct Args {
  ember_sampler s;
  const void* z;
  int V;
  int64_t stride;
  const float* u;
  int32_t* ids;
  float* probs;
  int bits;        // s of the comment above, at most 51
  int cell_shift;  // the last pass sums cells of kCell << cell_shift tokens, at most kBins of them
};

// Ascending in the logit; -0 as +0; 0 for what is never drawn (NaN, -inf), so every other key is larger.
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.0f);
  if (z != z || b == 0xff800000u) return 0;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

struct Shared {
  alignas(16) u64 bin[kBins];
  union {
    u64 list[kCap];  // gathered: bits of the logit, index above them
    struct {
      u64 cell[kBins];
      uint32_t cell_ties[kBins];
    };
  };
  u64 wave[kWaves], meta[kWaves];
  u64 got[3];
  uint32_t counts[kWaves];  // gathered tokens of each wave
};

// The row's logits, -inf past its end. ALIGNED: every lane's 4 tokens can be loaded at once. (Passes compare logits, not keys: 2
// instructions a token where the keys took 13, and a pass over 131072 tokens 11 us of nothing else. NaN compares false. Every pass loads
// them again: kept in registers, a row of 32000 left too few for the weights, 52 us against 46.)
template <int T, bool ALIGNED>
struct Row {
  const char* p;
  int V;

  __device__ __forceinline__ void load(int at, float (&z)[4]) const {
    constexpr int size = T == EMBER_TYPE_F32 ? 4 : 2;
    typedef float f4 __attribute__((ext_vector_type(4)));
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    typedef uint16_t w4 __attribute__((ext_vector_type(4)));
    const char* const q = p + (int64_t)at * size;
    if (ALIGNED && at + 4 <= V) {
      if constexpr (T == EMBER_TYPE_F32) {
        const f4 y = *reinterpret_cast<const f4*>(q);
        for (int e = 0; e < 4; ++e) z[e] = y[e];
      } else if constexpr (T == EMBER_TYPE_F16) {
        const h4 y = *reinterpret_cast<const h4*>(q);
        for (int e = 0; e < 4; ++e) z[e] = (float)y[e];
      } else {
        const w4 y = *reinterpret_cast<const w4*>(q);
        for (int e = 0; e < 4; ++e) z[e] = ember_moe::bf16_f32(y[e]);
      }
    } else {
      for (int e = 0; e < 4; ++e) {
        z[e] = -INFINITY;
        if (at + e >= V) continue;
        if constexpr (T == EMBER_TYPE_F32) z[e] = reinterpret_cast<const float*>(q)[e];
        else if constexpr (T == EMBER_TYPE_F16) z[e] = (float)reinterpret_cast<const _Float16*>(q)[e];
        else z[e] = ember_moe::bf16_f32(reinterpret_cast<const uint16_t*>(q)[e]);
      }
    }
  }
  static __device__ int first() { return (int)(threadIdx.x >> 6) * kCell + (int)(threadIdx.x & 63) * 4; }
  // f(index of the first, logits) for this thread's tokens, 4 at a time; whole waves together.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
      for (int c0 = 0; c0 < V; c0 += kAhead * kWaves * kCell) {
        float x[kAhead][4];
#pragma unroll
        for (int c = 0; c < kAhead; ++c) load(first() + c0 + c * kWaves * kCell, x[c]);
#pragma unroll
        for (int c = 0; c < kAhead; ++c)
          if (c0 + c * kWaves * kCell < V) f(first() + c0 + c * kWaves * kCell, x[c]);
      }
  }
};

// x of lane l - N of the row of 16 (N < 16), or of the last lane of the row before (rows 1 and 3; or 2 and 3, from lane 31); 0 for none.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t from_lane(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 from_lane(u64 x) {
  return (u64)from_lane<CTRL, ROWS>((uint32_t)(x >> 32)) << 32 | from_lane<CTRL, ROWS>((uint32_t)x);
}
// f over the lanes up to this one (0 leaves a value as it is). By data-parallel moves: the shuffles go through LDS, 6 of them one after
// the other some 900 cycles for 64 bits.
template <class V, class F>
__device__ __forceinline__ V wave_scan(V x, F f) {
  x = f(x, from_lane<0x111, 0xf>(x));
  x = f(x, from_lane<0x112, 0xf>(x));
  x = f(x, from_lane<0x114, 0xf>(x));
  x = f(x, from_lane<0x118, 0xf>(x));
  x = f(x, from_lane<0x142, 0xa>(x));
  return f(x, from_lane<0x143, 0xc>(x));
}
__device__ __forceinline__ u64 last_lane(u64 x) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ uint32_t last_lane(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); }
template <class V>
__device__ __forceinline__ V wave_upto(V x) {
  return wave_scan(x, [](V p, V q) { return p + q; });
}
template <class V>
__device__ __forceinline__ V wave_sum(V x) {
  return last_lane(wave_upto(x));
}
template <class V>
__device__ __forceinline__ V wave_max(V x) {
  return last_lane(wave_scan(x, [](V p, V q) { return p > q ? p : q; }));
}
// Sum over the block. Ends with a barrier, as find_bin.
__device__ __forceinline__ u64 block_sum(Shared& sh, u64 x) {
  x = wave_sum(x);
  if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = x;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) t += sh.wave[w];
  __syncthreads();
  return t;
}
// Of n <= kBins bins, from the highest (down) or lowest on, the one at which the running sum from `run` reaches need: sh.got = {bin, the sum
// before it, the sum with it}. Leaves the bins cleared.
__device__ __forceinline__ void find_bin(Shared& sh, u64* bins, int n, bool down, u64 run, u64 need) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // four bins side by side per thread: 32 bytes at once (downwards n is a multiple of four)
  typedef u64 u64x2 __attribute__((ext_vector_type(2)));
  const int at = kBinPer * (int)threadIdx.x, b0 = down ? max(n - kBinPer - at, 0) : at;
  u64x2* const q = reinterpret_cast<u64x2*>(bins + b0);
  const u64x2 q0 = q[0], q1 = q[1];
  if (at < n) q[0] = q[1] = u64x2{0, 0};
  const u64 y[kBinPer] = {q0[0], q0[1], q1[0], q1[1]};
  u64 x[kBinPer], mine = 0;
  int b[kBinPer];
#pragma unroll
  for (int e = 0; e < kBinPer; ++e) {
    b[e] = down ? n - 1 - at - e : at + e;
    x[e] = at + e >= n ? 0 : down ? y[kBinPer - 1 - e] : y[e];
    mine += x[e];
  }
  const u64 upto = wave_upto(mine);
  if (lane == 63) sh.wave[wave] = upto;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) run += w < wave ? sh.wave[w] : 0;
  run += upto - mine;
#pragma unroll
  for (int e = 0; e < kBinPer; ++e) {
    if (run < need && run + x[e] >= need) {
      sh.got[0] = (u64)b[e];
      sh.got[1] = run;
      sh.got[2] = run + x[e];
    }
    run += x[e];
  }
  __syncthreads();
}

// exp((z - top) / temperature), as p 2^n: 2^f for the fraction f, by its Taylor series to the 11th power (at |f| <= 1/2 the rest is under 2^-47),
// n rounded off by adding 1.5 2^52 and scaled by adding to the exponent: some 25 instructions, no conversion among them but the logit's. Infinite logits count as 2^200, which is as far from every finite one as it takes.
struct Weigh {
  float top;
  double far, c;  // min(top, 2^200); log2(e) / temperature
  int s;          // weights are summed as integers, times 2^s
  __device__ __forceinline__ double part(float z, int& n) const {
    const double y = fmax((fmin((double)z, 0x1p200) - far) * c, -900.0), t = y + 0x1.8p52, f = y - (t - 0x1.8p52);
    n = (int)(uint32_t)__double_as_longlong(t);
    double p = 4.44553827187081e-10;
    p = __builtin_fma(p, f, 7.054911620801121e-09);
    p = __builtin_fma(p, f, 1.0178086009239696e-07);
    p = __builtin_fma(p, f, 1.3215486790144305e-06);
    p = __builtin_fma(p, f, 1.5252733804059838e-05);
    p = __builtin_fma(p, f, 0.00015403530393381606);
    p = __builtin_fma(p, f, 0.0013333558146428441);
    p = __builtin_fma(p, f, 0.009618129107628477);
    p = __builtin_fma(p, f, 0.055504108664821576);
    p = __builtin_fma(p, f, 0.2402265069591007);
    p = __builtin_fma(p, f, 0.6931471805599453);
    return __builtin_fma(p, f, 1.0);
  }
  __device__ __forceinline__ double e(float z) const {
    int n;
    const double p = part(z, n);
    return scaled(p, n);
  }
  __device__ __forceinline__ double e(uint32_t key) const { return e(value_of(key)); }
  // x 2^n, both normal
  static __device__ __forceinline__ double scaled(double x, int n) {
    const u64 b = (u64)__double_as_longlong(x);
    return __longlong_as_double((long long)((u64)((uint32_t)(b >> 32) + ((uint32_t)n << 20)) << 32 | (uint32_t)b));
  }
  // e 2^s (at most 2^51) to the nearest integer: the low bits of 2^52 plus it
  static __device__ __forceinline__ u64 integer(double e) { return (u64)__double_as_longlong(e + 0x1p52) & 0xfffffffffffffull; }
  __device__ __forceinline__ u64 fix(double e) const { return integer(scaled(e, s)); }
  __device__ __forceinline__ u64 at(float z) const {
    int n;
    const double p = part(z, n);
    return integer(scaled(p, n + s));
  }
  // Of four, 0 for what is never drawn: side by side, without branches (each step waits for the one before: a token at a time a pass over 131072 took 11 us more).
  __device__ __forceinline__ void at4(const float (&z)[4], u64 (&x)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = at(fmaxf(z[e], -INFINITY));  // (NaN: -inf, whose weight is 0)
  }
};

// Over the threads' items (the first n, the same for a wave; amount a[i], 0: none): the largest key t in [lo, hi] whose keys >= t hold `need` together with `above`, which
// gets what the keys > t hold. Eleven bits of the difference to lo at a time.
template <int N>
__device__ __forceinline__ uint32_t select_items(Shared& sh, const uint32_t (&key)[N], const u64 (&a)[N], int n, uint32_t lo, uint32_t hi, u64 need, u64& above) {
  uint32_t width = hi - lo;
  int s = max(0, 32 - __clz((int)width) - 11);
  for (;;) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n && a[i] && key[i] - lo <= width) atomicAdd(&sh.bin[(key[i] - lo) >> s], a[i]);  // (a key under lo is far above width)
    __syncthreads();
    find_bin(sh, sh.bin, kBins, true, above, need);
    lo += (uint32_t)sh.got[0] << s;
    above = sh.got[1];
    if (s == 0) return lo;
    width = (1u << s) - 1;
    s = max(0, s - 11);
  }
}

// Gathers the tokens that `is` picks (by their logit; none that is never drawn), each wave those of its cells, in any order; whether they fit.
// (A list for all, its places given out by an atomic, had every wave wait for LDS at each cell: 9 us of 42 for a row of 32000.)
template <class R, class F>
__device__ __forceinline__ bool gather(const R& r, Shared& sh, F is) {
  const int wave = threadIdx.x >> 6, base = wave * kPer * 64;
  uint32_t count = 0;  // the wave's
  r.each([&](int i, const float (&z)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = is(z[e]);
      const u64 mask = __ballot(in);
      if (!mask) continue;
      const uint32_t at = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
      if (in && at < kPer * 64) {
        sh.list[base + at] = (u64)(uint32_t)(i + e) << 32 | __float_as_uint(z[e]);
      }
      count += (uint32_t)__popcll(mask);
    }
  });
  if ((threadIdx.x & 63) == 0) sh.counts[wave] = count;
  __syncthreads();
  bool fits = true;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) fits &= sh.counts[v] <= kPer * 64;
  __syncthreads();
  return fits;
}
// This thread's gathered item i, whether there is one; the wave's number of items per thread.
__device__ __forceinline__ bool item(const Shared& sh, int i, uint32_t& key, uint32_t& idx) {
  const int wave = threadIdx.x >> 6, at = i * 64 + (int)(threadIdx.x & 63);
  if (at >= (int)sh.counts[wave]) return false;
  const u64 x = sh.list[wave * kPer * 64 + at];
  key = key_of(__uint_as_float((uint32_t)x));
  idx = (uint32_t)(x >> 32);
  return true;
}
__device__ __forceinline__ int items(const Shared& sh) {
  return (__builtin_amdgcn_readfirstlane((int)sh.counts[threadIdx.x >> 6]) + 63) / 64;
}

// select_items over the whole row by the key's digits, for the keys above floor_key and `extra` for that key itself. MASS: by weight.
template <bool MASS, class R>
__device__ __forceinline__ uint32_t select_row(const R& r, Shared& sh, const Weigh& w, uint32_t floor_key, u64 extra, u64 need, u64& above) {
  uint32_t prefix = 0;
  above = 0;
  for (int p = 0; p < 3; ++p) {
    const int s = p == 0 ? 21 : p == 1 ? 10 : 0, bits = p == 2 ? 10 : 11, nb = 1 << bits;
    r.each([&](int, const float (&z)[4]) {
      for (int e = 0; e < 4; ++e) {
        const uint32_t k = key_of(z[e]);
        if (k > floor_key && (!p || (k >> (s + bits)) == prefix)) atomicAdd(&sh.bin[(k >> s) & (nb - 1)], MASS ? w.at(z[e]) : 1ull);
      }
    });
    if (extra && threadIdx.x == 0 && (!p || (floor_key >> (s + bits)) == prefix)) atomicAdd(&sh.bin[(floor_key >> s) & (nb - 1)], extra);
    __syncthreads();
    find_bin(sh, sh.bin, nb, true, above, need);
    prefix = (prefix << bits) | (uint32_t)sh.got[0];
    above = sh.got[1];
  }
  return prefix;
}

// Bins of equal width from the largest logit down to `low`.
struct Bins {
  float top, scale;
  __device__ __forceinline__ Bins(float top_, float low) : top(top_), scale((float)(kBins - 1) / fmaxf(top_ - low, 1e-30f)) {}
  // (each step of it is monotone in z, rounded or not, and what overflows to NaN comes last, after infinity)
  __device__ __forceinline__ int operator()(float z) const { return kBins - 1 - (int)fminf((top - z) * scale, (float)(kBins - 1)); }
  // a logit that none of the tokens in bin b and higher ones is under
  __device__ __forceinline__ float from(int b) const {
    if (b == 0) return -3.4028235e38f;
    const float z = top - (float)(kBins - b) / scale;
    return fmaxf(z - 1e-5f * (fabsf(z) + fabsf(top)), -3.4028235e38f);  // (the steps' roundings: some 2^-22 of either)
  }
};

// The bin that holds the threshold, of the keys above floor_key and `extra` for that key itself: sh.got as by find_bin. MASS: by weight, need
// being set to the share `share` of the whole.
template <bool MASS, class R>
__device__ __forceinline__ void bins_row(const R& r, Shared& sh, const Weigh& w, const Bins& bin_of, uint32_t floor_key, u64 extra, double share, u64& need) {
  u64 sum = threadIdx.x == 0 ? extra : 0;
  const float above = floor_key ? value_of(floor_key) : -INFINITY;
  r.each([&](int, const float (&z)[4]) {
    u64 x[4] = {1, 1, 1, 1};
    if (MASS) w.at4(z, x);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (z[e] > above && x[e]) {
        atomicAdd(&sh.bin[bin_of(z[e])], x[e]);
        sum += x[e];
      }
  });
  if (extra && threadIdx.x == 0) atomicAdd(&sh.bin[bin_of(above)], extra);
  if (MASS) need = max(1ull, (u64)ceil(share * (double)block_sum(sh, sum)));
  else __syncthreads();
  find_bin(sh, sh.bin, kBins, true, 0, need);
}

// The threshold itself, in bin b with `above` before it.
template <bool MASS, class R>
__device__ __forceinline__ uint32_t threshold_row(const R& r, Shared& sh, const Weigh& w, const Bins& bin_of, int b, uint32_t floor_key, u64 extra, u64 need,
                                                  u64& above) {
  const float under = floor_key ? value_of(floor_key) : -INFINITY;
  if (!gather(r, sh, [&](float z) { return z > under && bin_of(z) == b; })) return select_row<MASS>(r, sh, w, floor_key, extra, need, above);
  uint32_t key[kPer], lo = ~0u, hi = 0;
  u64 x[kPer], here = 0;
  const int n = items(sh);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    uint32_t idx;
    key[i] = 0;
    x[i] = 0;
    if (i < n && item(sh, i, key[i], idx)) {
      x[i] = MASS ? w.fix(w.e(key[i])) : 1ull;
      here += x[i];
      lo = min(lo, key[i]), hi = max(hi, key[i]);
    }
  }
  if (extra) {  // should the bin's tokens not reach `need`, it is the floor key, in the same bin, that does
    here = block_sum(sh, here);
    if (above + here < need) {
      above += here;
      return floor_key;
    }
  }
  lo = ~wave_max(~lo);
  hi = wave_max(hi);
  if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = (u64)hi << 32 | lo;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    lo = min(lo, (uint32_t)sh.wave[v]);
    hi = max(hi, (uint32_t)(sh.wave[v] >> 32));
  }
  __syncthreads();
  return select_items(sh, key, x, n, lo, hi, need, above);
}

template <int T, bool ALIGNED>
__global__ __launch_bounds__(kThreads) void sample_kernel(Args a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  Shared& sh = *reinterpret_cast<Shared*>(lds);
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  float temp = a.s.temperatures ? a.s.temperatures[row] : a.s.temperature;
  const int top_k = a.s.top_ks ? a.s.top_ks[row] : a.s.top_k;
  float top_p = a.s.top_ps ? a.s.top_ps[row] : a.s.top_p;
  float min_p = a.s.min_ps ? a.s.min_ps[row] : a.s.min_p;
  if (temp != temp) temp = 1.0f;
  if (top_p != top_p) top_p = 1.0f;
  if (!(min_p > 0.0f)) min_p = 0.0f;
  min_p = fminf(min_p, 1.0f);
  float u = a.u[row];
  u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
  Row<T, ALIGNED> r;
  r.p = static_cast<const char*>(a.z) + row * a.stride * (T == EMBER_TYPE_F32 ? 4 : 2);
  r.V = a.V;

  // the largest logit of the row and of this thread's four groups, which four tokens first held its largest, how many can be drawn
#pragma unroll
  for (int i = 0; i < kBinPer; ++i) sh.bin[i * kThreads + tid] = 0;
  float group[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, best = -INFINITY;
  uint32_t best_i = 0, n_valid = 0;
  r.each([&](int i, const float (&z)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      group[e] = fmaxf(group[e], z[e]);
      n_valid += (uint32_t)__popcll(__ballot(z[e] > -INFINITY));  // (the wave's)
    }
    const float m = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
    if (m > best) best = m, best_i = (uint32_t)i;  // (a thread's indices ascend)
  });
  uint32_t group_key[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) group_key[e] = key_of(group[e]);
  u64 first = wave_max((u64)key_of(best) << 32 | (uint32_t)~best_i);
  // the smallest of the groups' largest (0: a group without a token that can be drawn)
  uint32_t least = ~wave_max(~min(min(group_key[0], group_key[1]), min(group_key[2], group_key[3])));
  if (lane == 0) {
    sh.wave[wave] = first;
    sh.meta[wave] = (u64)n_valid << 32 | least;
  }
  __syncthreads();
  n_valid = 0;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    first = sh.wave[v] > first ? sh.wave[v] : first;
    least = min(least, (uint32_t)sh.meta[v]);
    n_valid += (uint32_t)(sh.meta[v] >> 32);
  }
  __syncthreads();
  const uint32_t top_key = (uint32_t)(first >> 32);
  if (top_key == 0 || temp <= 0.0f || top_k == 1 || top_p <= 0.0f) {
    if (tid == 0) {
      int id = -1;
      if (top_key) {  // the first of the four
        float z[4];
        r.load((int)~(uint32_t)first, z);
        id = (int)~(uint32_t)first + (key_of(z[0]) == top_key ? 0 : key_of(z[1]) == top_key ? 1 : key_of(z[2]) == top_key ? 2 : 3);
      }
      a.ids[row] = id;
      if (a.probs) a.probs[row] = top_key ? 1.0f : 0.0f;
    }
    return;
  }
  const float top = value_of(top_key);
  const Weigh w{top, fmin((double)top, 0x1p200), top > 3.4028235e38f ? 1.0 : 1.4426950408889634074 / (double)temp, a.bits};
  bool by_k = top_k > 0 && (uint32_t)top_k < n_valid, by_p = top_p < 1.0f;

  // a key that no token to be kept is under: `low` of all, `floor` (0: none) where few tokens are at or above it
  uint32_t low = 1, floor = 0;
  if (min_p > 0.0f && !by_p && !by_k) {
    // the logit of weight min_p, less what its rounding may be off by
    const double z = (double)w.top + (double)temp * log((double)min_p), off = 1e-6 * (fabs(z) + (double)temp);
    low = floor = max(low, key_of((float)(z - off)));
  }
  if (n_valid <= kCap) floor = low;
  if (by_k && top_k <= kGroupMaxK && !floor) {
    u64 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = group_key[e] != 0;
    u64 above = 0;
    if (block_sum(sh, x[0] + x[1] + x[2] + x[3]) >= (u64)top_k) low = floor = select_items(sh, group_key, x, 4, max(least, 1u), top_key, (u64)top_k, above);
  }
  auto from = [](float bound) { return [bound](float z) { return z >= bound; }; };
  // (key 1 is a NaN's neighbour: the lowest logit that can be drawn)
  bool listed = floor && gather(r, sh, from(floor == 1 ? -3.4028235e38f : value_of(floor)));
  // of the threshold key, if it is known before the tokens are gathered, how many of the logits equal to it belong; the weight that top-p
  // needs, if it is known (0: not)
  uint32_t t = 0;
  u64 ties = ~0ull, need_p = 0;
  if (!listed && by_k) {
    u64 need = (u64)top_k;
    // (twice as far down as the groups' largest reach: what is further comes into the last bin)
    const float reach = least > 1 ? w.top - 2.0f * (w.top - value_of(least)) : -3.4028235e38f;
    const Bins bin_of(w.top, fmaxf(reach, low > 1 ? value_of(low) : reach));
    bins_row<false>(r, sh, w, bin_of, 0, 0, 0.0, need);
    const int b = (int)sh.got[0];
    u64 above = sh.got[1];
    const u64 upto = sh.got[2];
    if (upto <= kCap) {
      listed = gather(r, sh, from(bin_of.from(b)));
    }
    if (!listed) {
      t = threshold_row<false>(r, sh, w, bin_of, b, 0, 0, need, above);
      ties = need - above;
      by_k = false;
      low = t;
      // (the k tokens and the ties)
      if ((u64)top_k <= kCap) listed = gather(r, sh, from(value_of(t)));
    }
  }
  if (!listed && by_p) {
    // (weights under e^-43 are 0: tokens further down hold nothing)
    const u64 extra = t ? ties * w.fix(w.e(t)) : 0;
    const Bins bin_of(w.top, fmaxf(max(t, low) > 1 ? value_of(max(t, low)) : -3.4028235e38f, w.top - 43.0f * temp));
    bins_row<true>(r, sh, w, bin_of, t, extra, (double)top_p, need_p);
    const int b = (int)sh.got[0];
    u64 above = sh.got[1];
    if (!t) listed = gather(r, sh, from(bin_of.from(b)));
    if (!listed) {
      const uint32_t t2 = threshold_row<true>(r, sh, w, bin_of, b, t, extra, need_p, above);
      const u64 each_ = w.fix(w.e(t2)), n = (need_p - above + each_ - 1) / each_;
      ties = t2 == t ? min(ties, n) : n;
      t = low = t2;
      by_p = false;
      listed = gather(r, sh, from(value_of(t)));
    }
  }

  if (listed) {
    uint32_t key[kPer], idx[kPer];  // idx: inverted, so that the first index is the largest
    u64 x[kPer];
    const uint32_t inv_lo = ~(uint32_t)(a.V - 1);
    const int n = items(sh);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      key[i] = 0;
      idx[i] = ~0u;
      x[i] = i < n && item(sh, i, key[i], idx[i]);
      idx[i] = ~idx[i];
    }
    // keeps of the items equal to t the first `keep` by index, and none under it
    auto cut = [&](uint32_t t_, u64 keep) {
      u64 eq[kPer], mine = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        eq[i] = 0;
        if (i >= n) continue;
        if (key[i] < t_) x[i] = 0;
        eq[i] = x[i] && key[i] == t_;
        mine += eq[i];
      }
      if (block_sum(sh, mine) <= keep) return;
      u64 before = 0;
      const uint32_t last = select_items(sh, idx, eq, n, inv_lo, ~0u, keep, before);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (eq[i] && idx[i] < last) x[i] = 0;
    };
    if (t) cut(t, ties);
    if (by_k) {
      u64 above = 0;
      const uint32_t t_ = select_items(sh, key, x, n, low, top_key, (u64)top_k, above);
      cut(t_, (u64)top_k - above);
    }
    uint32_t under = 0;  // bit i: item i has less than min_p
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < n && x[i]) {
        const double e = w.e(key[i]);
        x[i] = w.fix(e);
        under |= (uint32_t)(e < (double)min_p) << i;
      }
    if (by_p) {
      u64 mine = 0, above = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) mine += x[i];
      const u64 need = need_p ? need_p : max(1ull, (u64)ceil((double)top_p * (double)block_sum(sh, mine)));
      const uint32_t t_ = select_items(sh, key, x, n, low, top_key, need, above);
      const u64 each_ = w.fix(w.e(t_));
      cut(t_, (need - above + each_ - 1) / each_);
    }
    u64 mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (under >> i & 1) x[i] = 0;
      mine += x[i];
    }
    const u64 sum = block_sum(sh, mine), target = (u64)((double)u * (double)sum);
    u64 before = 0;
    const uint32_t drawn = select_items(sh, idx, x, n, inv_lo, ~0u, target + 1, before);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (x[i] && idx[i] == drawn) {
        a.ids[row] = (int32_t)~drawn;
        if (a.probs) a.probs[row] = (float)((double)x[i] / (double)sum);
      }
    return;
  }

  // Too many to gather: the weights of the tokens above t, and the tokens equal to it, by cells of consecutive tokens, a wave a cell.
  auto weight = [&](float z) -> u64 {
    const double e = w.e(fmaxf(z, -INFINITY));
    return e >= (double)min_p ? Weigh::integer(Weigh::scaled(e, w.s)) : 0;
  };
  const float tz = t ? value_of(t) : -INFINITY;
  const u64 wt = t ? weight(tz) : 0;
  const int cells = (a.V + (kCell << a.cell_shift) - 1) / (kCell << a.cell_shift);
  for (int c = wave; c < cells; c += kWaves) {
    u64 x = 0;
    uint32_t eq = 0;
    for (int sub = 0; sub < 1 << a.cell_shift; ++sub) {
      float z[4];
      u64 y[4];
      r.load(((c << a.cell_shift) + sub) * kCell + lane * 4, z);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = weight(z[e]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x += z[e] > tz ? y[e] : 0;
        eq += t && z[e] == tz;
      }
    }
    x = wave_sum(x);
    eq = wave_sum(eq);
    if (lane == 0) {
      sh.cell[c] = x;
      sh.cell_ties[c] = eq;
    }
  }
  __syncthreads();
  // of the equal ones the first `ties` count
  {
    u64 n[kBinPer], all = 0;
#pragma unroll
    for (int e = 0; e < kBinPer; ++e) {
      n[e] = kBinPer * tid + e < cells ? sh.cell_ties[kBinPer * tid + e] : 0;
      all += n[e];
    }
    const u64 upto = wave_upto(all);
    if (lane == 63) sh.wave[wave] = upto;
    __syncthreads();
    u64 before = upto - all, mine = 0;
    for (int v = 0; v < wave; ++v) before += sh.wave[v];
#pragma unroll
    for (int e = 0; e < kBinPer; ++e) {
      const int c = kBinPer * tid + e;
      const u64 kept = before >= ties ? 0 : min(n[e], ties - before);
      if (c < cells) {
        sh.cell[c] += kept * wt;
        sh.bin[c] = kept;
        mine += sh.cell[c];
      }
      before += n[e];
    }
    __syncthreads();
    const u64 sum = block_sum(sh, mine), target = (u64)((double)u * (double)sum);
    find_bin(sh, sh.cell, cells, false, 0, target + 1);
    if (wave) return;
    const int c = (int)sh.got[0];
    u64 run = sh.got[1], left = sh.bin[c];
    for (int sub = 0; sub < 1 << a.cell_shift; ++sub) {
      float z[4];
      const int at = ((c << a.cell_shift) + sub) * kCell + lane * 4;
      r.load(at, z);
      uint32_t eq = 0;
      for (int e = 0; e < 4; ++e) eq += t && z[e] == tz;
      const uint32_t eq_upto = wave_upto(eq);
      u64 rank = eq_upto - eq, x[4], mine_ = 0;
      for (int e = 0; e < 4; ++e) {
        x[e] = z[e] > tz ? weight(z[e]) : 0;
        if (t && z[e] == tz) x[e] = rank++ < left ? wt : 0;
        mine_ += x[e];
      }
      const u64 upto = wave_upto(mine_);
      u64 at_run = run + upto - mine_;
      for (int e = 0; e < 4; ++e) {
        if (at_run <= target && target < at_run + x[e]) {
          a.ids[row] = at + e;
          if (a.probs) a.probs[row] = (float)((double)x[e] / (double)sum);
        }
        at_run += x[e];
      }
      run += last_lane(upto);
      left -= min(left, (u64)last_lane(eq_upto));
    }
  }
}

template <int T>
int launch(const Args& a, int n, bool aligned, hipStream_t st) {
  auto go = [&](auto* kernel) {
    static_assert(sizeof(Shared) <= 160 * 1024, "LDS of a CU");
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared)) != hipSuccess)
      return (int)EMBER_ERR_LAUNCH;
    kernel<<<n, kThreads, sizeof(Shared), st>>>(a);
    return hipGetLastError() == hipSuccess ? (int)EMBER_OK : (int)EMBER_ERR_LAUNCH;
  };
  return aligned ? go(sample_kernel<T, true>) : go(sample_kernel<T, false>);
}

}  // namespace

extern "C" int ember_sample(const ember_sampler* s, const void* logits, int type, int n, int V, int64_t stride, const float* u,
                            int32_t* ids, float* probs, hipStream_t stream) {
  if (!s) return EMBER_ERR_NULL;
  if (type != EMBER_TYPE_F32 && type != EMBER_TYPE_F16 && type != EMBER_TYPE_BF16) return EMBER_ERR_TYPE;
  // (the runtime counts a launch's threads in 32 bits)
  if (n < 0 || n > (1 << 23) - 1 || V < 1 || V > (1 << 24) || stride < V || stride > (int64_t)1 << 40) return EMBER_ERR_SHAPE;
  if (n == 0) return EMBER_OK;
  if (!logits || !u || !ids) return EMBER_ERR_NULL;
  const uintptr_t size = type == EMBER_TYPE_F32 ? 4 : 2;
  auto off = [](const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; };
  if (off(logits, size) || off(u, 4) || off(ids, 4) || off(probs, 4) || off(s->temperatures, 4) || off(s->top_ks, 4) ||
      off(s->top_ps, 4) || off(s->min_ps, 4))
    return EMBER_ERR_ALIGN;
  int bits = 0, shift = 0;
  while ((1 << bits) < V) ++bits;
  while (((V + (kCell << shift) - 1) / (kCell << shift)) > kBins) ++shift;
  const bool aligned = !off(logits, 4 * size) && (n == 1 || stride % 4 == 0);
  const Args a{*s, logits, V, stride, u, ids, probs, std::min(51, 61 - bits), shift};
  switch (type) {
    case EMBER_TYPE_F32: return launch<EMBER_TYPE_F32>(a, n, aligned, stream);
    case EMBER_TYPE_F16: return launch<EMBER_TYPE_F16>(a, n, aligned, stream);
    default: return launch<EMBER_TYPE_BF16>(a, n, aligned, stream);
  }
}
