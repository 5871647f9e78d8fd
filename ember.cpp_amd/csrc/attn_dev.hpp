// What the attention kernels share (device side): matrix-core operands, the cache's tiles in LDS, masks and scores.
//
// Scores are computed transposed, S^T = K Q^T: the lane that holds a score's column then holds several keys of ONE query row,
// so the softmax needs few exchanges between lanes, and the weights already lie as the operand that O^T = V^T P^T takes (a
// contraction may go through the keys in any order, so V is read in the order that the scores came out in). V^T comes out
// of row-major LDS by the transposing reads. Both tiles lie in LDS with their 16-byte chunks permuted within the row by the
// key, so that reads down a column of rows touch all banks.
#pragma once
#include "attn_internal.hpp"
#include "moe_conv.hpp"

namespace ember_attn_impl {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef int i2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
#define EMBER_LDS(T) __attribute__((address_space(3))) T

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoScore = -1e30f;  // the running maximum before any score: finite, so that no difference is NaN

// Cache type T: what its tiles and operands are. BF16 caches multiply in bf16, F16 and Q8_0 ones in fp16 (an int8 code is
// exact in either; code * scale, rounded to fp16's 11 bits, is off by 2^-12 of itself at most, in bf16 it were 2^-9).
template <int T>
struct Op {
  static constexpr bool kBf16 = T == EMBER_TYPE_BF16;
  static constexpr bool kQ8 = T == EMBER_TYPE_Q8_0;
  static constexpr int kBytes = kQ8 ? 1 : 2;
};

template <bool BF16>
__device__ inline f4 mma16(s8 a, s8 b, f4 c) {
  if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
// Two floats to two operand halves, nearest even.
template <bool BF16>
__device__ inline uint32_t pack2(float x, float y) {
  if constexpr (BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, b2{(__bf16)x, (__bf16)y});
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, h2{(_Float16)x, (_Float16)y});
  }
}
__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Four int8 codes (the bytes of w) as fp16, exactly: 0x6400 | byte is 1024 + byte.
__device__ inline u2 codes_to_half(uint32_t w) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  const uint32_t x = w ^ 0x80808080u;  // code + 128
  const uint32_t lo = __builtin_amdgcn_perm(x, 0x64646464u, 0x00050004u), hi = __builtin_amdgcn_perm(x, 0x64646464u, 0x00070006u);
  const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
  return u2{__builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, lo) - off), __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, hi) - off)};
}
// 8 codes times a scale (the same for all, or one each in `s`).
__device__ inline s8 codes_times(u2 w, h8 s) {
  const u2 a = codes_to_half(w[0]), b = codes_to_half(w[1]);
  const u4 c = {a[0], a[1], b[0], b[1]};
  return __builtin_bit_cast(s8, __builtin_bit_cast(h8, c) * s);
}

// 16 bytes per lane from global memory into LDS, lane after lane from `lds` on, without registers.
__device__ inline void load_to_lds(const void* g, char* lds) {
  __builtin_amdgcn_global_load_lds(g, (EMBER_LDS(void)*)lds, 16, 0, 0);
}
// All of this wave's loads, to registers and to LDS, have arrived; all its LDS reads are done.
__device__ inline void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  asm volatile("" ::: "memory");
}
__device__ inline void wait_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
}

// Whether one of 8 halves is infinite or NaN.
template <bool BF16>
__device__ inline bool not_finite(u4 v) {
  constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
  bool r = false;
#pragma unroll
  for (int w = 0; w < 4; ++w) r |= (v[w] & e) == e || (v[w] & (e << 16)) == (e << 16);
  return r;
}

// Largest value over the lanes that hold the same query row.
__device__ inline float max_lanes32(float x) {  // lanes l, l ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float max_lanes16(float x) {  // lanes l, l ^ 16
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float sum_lanes32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ inline float sum_lanes16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Byte offset of 16-byte chunk c of key row `key` in a K tile of rows of CH chunks. Lanes read 16 keys at one chunk:
// they are spread over the chunk places of a 256-byte stretch (64 banks).
template <int CH>
__device__ inline int k_at(int key, int c) {
  constexpr int R = CH >= 16 ? 1 : 16 / CH;  // rows in 256 bytes
  return (key * CH + (c ^ ((key / R) & ((CH < 16 ? CH : 16) - 1)))) * 16;
}
// The same in a V tile, which the transposing reads go through: of halves 32 bytes (16 columns) of 4 keys at once and of the
// next 4 in the next 16 lanes, so pairs of chunks move together; of codes 16 bytes of keys n .. n + 3 and n + 16 .. n + 19.
template <int CH, bool Q8>
__device__ inline int v_at(int key, int c) {
  if constexpr (Q8) {
    constexpr int R = CH >= 16 ? 1 : 16 / CH;
    return (key * CH + (c ^ (((key / R) ^ ((key >> 4) * (CH / 2))) & (CH - 1)))) * 16;
  } else {
    constexpr int R = CH >= 16 ? 1 : 16 / CH, P = CH / 2 < 8 ? CH / 2 : 8;
    return (key * CH + ((((c >> 1) ^ ((key / R) & (P - 1))) << 1) | (c & 1))) * 16;
  }
}

// The keys that a query at position p sees: [lo, hi).
struct Span {
  int lo, hi;
};
__device__ inline Span visible(const AttnArgs& a, int64_t p, int len, int prefix) {
  if (p < 0) return {0, 0};
  const int lo = a.window > 0 ? (int)max((int64_t)0, p - a.window + 1) : 0;
  return {lo, (int)min((int64_t)len, max(p + 1, (int64_t)prefix))};
}

// Scores in units of log2 from products s: c = scale log2(e); where they are capped c = scale * 2 / softcap * log2(e), for the exponential in
// tanh x = 1 - 2 / (1 + exp(2 x)), whose error is absolute, a few 2^-24 of the cap. Both options are the same for a launch: loops of their own.
struct Scores {
  float c, cap, slope;  // cap: softcap * log2(e), 0 if there is none; slope: slopes[h] * log2(e), used if `sloped`
  bool sloped;
  // N scores, of the keys at distance dist + key(i)
  template <int N, class S, class K>
  __device__ __forceinline__ void operator()(S&& s, int dist, K key) const {
    if (cap > 0.0f) {
#pragma unroll
      for (int i = 0; i < N; ++i) s(i) = __builtin_fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(1.0f + exp2_fast(s(i) * c)), cap);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) s(i) *= c;
    }
    if (sloped) {
      const float d = (float)dist;
#pragma unroll
      for (int i = 0; i < N; ++i) s(i) = __builtin_fmaf(-slope, __builtin_fabsf(d + (float)key(i)), s(i));
    }
  }
};
// -inf for the scores of keys outside [from, to), key(i) being score i's.
template <int N, class S, class K>
__device__ __forceinline__ void mask_scores(S&& s, int from, int to, K key) {
  const uint32_t span = (uint32_t)max(to - from, 0);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if ((uint32_t)(key(i) - from) >= span) s(i) = -INFINITY;
}

// Where partial results go: for part s and row r of the call (token * n_heads + head) the sum of weighted values o[s][r][D], not
// yet divided, and the maximum (log2 units) and sum of weights ml[s][r][2].
struct Parts {
  float* o;
  float* ml;
  int64_t rows;  // n_tokens * n_heads
  int n;         // parts; 1 with o null: results go to `out`
};

}  // namespace ember_attn_impl
