// K and V rows into and out of the paged cache (ember_kv_store, ember_kv_load).
//
// A row's values go through in chunks of 8 (one 16-byte load of halves), consecutive threads on consecutive chunks, so
// rows are read and pages written in whole 128-byte lines; a Q8_0 block of 32 is four neighbouring lanes, whose largest
// magnitude takes two lane exchanges. The place of a row in the cache depends on its token alone: each block looks its
// few tokens up once (a wave per token counts the sequence starts at or below it, all lanes at once, since a
// binary search would wait for one load after the other) and keeps them in LDS.
// Bound by bytes where rows are many (53600 tokens of Q8_0 read back, 439 MB, in 97 us, 4.5 TB/s; 16200 of fp16 stored as Q8_0 and read back, 260 MB, in 60), by
// two dependent rounds of loads, starts and page, where they are few (4.5 us).
#include "attn_internal.hpp"
#include "moe_conv.hpp"

namespace ember_attn_impl {
namespace {

constexpr int kThreads = 256;
// Chunks of K, and as many of V, per thread: their loads are all on the way before the first is used. One where blocks are few: their
// look-ups are then all of their time.
constexpr int kManyItems = 4;

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Cache row of token i, or what place_of gives in its stead.
__device__ inline int64_t token_place(const CacheArgs& c, int i, int lane) {
  int b = i, first = i, end = i + 1, len = 0;
  if (c.q_start) {
    // 64 sequences at a time: their starts, ends and lengths at once, then the lane whose sequence it is
    int s = 0, n = 64;
    for (; s < c.n_seqs; s += 64) {
      const bool in = s + lane < c.n_seqs;
      first = in ? c.q_start[s + lane] : 0;
      end = in ? c.q_start[s + lane + 1] : INT32_MAX;
      len = in ? c.kv_len[s + lane] : 0;
      n = __popcll(__ballot(end <= i));
      if (n < 64) break;
    }
    b = s + n;
    if (b >= c.n_seqs) return kNoSeq;
    first = __builtin_amdgcn_readlane(first, n);
    end = __builtin_amdgcn_readlane(end, n);
    len = __builtin_amdgcn_readlane(len, n);
  } else {
    if (b >= c.n_seqs) return kNoSeq;
    len = c.kv_len[b];
  }
  return place_of(c, b, first, end, len, i);
}

// 8 values of type T as they lie in memory: of Q8_0 their codes.
template <int T>
struct Raw {
  uint32_t w[T == EMBER_TYPE_F32 ? 8 : T == EMBER_TYPE_Q8_0 ? 2 : 4];
};
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int T>
__device__ inline Raw<T> load8(const void* p, int64_t at) {
  Raw<T> r;
  if constexpr (T == EMBER_TYPE_Q8_0) {
    const u32x2 a = *reinterpret_cast<const u32x2*>(static_cast<const char*>(p) + at);
    r.w[0] = a[0], r.w[1] = a[1];
  } else {
    const u32x4* s = reinterpret_cast<const u32x4*>(static_cast<const char*>(p) + at * (T == EMBER_TYPE_F32 ? 4 : 2));
    for (int i = 0; i < (T == EMBER_TYPE_F32 ? 2 : 1); ++i) {
      const u32x4 a = s[i];
      for (int e = 0; e < 4; ++e) r.w[4 * i + e] = a[e];
    }
  }
  return r;
}
template <int T>
__device__ inline void save8(void* p, int64_t at, const Raw<T>& r) {
  if constexpr (T == EMBER_TYPE_Q8_0) {
    *reinterpret_cast<u32x2*>(static_cast<char*>(p) + at) = u32x2{r.w[0], r.w[1]};
  } else {
    u32x4* s = reinterpret_cast<u32x4*>(static_cast<char*>(p) + at * (T == EMBER_TYPE_F32 ? 4 : 2));
    for (int i = 0; i < (T == EMBER_TYPE_F32 ? 2 : 1); ++i) s[i] = u32x4{r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]};
  }
}
template <int T>
__device__ inline void values(const Raw<T>& r, float (&x)[8]) {
  for (int i = 0; i < 8; ++i) {
    if constexpr (T == EMBER_TYPE_F32) x[i] = __uint_as_float(r.w[i]);
    else if constexpr (T == EMBER_TYPE_Q8_0) x[i] = (float)(int8_t)(r.w[i / 4] >> (8 * (i % 4)));
    else if constexpr (T == EMBER_TYPE_BF16) x[i] = ember_moe::bf16_f32((uint16_t)(r.w[i / 2] >> (16 * (i % 2))));
    else x[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(r.w[i / 2] >> (16 * (i % 2))));
  }
}
template <int T>
__device__ inline Raw<T> raw(const float (&x)[8]) {
  Raw<T> r;
  if constexpr (T == EMBER_TYPE_F32) {
    for (int i = 0; i < 8; ++i) r.w[i] = __float_as_uint(x[i]);
  } else {
    for (int i = 0; i < 4; ++i) {
      uint32_t h[2];
      for (int e = 0; e < 2; ++e)
        h[e] = T == EMBER_TYPE_BF16 ? ember_moe::bf16_rne(x[2 * i + e]) : __builtin_bit_cast(uint16_t, (_Float16)x[2 * i + e]);
      r.w[i] = h[0] | h[1] << 16;
    }
  }
  return r;
}

// The code of x at scale d (h = d / 2, inv ~ 1 / d): the integer nearest to the exact quotient, ties to even. n is at
// most one off; x - n d is exact in f32 (d has 11 bits, n 8, and the difference is a multiple of x's last bit no larger
// than d), so comparing it with d / 2 decides.
__device__ inline int code_of(float x, float d, float h, float inv) {
  float n = rintf(x * inv);
  n = fminf(fmaxf(n, -128.0f), 128.0f);
  const float e = __builtin_fmaf(-n, d, x);
  const bool odd = ((int)n & 1) != 0;
  if (e > h || (e == h && odd)) n += 1.0f;
  if (e < -h || (e == -h && odd)) n -= 1.0f;
  return (int)fminf(fmaxf(n, -127.0f), 127.0f);
}

// The codes of 8 values. x / d is within 2^-16 of x inv here, so its nearest integer is that of x inv wherever this is over 10^-4 from the middle
// between two (as bits of 1.5 2^23 + n, whose low byte is the code: some 6 instructions a value, where code_of takes 18: 16200 tokens stored
// in 37 us, by code_of alone in 46); code_of decides the others.
__device__ __forceinline__ Raw<EMBER_TYPE_Q8_0> codes_of(const float (&x)[8], float d) {
  constexpr float kMagic = 12582912.0f;
  const float inv = 1.0f / d;
  float t[8], off = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    t[i] = __builtin_fmaf(x[i], inv, kMagic);
    off = fmaxf(off, fabsf(__builtin_fmaf(x[i], inv, kMagic - t[i])));
    t[i] = __builtin_amdgcn_fmed3f(t[i], kMagic - 127.0f, kMagic + 127.0f);
  }
  Raw<EMBER_TYPE_Q8_0> r;
  if (off < 0.4999f) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(t[4 * w + 1]), __float_as_uint(t[4 * w]), 0x0c0c0400u);
      const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(t[4 * w + 3]), __float_as_uint(t[4 * w + 2]), 0x04000c0cu);
      r.w[w] = lo | hi;
    }
  } else {
    r.w[0] = r.w[1] = 0;
    for (int i = 0; i < 8; ++i) r.w[i / 4] |= (uint32_t)(uint8_t)code_of(x[i], d, 0.5f * d, inv) << (8 * (i % 4));
  }
  return r;
}

struct Rows {
  void *k, *v;
  int64_t ks, vs;
};

// Eight values into the cache at `to`, the scale's place being `row`.
template <int C>
__device__ inline void put(void* held, _Float16* scales, int64_t to, int64_t scale_at, bool first, float (&x)[8]) {
  if constexpr (C == EMBER_TYPE_Q8_0) {
    float m = 0.0f;
    bool nan = false;
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[i])), nan |= x[i] != x[i];
    if (nan) m = __builtin_nanf("");
    for (int s = 1; s <= 2; s <<= 1) {
      const float o = __shfl_xor(m, s, 4);
      m = m != m || o != o ? __builtin_nanf("") : fmaxf(m, o);
    }
    const float q = m / 127.0f;
    const _Float16 dh = (_Float16)(q > 515.5f ? 515.5f : q);  // (NaN passes)
    const float d = (float)dh;
    Raw<C> r = {{0, 0}};
    if (d > 0.0f) r = codes_of(x, d);
    save8<C>(held, to, r);
    if (first) scales[scale_at] = dh;
  } else {
    save8<C>(held, to, raw<C>(x));
  }
}

template <int T, int C, bool STORE, int kItems>
__global__ __launch_bounds__(kThreads) void kv_rows_kernel(CacheArgs c, Rows r, FastDiv chunks, FastDiv per_head) {
  constexpr int kBlock = kThreads * kItems;
  __shared__ int64_t place[kBlock / 4 + 2];  // of the tokens that the block's chunks touch: rows have at least 4 chunks
  const int64_t total = (int64_t)c.n_tokens * chunks.d, base = (int64_t)blockIdx.x * kBlock;
  const int64_t last = min(base + kBlock, total) - 1;
  const int i0 = base < 0x7fffffff ? (int)div_by((uint32_t)base, chunks) : (int)(base / chunks.d);
  const int i1 = last < 0x7fffffff ? (int)div_by((uint32_t)last, chunks) : (int)(last / chunks.d);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = i0 + wave; i <= i1; i += kThreads / 64) {
    const int64_t p = token_place(c, i, lane);
    if (lane == 0) place[i - i0] = p;
  }
  __syncthreads();
  const uint32_t off0 = (uint32_t)(base - (int64_t)i0 * chunks.d);  // chunk of token i0 that the block begins with
  // Item u's places. (Whole rows and blocks of 32 values: the four lanes of one do the same, or nothing.)
  int64_t in_k[kItems], in_v[kItems], at[kItems], scale_at[kItems];
  bool todo[kItems], zero[kItems], first[kItems];
  constexpr int L = STORE ? T : C;  // what is loaded
  Raw<L> k[kItems], v[kItems];
  _Float16 ks[kItems], vs[kItems];
#pragma unroll
  for (int u = 0; u < kItems; ++u) {
    const uint32_t n = u * kThreads + threadIdx.x, f = off0 + n, tok = min(div_by(f, chunks), (uint32_t)(i1 - i0));
    const int64_t p = place[tok];
    const uint32_t ch = f - tok * chunks.d, head = div_by(ch, per_head), d8 = ch - head * per_head.d;
    todo[u] = base + n < total && p != kNoSeq && (!STORE || p >= 0);
    zero[u] = p < 0;
    const int64_t row = (zero[u] ? 0 : p) + (int64_t)head * c.page.d;
    in_k[u] = (int64_t)(i0 + tok) * r.ks + ch * 8;
    in_v[u] = (int64_t)(i0 + tok) * r.vs + ch * 8;
    at[u] = row * c.D + d8 * 8;
    scale_at[u] = row * (c.D / 32) + d8 / 4;
    first[u] = (d8 & 3) == 0;
    if (todo[u]) {
      k[u] = load8<L>(STORE ? r.k : c.k, STORE ? in_k[u] : at[u]);
      v[u] = load8<L>(STORE ? r.v : c.v, STORE ? in_v[u] : at[u]);
      if constexpr (!STORE && C == EMBER_TYPE_Q8_0) {
        ks[u] = c.ks[scale_at[u]];
        vs[u] = c.vs[scale_at[u]];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kItems; ++u) {
    if (!todo[u]) continue;
    float x[8], y[8];
    values<L>(k[u], x);
    values<L>(v[u], y);
    if constexpr (STORE) {
      put<C>(c.k, c.ks, at[u], scale_at[u], first[u], x);
      put<C>(c.v, c.vs, at[u], scale_at[u], first[u], y);
    } else {
      for (int i = 0; i < 8; ++i) {
        if constexpr (C == EMBER_TYPE_Q8_0) x[i] *= (float)ks[u], y[i] *= (float)vs[u];
        if (zero[u]) x[i] = y[i] = 0.0f;
      }
      save8<T>(r.k, in_k[u], raw<T>(x));
      save8<T>(r.v, in_v[u], raw<T>(y));
    }
  }
}

template <int T, bool STORE>
int launch(const CacheArgs& c, const Rows& r, hipStream_t st) {
  const uint32_t per_row = (uint32_t)(c.n_kv * c.D / 8);
  const int64_t chunks = (int64_t)c.n_tokens * per_row;
  const bool many = chunks >= (int64_t)512 * kThreads * kManyItems;
  const int64_t block = kThreads * (many ? kManyItems : 1), blocks = (chunks + block - 1) / block;
  if (blocks > kMaxBlocks) return EMBER_ERR_SHAPE;
  const FastDiv f = fast_div(per_row), h = fast_div((uint32_t)c.D / 8);
  auto go = [&](auto* kernel) { kernel<<<(unsigned)blocks, kThreads, 0, st>>>(c, r, f, h); };
  auto pick = [&](auto* few, auto* lots) { many ? go(lots) : go(few); };
  switch (c.type) {
    case EMBER_TYPE_F16: pick(kv_rows_kernel<T, EMBER_TYPE_F16, STORE, 1>, kv_rows_kernel<T, EMBER_TYPE_F16, STORE, kManyItems>); break;
    case EMBER_TYPE_BF16: pick(kv_rows_kernel<T, EMBER_TYPE_BF16, STORE, 1>, kv_rows_kernel<T, EMBER_TYPE_BF16, STORE, kManyItems>); break;
    default: pick(kv_rows_kernel<T, EMBER_TYPE_Q8_0, STORE, 1>, kv_rows_kernel<T, EMBER_TYPE_Q8_0, STORE, kManyItems>); break;
  }
  return hipGetLastError() == hipSuccess ? EMBER_OK : EMBER_ERR_LAUNCH;
}

template <bool STORE>
int launch_type(const CacheArgs& c, const Rows& r, int type, hipStream_t st) {
  switch (type) {
    case EMBER_TYPE_F32: return launch<EMBER_TYPE_F32, STORE>(c, r, st);
    case EMBER_TYPE_F16: return launch<EMBER_TYPE_F16, STORE>(c, r, st);
    default: return launch<EMBER_TYPE_BF16, STORE>(c, r, st);
  }
}

}  // namespace

int launch_kv_store(const CacheArgs& c, const void* k, int64_t ks, const void* v, int64_t vs, int type, hipStream_t st) {
  return launch_type<true>(c, Rows{const_cast<void*>(k), const_cast<void*>(v), ks, vs}, type, st);
}
int launch_kv_load(const CacheArgs& c, void* k, int64_t ks, void* v, int64_t vs, int type, hipStream_t st) {
  return launch_type<false>(c, Rows{k, v, ks, vs}, type, st);
}

}  // namespace ember_attn_impl
