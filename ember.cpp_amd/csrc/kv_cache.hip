// K and V rows into and out of the paged cache (ember_kv_store, ember_kv_load).
//
// A row's values go through in chunks of 8 (one 16-byte load of halves), consecutive threads on consecutive chunks, so
// rows are read and pages written in whole 128-byte lines; a Q8_0 block of 32 is four neighbouring lanes, whose largest
// magnitude takes two lane exchanges. The place of a row in the cache depends on its token alone: each block looks its
// few tokens up once (a wave per token counts the sequence starts at or below it, all lanes at once, since a
// binary search would wait for one load after the other) and keeps them in LDS.
#include "attn_internal.hpp"
#include "moe_conv.hpp"

namespace ember_attn_impl {
namespace {

constexpr int kThreads = 256;
constexpr int kItems = 4;       // chunks per thread: the look-up is paid once for 1024 of them
constexpr int kMaxTok = 258;    // tokens that 1024 chunks touch: rows have at least 4 chunks

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int64_t kNoSeq = -1, kNoPage = -2;

// Cache row of token i (cache_row); kNoSeq: the row belongs to no sequence; kNoPage: its place is in no page.
__device__ inline int64_t token_place(const CacheArgs& c, int i, int lane) {
  int b = i;
  if (c.q_start) {
    b = 0;
    for (int s = 0; s < c.n_seqs; s += 64) {
      const bool below = s + lane < c.n_seqs && c.q_start[s + lane + 1] <= i;
      const int n = __popcll(__ballot(below));
      b += n;
      if (n < 64) break;
    }
  }
  if (b >= c.n_seqs) return kNoSeq;
  int first, count;
  seq_rows(c, b, first, count);
  // (the sequence's own count, not what n_tokens leaves of it, is what ends at its length)
  const int len = seq_len(c, b), total = c.q_start ? c.q_start[b + 1] - first : 1;
  if (i < first || i - first >= count) return kNoSeq;
  const int64_t pos = (int64_t)len - total + (i - first);
  if (pos < 0 || pos >= c.cap) return kNoPage;
  const int64_t row = cache_row(c, b, (int)pos);
  return row < 0 ? kNoPage : row;
}

template <int T>
__device__ inline void load8(const void* p, int64_t at, float (&x)[8]) {
  if constexpr (T == EMBER_TYPE_F32) {
    const f32x4* s = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
    const f32x4 a = s[0], b = s[1];
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else if constexpr (T == EMBER_TYPE_F16) {
    const h8 a = *reinterpret_cast<const h8*>(static_cast<const _Float16*>(p) + at);
    for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
  } else {
    const u16x8 a = *reinterpret_cast<const u16x8*>(static_cast<const uint16_t*>(p) + at);
    for (int i = 0; i < 8; ++i) x[i] = ember_moe::bf16_f32(a[i]);
  }
}
template <int T>
__device__ inline void save8(void* p, int64_t at, const float (&x)[8]) {
  if constexpr (T == EMBER_TYPE_F32) {
    f32x4* s = reinterpret_cast<f32x4*>(static_cast<float*>(p) + at);
    s[0] = f32x4{x[0], x[1], x[2], x[3]};
    s[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else if constexpr (T == EMBER_TYPE_F16) {
    h8 a;
    for (int i = 0; i < 8; ++i) a[i] = (_Float16)x[i];
    *reinterpret_cast<h8*>(static_cast<_Float16*>(p) + at) = a;
  } else {
    u16x8 a;
    for (int i = 0; i < 8; ++i) a[i] = ember_moe::bf16_rne(x[i]);
    *reinterpret_cast<u16x8*>(static_cast<uint16_t*>(p) + at) = a;
  }
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

struct Rows {
  void *k, *v;
  int64_t ks, vs;
};

template <int T, int C, bool STORE>
__global__ __launch_bounds__(kThreads) void kv_rows_kernel(CacheArgs c, Rows r, FastDiv chunks) {
  __shared__ int64_t place[kMaxTok];
  const int64_t total = (int64_t)c.n_tokens * chunks.d;
  const int64_t base = (int64_t)blockIdx.x * (kThreads * kItems);
  const int i0 = (int)(base / chunks.d);
  const int i1 = (int)((min(base + kThreads * kItems, total) - 1) / chunks.d);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = i0 + wave; i <= i1; i += kThreads / 64) {
    const int64_t p = token_place(c, i, lane);
    if (lane == 0) place[i - i0] = p;
  }
  __syncthreads();
  const bool is_v = blockIdx.y != 0;
  void* rows = is_v ? r.v : r.k;
  const int64_t stride = is_v ? r.vs : r.ks;
  void* held = is_v ? c.v : c.k;
  _Float16* scales = is_v ? c.vs : c.ks;
  const uint32_t off0 = (uint32_t)(base - (int64_t)i0 * chunks.d);  // chunk of token i0 that the block begins with
  const int per_head = c.D / 8;
#pragma unroll
  for (int u = 0; u < kItems; ++u) {
    const uint32_t n = u * kThreads + threadIdx.x;
    if (base + n >= total) continue;  // (whole rows, so all four lanes of a block of 32 or none)
    const uint32_t at = off0 + n, tok = div_by(at, chunks);
    const int64_t p = place[tok];
    const int ch = (int)(at - tok * chunks.d), head = ch / per_head, d8 = ch - head * per_head;
    const int64_t row = p + (int64_t)head * c.page.d;
    const int64_t in = (int64_t)(i0 + tok) * stride + ch * 8, to = row * c.D + d8 * 8;
    float x[8];
    if constexpr (STORE) {
      if (p < 0) continue;  // (the same for the four lanes)
      load8<T>(rows, in, x);
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
        const float d = (float)dh, h = 0.5f * d, inv = 1.0f / d;
        uint64_t codes = 0;
        if (d > 0.0f)
          for (int i = 0; i < 8; ++i) codes |= (uint64_t)(uint8_t)code_of(x[i], d, h, inv) << (8 * i);
        *reinterpret_cast<uint64_t*>(static_cast<int8_t*>(held) + to) = codes;
        if ((d8 & 3) == 0) scales[row * (c.D / 32) + d8 / 4] = dh;
      } else {
        save8<C>(held, to, x);
      }
    } else {
      if (p < 0) {
        if (p == kNoSeq) continue;
        for (int i = 0; i < 8; ++i) x[i] = 0.0f;
      } else if constexpr (C == EMBER_TYPE_Q8_0) {
        const uint64_t codes = *reinterpret_cast<const uint64_t*>(static_cast<const int8_t*>(held) + to);
        const float d = (float)scales[row * (c.D / 32) + d8 / 4];
        for (int i = 0; i < 8; ++i) x[i] = d * (float)(int8_t)(codes >> (8 * i));
      } else {
        load8<C>(held, to, x);
      }
      save8<T>(rows, in, x);
    }
  }
}

template <int T, bool STORE>
int launch(const CacheArgs& c, const Rows& r, hipStream_t st) {
  const uint32_t per_row = (uint32_t)(c.n_kv * c.D / 8);
  const int64_t blocks = ((int64_t)c.n_tokens * per_row + kThreads * kItems - 1) / (kThreads * kItems);
  if (blocks > 0x7fffffff) return EMBER_ERR_SHAPE;
  const dim3 grid((unsigned)blocks, 2);
  const FastDiv f = fast_div(per_row);
  switch (c.type) {
    case EMBER_TYPE_F16: kv_rows_kernel<T, EMBER_TYPE_F16, STORE><<<grid, kThreads, 0, st>>>(c, r, f); break;
    case EMBER_TYPE_BF16: kv_rows_kernel<T, EMBER_TYPE_BF16, STORE><<<grid, kThreads, 0, st>>>(c, r, f); break;
    default: kv_rows_kernel<T, EMBER_TYPE_Q8_0, STORE><<<grid, kThreads, 0, st>>>(c, r, f); break;
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
