// Attention of a few new tokens per sequence (tiles of 16 query rows per KV head) over the cache; instantiated per cache type by
// attn_step_*.hip.
//
// Bound by the cache's bytes: every key and value is read once, for all heads that share it. A block takes one KV head of one
// sequence (and one part of its keys, where sequences are few or long: the parts are joined by attn_join_kernel), its four
// waves take tiles of 32 or 64 keys in turn, each on its own: no barrier until the waves' results are joined at the end. A tile
// passes through LDS, which K leaves as the matrix cores' A operand and V transposed: rows of halves by way of registers, loaded while
// the tile before is computed (two blocks per CU, some 100 KB of loads on the way: 131000 bf16 tokens, 537 MB, in 102 us, 5.2 TB/s,
// what a copy reaches); codes straight into LDS, which leaves registers for three blocks per CU, whose waves take turns
// (48 sequences of 6000 tokens, 627 MB, in 127 us, 4.9 TB/s; by way of registers, two blocks, 145). 16 query rows fill an operand's
// columns; with 4 heads per KV head three quarters of it are idle, which costs nothing while the loads take longer. More
// rows than 16 are tiles of their own, which read the cache again.
#pragma once
#include "attn_dev.hpp"

namespace ember_attn_impl {

constexpr int kStepThreads = 256, kStepWaves = 4;

template <int T, int DP>
struct StepLds {
  static constexpr int kKeys = DP <= 64 ? 64 : 32;
  static constexpr int kCH = DP * Op<T>::kBytes / 16;  // 16-byte chunks of a row
  static constexpr int kTileBytes = kKeys * kCH * 16;
  static constexpr int kScaleBytes = Op<T>::kQ8 ? 2 * (DP / 32) * kKeys * 2 : 0;  // of K by key, of V by block
  static constexpr int kWave = 2 * kTileBytes + kScaleBytes;
  static constexpr int kJoin = 16 * DP * 4;  // a wave's result
  static constexpr int kPerWave = kWave > kJoin ? kWave : kJoin;
  static constexpr int kBytes = kStepWaves * kPerWave;
};

// The scales of a Q8_0 row: KS of them if EXACT, otherwise nb and zeros.
template <int KS>
using RowScales __attribute__((ext_vector_type(KS))) = _Float16;
template <int KS, bool EXACT>
__device__ inline RowScales<KS> row_scales(const _Float16* p, uint32_t row, int nb) {
  row = row == ~0u ? 0 : row;
  if constexpr (EXACT) {
    return *reinterpret_cast<const RowScales<KS>*>(p + (int64_t)row * KS);
  } else {
    RowScales<KS> r;
#pragma unroll
    for (int i = 0; i < KS; ++i) r[i] = i < nb ? p[(int64_t)row * nb + i] : (_Float16)0.0f;
    return r;
  }
}

// EXACT: rows of DP columns, not fewer.
template <int T, int IO, int DP, bool GEN, bool EXACT>
__global__ __launch_bounds__(kStepThreads, DP > 128 ? (Op<T>::kQ8 ? 2 : 1) : Op<T>::kQ8 ? 3 : 2) void attn_step_kernel(AttnArgs a, Parts parts, int part0, int tiles, int chunk, int begin) {
  using O = Op<T>;
  using L = StepLds<T, DP>;
  constexpr int KT = L::kKeys, CH = L::kCH, NL = KT * CH / 64, KS = DP / 32, DT = DP / 16, NT = KT / 16;
  extern __shared__ __attribute__((aligned(256))) char lds[];
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, n16 = lane & 15;
  // (splits slowest: the last ones are empty for short sequences, and were they neighbours, whole XCDs would be: blocks go to these in turn)
  const int kvh = blockIdx.x, b = blockIdx.y, split = blockIdx.z / tiles, r0 = (blockIdx.z - split * tiles) * 16;
  int first, count;
  seq_rows(c, b, first, count);
  const int nrows = min(16, min(count, c.max_q) * a.G - r0);  // rows of this tile: r0 + n is head n % G of token n / G
  if (nrows <= 0) return;
  const int len = seq_len(c, b), total = c.q_start ? c.q_start[b + 1] - first : 1;
  const int64_t p0 = (int64_t)len - total;
  const int prefix = a.prefix ? a.prefix[b] : 0;
  // positions of the tile's first and last row, keys that any of its rows sees, and keys that all see
  const int64_t pa = p0 + r0 / a.G, pz = p0 + (r0 + nrows - 1) / a.G;
  const Span sa = visible(a, pa, len, prefix), sz = visible(a, pz, len, prefix);
  const int lo = max(visible(a, max(pa, (int64_t)0), len, prefix).lo, begin), hi = sz.hi;
  const int all_lo = sz.lo, all_hi = sa.hi;  // (none where the first row is before the first position)
  const int k0 = (lo & ~(KT - 1)) + split * chunk, k1 = min(hi, k0 + chunk);

  // the query rows as B operands: column n16, and for step s the columns of d that K's operand holds in this lane
  s8 qf[KS];
  float c_row, slope;
  Span see;
  int pos;
  {
    const int r = r0 + n16, tok = r / a.G, h = kvh * a.G + (r - tok * a.G);
    const bool ok = n16 < nrows;
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (ok ? (int64_t)(first + tok) * a.q_stride + (int64_t)h * c.D : 0);
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = O::kQ8 ? 16 * (g + 4 * (s >> 1)) + 8 * (s & 1) : 32 * s + 8 * g;
      qf[s] = s8{0, 0, 0, 0, 0, 0, 0, 0};
      if (ok && d < c.D) qf[s] = *reinterpret_cast<const s8*>(q + d);
      if constexpr (IO == EMBER_TYPE_BF16 && !O::kBf16)
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(ember_moe::bf16_f32((uint16_t)qf[s][i])));
    }
    float mul = a.scale * (GEN && a.softcap > 0.0f ? 2.0f / a.softcap : 1.0f) * kLog2e;
    if constexpr (IO == EMBER_TYPE_BF16 && !O::kBf16) {
      // bf16 queries as fp16: each row by a power of two that puts its largest value into [0.5, 1), undone in the scores; exact but
      // for values under 2^-14 of the largest, whose last bits go
      top = max_lanes32(max_lanes16(top));
      int e = 0;
      if (top > 0.0f && top <= 3.4028235e38f) (void)__builtin_frexpf(top, &e);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        h8 x;
        for (int i = 0; i < 8; ++i) x[i] = (_Float16)__builtin_ldexpf(ember_moe::bf16_f32((uint16_t)qf[s][i]), -e);
        qf[s] = __builtin_bit_cast(s8, x);
      }
      mul = fminf(__builtin_ldexpf(mul, e), 3e38f);
    }
    c_row = mul;
    see = ok ? visible(a, p0 + tok, len, prefix) : Span{0, INT32_MAX};
    pos = (int)(p0 + tok);
    slope = GEN && a.slopes && ok ? a.slopes[h] * kLog2e : 0.0f;
  }
  const float cap = GEN && a.softcap > 0.0f ? a.softcap * kLog2e : 0.0f;

  f4 o[DT];
  float m = kNoScore, l = 0.0f;
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f4{0, 0, 0, 0};

  char* const kt_ = lds + wave * L::kPerWave;
  char* const vt_ = kt_ + L::kTileBytes;
  _Float16* const vs_ = reinterpret_cast<_Float16*>(vt_ + L::kTileBytes);
  RowScales<KS>* const ks_ = reinterpret_cast<RowScales<KS>*>(vs_ + KS * KT);
  const int ch = c.D * O::kBytes / 16;  // chunks of a row (CH with columns past D, which are zero)

  // cache row (kvh's) of key kt + lane % KT, clamped into the sequence; ~0: in no page
  auto look_up = [&](int kt) -> uint32_t {
    const int j = min(kt + (lane & (KT - 1)), hi - 1);
    const int64_t r = cache_row(c, b, j);
    return r < 0 ? ~0u : (uint32_t)(r + (int64_t)kvh * c.page.d);
  };
  // a tile's rows, in order, 16 bytes a lane: halves by way of registers, since values may have to be put out; codes straight into LDS,
  // where lane l's 16 bytes come to lie at 16 l: it fetches the chunk that belongs there (k_at, v_at). Of Q8_0 the scales of key lane %
  // KT as well, in registers: what is put out there is a value's scale
  u4 kr[O::kQ8 ? 1 : NL], vr[O::kQ8 ? 1 : NL];
  RowScales<KS> ksc, vsc;
  auto row_of = [&](uint32_t rows, int key) {
    const uint32_t row = __shfl(rows, key);
    return (int64_t)(row == ~0u ? 0 : row) * c.D * O::kBytes;
  };
  auto load = [&](uint32_t rows) {
    if constexpr (!O::kQ8) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int flat = i * 64 + lane, key = flat / CH, cc = flat % CH;
        const int64_t at = row_of(rows, key) + cc * 16;
        kr[i] = vr[i] = u4{0, 0, 0, 0};
        if (EXACT || cc < ch) {
          kr[i] = *reinterpret_cast<const u4*>(static_cast<const char*>(c.k) + at);
          vr[i] = *reinterpret_cast<const u4*>(static_cast<const char*>(c.v) + at);
        }
      }
    }
  };
  // (columns past D: any codes, of scale 0)
  auto load_k = [&](uint32_t rows) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int key = (i * 64 + lane) / CH, cc = (k_at<CH>(key, lane % CH) >> 4) % CH;
      load_to_lds(static_cast<const char*>(c.k) + row_of(rows, key) + (EXACT || cc < ch ? cc : 0) * 16, kt_ + i * 1024);
    }
    ksc = row_scales<KS, EXACT>(c.ks, rows, c.D / 32);
  };
  auto load_v = [&](uint32_t rows) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int key = (i * 64 + lane) / CH, cc = (v_at<CH, true>(key, lane % CH) >> 4) % CH;
      load_to_lds(static_cast<const char*>(c.v) + row_of(rows, key) + (EXACT || cc < ch ? cc : 0) * 16, vt_ + i * 1024);
    }
    vsc = row_scales<KS, EXACT>(c.vs, rows, c.D / 32);
  };

  int kt = k0 + wave * KT;
  uint32_t rows = 0, rows_next = 0;
  if (kt < k1) {
    rows = look_up(kt);
    if constexpr (O::kQ8) {
      load_k(rows);
      load_v(rows);
    } else {
      load(rows);
    }
    rows_next = look_up(kt + kStepWaves * KT);
  }
  for (; kt < k1; kt += kStepWaves * KT) {
    // values of keys outside the rows' span count for none of them, whatever they hold: stored as zeros. So are, in a tile that
    // some rows see in part only, values that are not finite (a weight of 0 times one is NaN), and their keys are noted
    const bool inside = kt >= lo && kt + KT <= hi;
    const bool masked = kt < all_lo || kt + KT > all_hi || !inside, part = masked && pa != pz;
    const bool more = kt + kStepWaves * KT < k1;
    uint64_t odd = 0;
    const uint32_t here = rows;
    if constexpr (!O::kQ8) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int flat = i * 64 + lane, key = flat / CH, cc = flat % CH;
        *reinterpret_cast<u4*>(kt_ + k_at<CH>(key, cc)) = kr[i];
        u4 v = vr[i];
        if (!inside && (kt + key < lo || kt + key >= hi)) v = u4{0, 0, 0, 0};
        if (part && not_finite<O::kBf16>(v)) {
          v = u4{0, 0, 0, 0};
          odd |= 1ull << key;
        }
        *reinterpret_cast<u4*>(vt_ + v_at<CH, false>(key, cc)) = v;
      }
      // the next tile's loads, over this tile's registers
      if (more) {
        rows = rows_next;
        load(rows);
        rows_next = look_up(kt + 2 * kStepWaves * KT);
      }
    } else {
      wait_loads();
      if (lane < KT) {
        const bool out = kt + lane < lo || kt + lane >= hi;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          _Float16 sc = out ? (_Float16)0.0f : vsc[i];
          if (part && (__builtin_bit_cast(uint16_t, sc) & 0x7c00u) == 0x7c00u) {
            sc = (_Float16)0.0f;
            odd |= 1ull << lane;
          }
          vs_[i * KT + lane] = sc;
        }
        ks_[lane] = ksc;
      }
    }

    f4 s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int key = t * 16 + n16;
      s[t] = f4{0, 0, 0, 0};
      if constexpr (O::kQ8) {
        const RowScales<KS> k_scale = ks_[key];
#pragma unroll
        for (int u = 0; u < KS / 2; ++u) {
          const u4 w = *reinterpret_cast<const u4*>(kt_ + k_at<CH>(key, g + 4 * u));
          const _Float16 sc = g < 2 ? k_scale[2 * u] : k_scale[2 * u + 1];  // (of 16 codes of block (g + 4 u) / 2)
          const h8 sc8 = {sc, sc, sc, sc, sc, sc, sc, sc};
          s[t] = mma16<false>(codes_times(u2{w[0], w[1]}, sc8), qf[2 * u], s[t]);
          s[t] = mma16<false>(codes_times(u2{w[2], w[3]}, sc8), qf[2 * u + 1], s[t]);
        }
      } else {
#pragma unroll
        for (int u = 0; u < KS; ++u) s[t] = mma16<O::kBf16>(*reinterpret_cast<const s8*>(kt_ + k_at<CH>(key, 4 * u + g)), qf[u], s[t]);
      }
    }

    if constexpr (O::kQ8) {
      if (more) {  // the next tile's K over this one's, which has been read
        wait_lds();
        rows = rows_next;
        load_k(rows);
        rows_next = look_up(kt + 2 * kStepWaves * KT);
      }
    }

    uint64_t bad = __ballot(here == ~0u);  // keys in no page: their scores are NaN
    if constexpr (KT < 64) bad &= (1ull << KT) - 1;
    float x[NT * 4];
#pragma unroll
    for (int i = 0; i < NT * 4; ++i) x[i] = s[i >> 2][i & 3];
    auto score = [&](int i) -> float& { return x[i]; };
    auto key_of = [](int i) { return (i >> 2) * 16 + (i & 3); };  // (4 g further)
    Scores{c_row, cap, slope, GEN && a.slopes}.template operator()<NT * 4>(score, kt + g * 4 - pos, key_of);
    if (bad) {
#pragma unroll
      for (int i = 0; i < NT * 4; ++i)
        if (bad >> (key_of(i) + g * 4) & 1) x[i] = __builtin_nanf("");
    }
    if (masked) mask_scores<NT * 4>(score, max(see.lo, lo) - kt - g * 4, min(see.hi, hi) - kt - g * 4, key_of);
    float top = x[0];
#pragma unroll
    for (int i = 1; i < NT * 4; ++i) top = fmaxf(top, x[i]);
    top = max_lanes32(max_lanes16(top));
    // the maximum moves only when it is left behind by more than 2^8: weights then stay below 2^8, well inside fp16, and the
    // sums are seldom rescaled
    if (__ballot(top > m + 8.0f)) {
      const float m2 = fmaxf(m, top), al = exp2_fast(m - m2);
      m = m2;
      l *= al;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= al;
    }
#pragma unroll
    for (int i = 0; i < NT * 4; ++i) x[i] = exp2_fast(x[i] - m);
#pragma unroll
    for (int i = 0; i < NT * 4; i += 4) l += (x[i] + x[i + 1]) + (x[i + 2] + x[i + 3]);

    // by 32 keys: the weights as they lie, and V^T, columns 16 d + n16, its keys in their order
#pragma unroll
    for (int q = 0; q < KT / 32; ++q) {
      const float* const w = x + 8 * q;
      const s8 pf = __builtin_bit_cast(s8, u4{pack2<O::kBf16>(w[0], w[1]), pack2<O::kBf16>(w[2], w[3]), pack2<O::kBf16>(w[4], w[5]),
                                              pack2<O::kBf16>(w[6], w[7])});
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        s8 v;
        if constexpr (O::kQ8) {
          const int j = n16 >> 1, key = 32 * q + (j & 3) + (j >> 2) * 16 + g * 4;
          const i2 codes = __builtin_amdgcn_ds_read_tr8_b64_v2i32((EMBER_LDS(i2)*)(vt_ + v_at<CH, true>(key, d) + (n16 & 1) * 8));
          const _Float16* const at = vs_ + (d >> 1) * KT + 32 * q + g * 4;
          const u2 a0 = *reinterpret_cast<const u2*>(at), a1 = *reinterpret_cast<const u2*>(at + 16);
          v = codes_times(u2{(uint32_t)codes[0], (uint32_t)codes[1]}, __builtin_bit_cast(h8, u4{a0[0], a0[1], a1[0], a1[1]}));
        } else {
          const int key = 32 * q + g * 4 + (n16 >> 2), cc = 2 * d + ((n16 >> 1) & 1);
          const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EMBER_LDS(s4)*)(vt_ + v_at<CH, false>(key, cc) + (n16 & 1) * 8));
          const s4 z = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EMBER_LDS(s4)*)(vt_ + v_at<CH, false>(key + 16, cc) + (n16 & 1) * 8));
          v = s8{y[0], y[1], y[2], y[3], z[0], z[1], z[2], z[3]};
        }
        o[d] = mma16<O::kBf16>(v, pf, o[d]);
      }
    }
    if constexpr (O::kQ8) {
      if (more) {  // and its V
        wait_lds();
        load_v(rows);
      }
    }
    if (part && __ballot(odd != 0)) {  // a row that sees one of those keys: NaN by its sum of weights
      for (int k = 32; k; k >>= 1) odd |= __shfl_xor(odd, k);
      const int from = max(max(see.lo, lo) - kt, 0), to = min(min(see.hi, hi) - kt, KT);
      if (from < to && (odd >> from & (~0ull >> (64 - (to - from))))) l = __builtin_nanf("");
    }
  }

  // the four waves' results as one
  __shared__ float wm[kStepWaves][16], wl[kStepWaves][16];
  __syncthreads();
  l = sum_lanes32(sum_lanes16(l));
  if (g == 0) {
    wm[wave][n16] = m;
    wl[wave][n16] = l;
  }
  __syncthreads();
  float* const join = reinterpret_cast<float*>(lds + wave * L::kPerWave);
  {
    float M = wm[0][n16];
    for (int w = 1; w < kStepWaves; ++w) M = fmaxf(M, wm[w][n16]);
    const float al = exp2_fast(m - M);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      f4 x = o[d];
      x *= al;
      *reinterpret_cast<f4*>(join + n16 * DP + d * 16 + g * 4) = x;
    }
  }
  __syncthreads();
  // 4 columns of a row per thread
  for (int at = threadIdx.x; at < nrows * (DP / 4); at += kStepThreads) {
    const int r = at / (DP / 4), d = (at % (DP / 4)) * 4;
    if (d >= c.D) continue;
    float M = wm[0][r], sum = 0.0f;
    for (int w = 1; w < kStepWaves; ++w) M = fmaxf(M, wm[w][r]);
    f4 x = {0, 0, 0, 0};
    for (int w = 0; w < kStepWaves; ++w) {
      sum += wl[w][r] * exp2_fast(wm[w][r] - M);
      x += *reinterpret_cast<const f4*>(reinterpret_cast<const float*>(lds + w * L::kPerWave) + r * DP + d);
    }
    const int tok = (r0 + r) / a.G, h = kvh * a.G + (r0 + r - tok * a.G);
    if (parts.o) {
      const int64_t row = (int64_t)(part0 + split) * parts.rows + (int64_t)(first + tok) * a.H + h;
      *reinterpret_cast<f4*>(parts.o + row * c.D + d) = x;
      if (d == 0) {
        parts.ml[row * 2] = M;
        parts.ml[row * 2 + 1] = sum;
      }
    } else {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      x *= inv;
      const u2 y = {pack2<IO == EMBER_TYPE_BF16>(x[0], x[1]), pack2<IO == EMBER_TYPE_BF16>(x[2], x[3])};
      *reinterpret_cast<u2*>(static_cast<uint16_t*>(a.out) + (int64_t)(first + tok) * a.out_stride + (int64_t)h * c.D + d) = y;
    }
  }
}

template <int T, int IO, int DP>
int launch_step(const AttnArgs& a, const Parts& p, int part0, int splits, int chunk, int begin, hipStream_t st) {
  const int tiles = (a.c.max_q * a.G + 15) / 16;
  const dim3 grid(a.c.n_kv, a.c.n_seqs, splits * tiles);
  const size_t lds = StepLds<T, DP>::kBytes;
  auto go = [&](auto* kernel) {
    if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
      return (int)EMBER_ERR_LAUNCH;
    kernel<<<grid, kStepThreads, lds, st>>>(a, p, part0, tiles, chunk, begin);
    return hipGetLastError() == hipSuccess ? (int)EMBER_OK : (int)EMBER_ERR_LAUNCH;
  };
  const bool gen = a.softcap > 0.0f || a.slopes;
  if (a.c.D == DP) return gen ? go(attn_step_kernel<T, IO, DP, true, true>) : go(attn_step_kernel<T, IO, DP, false, true>);
  return gen ? go(attn_step_kernel<T, IO, DP, true, false>) : go(attn_step_kernel<T, IO, DP, false, false>);
}

template <int T, int IO>
int launch_step_type(const AttnArgs& a, const Parts& p, int part0, int splits, int chunk, int begin, hipStream_t st) {
  if (a.c.D <= 64) return launch_step<T, IO, 64>(a, p, part0, splits, chunk, begin, st);
  if (a.c.D <= 128) return launch_step<T, IO, 128>(a, p, part0, splits, chunk, begin, st);
  return launch_step<T, IO, 256>(a, p, part0, splits, chunk, begin, st);
}

}  // namespace ember_attn_impl
