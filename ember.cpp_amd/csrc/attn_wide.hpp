// Attention of many query rows over the cache: prompts, and the pages that a whole batch shares; instantiated per cache type by
// attn_wide_*.hip.
//
// Bound by the matrix cores. A block takes 128 query rows of one KV head (the heads that share it are rows too, so their keys
// are loaded once), 32 for each of its four waves, and goes through the keys in tiles that all waves read from LDS. The next tile
// comes into the other half of the LDS while this one is computed: rows of halves straight, quantised rows by way of
// registers, as fp16 (converted once for all four waves); one barrier per tile. 32 x 32 x 16 products: a lane holds half of the scores of one query row.
// A prompt of 8192 bf16 tokens, 32 heads over 8 KV heads of 128, 550 GFLOP: 610 us, 900 TFLOP/s, where a library product of 8192^3 reaches
// 1180. The matrix cores are busy in 36 % of the cycles and the vector units, which make weights of scores, in 33 %: a wave does one after the other, and
// with two blocks per CU the second wave of a SIMD fills in for it only in part.
#pragma once
#include "attn_dev.hpp"

namespace ember_attn_impl {

constexpr int kWideThreads = 256, kWideRows = 128;

template <bool BF16>
__device__ inline f16v mma32(s8 a, s8 b, f16v c) {
  if constexpr (BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

template <int DP>
struct WideLds {
  static constexpr int kKeys = DP <= 128 ? 64 : 32;  // per tile
  static constexpr int kCH = DP / 8;                 // 16-byte chunks of a row
  static constexpr int kTile = kKeys * kCH * 16;
  static constexpr int kStage = 2 * kTile;           // K and V
  static constexpr int kBytes = 2 * kStage;
};

// Asks the scheduler for N products, each fed by R reads from LDS, with the reads of AHEAD products on the way before the first: left to
// itself, short of registers, it waits for every read in turn.
template <int N, int R, int AHEAD>
__device__ __forceinline__ void lds_ahead() {
  constexpr int A = AHEAD < N ? AHEAD : N;
  __builtin_amdgcn_sched_group_barrier(0x100, A * R, 0);
#pragma unroll
  for (int i = 0; i < N - A; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x8, A, 0);
}

// The sequence of row i of the batch, n_seqs for rows of none.
__device__ inline int seq_of(const CacheArgs& c, int i) {
  if (!c.q_start) return i;
  int lo = 0, hi = c.n_seqs;  // the first b with q_start[b + 1] > i
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (c.q_start[mid + 1] > i) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// EXACT: rows of DP columns, not fewer. SHARED: the rows are those of the whole batch, the keys the first `end` of sequence 0's. Otherwise blockIdx.y is the sequence, and
// keys before `begin` are left out.
template <int T, int IO, int DP, bool GEN, bool SHARED, bool EXACT>
__global__ __launch_bounds__(kWideThreads, DP <= 128 ? 2 : 1) void attn_wide_kernel(AttnArgs a, Parts parts, int part0, int tiles, int splits,
                                                                                 int chunk, int begin, int end) {
  using O = Op<T>;
  using L = WideLds<DP>;
  constexpr int CH = L::kCH, KT = L::kKeys, NL = KT * CH / kWideThreads, KS = DP / 16, DT = DP / 32, NS = KT / 32;
  constexpr int RPI = kWideThreads / CH;  // rows of a tile that one load of all threads covers
  extern __shared__ __attribute__((aligned(256))) char lds[];
  __shared__ int bounds[4][4];
  __shared__ unsigned long long odd_keys[4];  // of tile n at n % 4: its keys whose values are not all finite
  const CacheArgs& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, n32 = lane & 31;
  // the block: KV head fastest (of 8, each stays on one XCD, whose L2 then holds its keys for all row tiles); the last rows, which
  // see the most keys, first. Where all blocks find a place at once (512), the second half in the other order, so that a CU's two are
  // a long and a short one
  int x = blockIdx.x;
  const int kvh = x % c.n_kv;
  x /= c.n_kv;
  const int split = x % splits, turn = x / splits, half_ = (tiles + 1) / 2;
  const int r0 = (gridDim.x * gridDim.y <= 512 && turn >= half_ ? turn - half_ : tiles - 1 - turn) * kWideRows;
  const int kv_seq = SHARED ? 0 : blockIdx.y;
  int first = 0, count = c.n_tokens, len = 0, prefix = 0;
  int64_t p0 = 0;
  if constexpr (!SHARED) {
    seq_rows(c, kv_seq, first, count);
    len = seq_len(c, kv_seq);
    p0 = (int64_t)len - (c.q_start ? c.q_start[kv_seq + 1] - first : 1);
    count = min(count, c.max_q);
    prefix = a.prefix ? a.prefix[kv_seq] : 0;
    if (r0 >= count * a.G) return;
  }
  // this lane's query row
  const int r = r0 + wave * 32 + n32, tok = r / a.G, h = kvh * a.G + (r - tok * a.G);
  bool ok = r < count * a.G;
  int64_t p = p0 + tok;
  if constexpr (SHARED) {
    int b = ok ? seq_of(c, tok) : c.n_seqs;
    ok = b < c.n_seqs;
    b = ok ? b : 0;
    int f, n;
    seq_rows(c, b, f, n);
    ok = ok && tok >= f && tok - f < min(n, c.max_q);
    len = seq_len(c, b);
    p = (int64_t)len - (c.q_start ? c.q_start[b + 1] - f : 1) + (tok - f);
    prefix = a.prefix ? a.prefix[b] : 0;
  }
  Span see = visible(a, p, len, prefix);
  see.lo = max(see.lo, begin);
  if constexpr (SHARED) see.hi = min(see.hi, end);
  const bool blind = !ok || see.lo >= see.hi;
  // keys that any row of the wave sees, of the block; and that all rows of the wave see
  int w_lo = blind ? INT32_MAX : see.lo, w_hi = blind ? 0 : see.hi, all_lo = ok ? see.lo : 0, all_hi = ok ? see.hi : INT32_MAX;
  for (int k = 16; k; k >>= 1) {
    w_lo = min(w_lo, __shfl_xor(w_lo, k));
    w_hi = max(w_hi, __shfl_xor(w_hi, k));
    all_lo = max(all_lo, __shfl_xor(all_lo, k));
    all_hi = min(all_hi, __shfl_xor(all_hi, k));
  }
  w_lo = __builtin_amdgcn_readfirstlane(w_lo);
  w_hi = __builtin_amdgcn_readfirstlane(w_hi);
  all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  all_hi = __builtin_amdgcn_readfirstlane(all_hi);
  if (lane == 0) {
    bounds[wave][0] = w_lo;
    bounds[wave][1] = w_hi;
    bounds[wave][2] = all_lo;
    bounds[wave][3] = all_hi;
  }
  if (tid < 4) odd_keys[tid] = 0;
  __syncthreads();
  const int lo = min(min(bounds[0][0], bounds[1][0]), min(bounds[2][0], bounds[3][0]));
  const int hi = max(max(bounds[0][1], bounds[1][1]), max(bounds[2][1], bounds[3][1]));
  const int b_lo = max(max(bounds[0][2], bounds[1][2]), max(bounds[2][2], bounds[3][2]));
  const int b_hi = min(min(bounds[0][3], bounds[1][3]), min(bounds[2][3], bounds[3][3]));
  // (lo is INT32_MAX and hi 0 where no row sees a key: no tiles)
  const int64_t k0l = hi ? (int64_t)(lo & ~(KT - 1)) + (int64_t)split * chunk : 0;
  const int k0 = (int)min(k0l, (int64_t)hi), k1 = (int)min((int64_t)hi, k0l + chunk);

  // the query row as B operand
  s8 qf[KS];
  float mul = a.scale * (GEN && a.softcap > 0.0f ? 2.0f / a.softcap : 1.0f) * kLog2e;
  {
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (ok ? (int64_t)(first + tok) * a.q_stride + (int64_t)h * c.D : 0);
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 16 * s + 8 * half;
      qf[s] = s8{0, 0, 0, 0, 0, 0, 0, 0};
      if (ok && d < c.D) qf[s] = *reinterpret_cast<const s8*>(q + d);
      if constexpr (IO == EMBER_TYPE_BF16 && !O::kBf16)
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(ember_moe::bf16_f32((uint16_t)qf[s][i])));
    }
    if constexpr (IO == EMBER_TYPE_BF16 && !O::kBf16) {
      // (as in attn_step_kernel: bf16 rows as fp16, scaled by a power of two)
      top = max_lanes32(top);
      int e = 0;
      if (top > 0.0f && top <= 3.4028235e38f) (void)__builtin_frexpf(top, &e);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        h8 y;
        for (int i = 0; i < 8; ++i) y[i] = (_Float16)__builtin_ldexpf(ember_moe::bf16_f32((uint16_t)qf[s][i]), -e);
        qf[s] = __builtin_bit_cast(s8, y);
      }
      mul = fminf(__builtin_ldexpf(mul, e), 3e38f);
    }
  }
  const Scores sc{mul, GEN && a.softcap > 0.0f ? a.softcap * kLog2e : 0.0f, GEN && a.slopes && ok ? a.slopes[h] * kLog2e : 0.0f, a.slopes != nullptr};
  const int pos = (int)p;
  if (!ok) see = {0, INT32_MAX};

  f16v o[DT];
  float m = kNoScore, l = 0.0f;
#pragma unroll
  for (int d = 0; d < DT; ++d)
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

  // Loads: row tid / CH (+ RPI i) of a tile, a chunk of 8 values: 16 bytes of halves or 8 codes. DMA: the 16 bytes at 16 tid (+ 4096 i) of the
  // stage's K and V, which hold the chunks that k_at and v_at put there.
  constexpr bool DMA = !O::kQ8 && EXACT;
  const int l_row = tid / CH, l_ch = tid % CH;
  const bool whole = !c.pages || c.page.d % KT == 0;  // a tile lies in one page
  u4 kr[DMA ? 1 : NL], vr[DMA ? 1 : NL];
  uint32_t ks_[NL], vs_[NL];  // Q8_0: the scales' bits
  uint32_t torn = 0;          // bit i: this thread's row i is in no page
  auto row_at = [&](int j) -> uint32_t {
    const int64_t rr = cache_row(c, kv_seq, j);
    return rr < 0 ? ~0u : (uint32_t)(rr + (int64_t)kvh * c.page.d);
  };
  // chunk of row `row` that is loaded for place (key, l_ch)
  auto k_chunk = [&](int key) { return DMA ? (k_at<CH>(key, l_ch) >> 4) % CH : l_ch; };
  auto v_chunk = [&](int key) { return DMA ? (v_at<CH, false>(key, l_ch) >> 4) % CH : l_ch; };
  auto load_row = [&](int i, const char* k, const char* v, int64_t k_off, int64_t v_off, int64_t s_off, int stage) {
    if constexpr (DMA) {
      char* const to = lds + stage * L::kStage + (i * kWideThreads + wave * 64) * 16;
      load_to_lds(k + k_off, to);
      load_to_lds(v + v_off, to + L::kTile);
    } else if (EXACT || l_ch * 8 < c.D) {
      if constexpr (O::kQ8) {
        const u2 kk = *reinterpret_cast<const u2*>(k + k_off), vv = *reinterpret_cast<const u2*>(v + v_off);
        kr[i] = u4{kk[0], kk[1], 0, 0};
        vr[i] = u4{vv[0], vv[1], 0, 0};
        ks_[i] = __builtin_bit_cast(uint16_t, c.ks[s_off]);
        vs_[i] = __builtin_bit_cast(uint16_t, c.vs[s_off]);
      } else {
        kr[i] = *reinterpret_cast<const u4*>(k + k_off);
        vr[i] = *reinterpret_cast<const u4*>(v + v_off);
      }
    } else {
      kr[i] = vr[i] = u4{0, 0, 0, 0};
      ks_[i] = vs_[i] = 0;
    }
  };
  auto load = [&](int kt, int stage) {
    const int64_t row_bytes = (int64_t)(EXACT ? DP : c.D) * O::kBytes;
    const int nb = (EXACT ? DP : c.D) / 32;
    const char *const ck = static_cast<const char*>(c.k), *const cv = static_cast<const char*>(c.v);
    const uint32_t base = whole ? row_at(kt) : 0;
    torn = 0;
    if (whole && kt + KT <= hi && base != ~0u) {  // the plain case: rows of one page, one after the other
      const char *const k = ck + base * row_bytes, *const v = cv + base * row_bytes;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int key = l_row + i * RPI, at = key * (int)row_bytes;
        load_row(i, k, v, at + k_chunk(key) * 8 * O::kBytes, at + v_chunk(key) * 8 * O::kBytes, (int64_t)base * nb + key * nb + l_ch / 4, stage);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int key = l_row + i * RPI, j = min(kt + key, hi - 1);
        uint32_t row = !whole ? row_at(j) : base == ~0u ? base : base + (uint32_t)(j - kt);
        if (row == ~0u) {
          torn |= 1u << i;
          row = 0;
        }
        load_row(i, ck, cv, row * row_bytes + k_chunk(key) * 8 * O::kBytes, row * row_bytes + v_chunk(key) * 8 * O::kBytes, (int64_t)row * nb + l_ch / 4, stage);
      }
    }
  };
  // Into the stage, if it is not there yet; values of keys that the block does not see as zeros. A tile that some rows see in part only
  // (`part`) must not hold values that are not finite, since a weight of 0 times one is NaN: they become zeros too, and their key is noted. A key
  // in no page becomes NaN, which makes its scores so.
  auto store = [&](int kt, int stage, bool part, unsigned long long* odd) {
    char* const kl = lds + stage * L::kStage;
    char* const vl = kl + L::kTile;
    const u4 nan = {0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu}, zero = {0, 0, 0, 0};
    if constexpr (DMA) {
      wait_loads();
      if (!part && torn == 0) return;
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int key = l_row + i * RPI;
      if constexpr (DMA) {
        char* const to = kl + (i * kWideThreads + tid) * 16;
        u4 vv = *reinterpret_cast<const u4*>(to + L::kTile);
        bool put = kt + key < lo || kt + key >= hi;
        if (!put && not_finite<O::kBf16>(vv)) {
          put = true;
          atomicOr(odd, 1ull << key);
        }
        if (put) *reinterpret_cast<u4*>(to + L::kTile) = zero;
        if (torn >> i & 1) *reinterpret_cast<u4*>(to) = nan;
      } else {
        u4 kk = kr[i], vv = vr[i];
        if constexpr (O::kQ8) {
          auto held = [](u4 w, uint32_t bits) {
            const _Float16 s_ = __builtin_bit_cast(_Float16, (uint16_t)bits);
            return __builtin_bit_cast(u4, codes_times(u2{w[0], w[1]}, h8{s_, s_, s_, s_, s_, s_, s_, s_}));
          };
          kk = held(kk, ks_[i]);
          vv = held(vv, vs_[i]);
        }
        if (part) {
          if (kt + key < lo || kt + key >= hi) vv = zero;
          if (not_finite<O::kBf16>(vv)) {
            vv = zero;
            atomicOr(odd, 1ull << key);
          }
        }
        if (torn >> i & 1) kk = nan;
        *reinterpret_cast<u4*>(kl + k_at<CH>(key, l_ch)) = kk;
        *reinterpret_cast<u4*>(vl + v_at<CH, false>(key, l_ch)) = vv;
      }
    }
  };
  auto in_part = [&](int kt) { return kt < b_lo || kt + KT > b_hi; };

  if (k0 < k1) {
    load(k0, 0);
    store(k0, 0, in_part(k0), &odd_keys[0]);
    __syncthreads();
  }
  wait_loads();  // (the query's too, on every path into the loop: else the first product of each tile waits for all loads)
  for (int kt = k0, n = 0; kt < k1; kt += KT, ++n) {
    const bool more = kt + KT < k1;
    if (more) load(kt + KT, (n + 1) & 1);
    if (tid == 0) odd_keys[(n + 2) & 3] = 0;  // (two barriers after it was read, one before it is written again)
    if (kt < w_hi && kt + KT > w_lo) {
      const char* const kl = lds + (n & 1) * L::kStage;
      const char* const vl = kl + L::kTile;
      f16v s[NS];
#pragma unroll
      for (int u = 0; u < NS; ++u) {
        for (int i = 0; i < 16; ++i) s[u][i] = 0.0f;
#pragma unroll
        for (int q = 0; q < KS; ++q) {
          const s8 kf = *reinterpret_cast<const s8*>(kl + k_at<CH>(u * 32 + n32, 2 * q + half));
          s[u] = mma32<O::kBf16>(kf, qf[q], s[u]);
        }
      }
      lds_ahead<NS * KS, 1, 6>();
      // key of score i of half-tile u: 8 (i / 4) + 4 half + i % 4
      const bool masked = kt < all_lo || kt + KT > all_hi;
      auto score = [&](int i) -> float& { return reinterpret_cast<float*>(&s[i >> 4])[i & 15]; };
      auto key_of = [](int i) { return (i >> 4) * 32 + 8 * (i >> 2 & 3) + (i & 3); };
      if (GEN) sc.template operator()<NS * 16>(score, kt + 4 * half - pos, key_of);
      if (masked) {
        mask_scores<NS * 16>(score, see.lo - kt - 4 * half, see.hi - kt - 4 * half, key_of);
        if (const uint64_t odd = odd_keys[n & 3]) {  // a row that sees one of them: NaN by its sum of weights
          const int from = max(see.lo - kt, 0), to = min(see.hi - kt, KT);
          if (from < to && (odd >> from & (~0ull >> (64 - (to - from))))) l = __builtin_nanf("");
        }
      }
      float top = s[0][0];
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
      top = max_lanes32(top);
      const float mc = GEN ? 1.0f : mul;
      top *= mc;
      if (__ballot(top > m + 8.0f)) {  // (as in attn_step_kernel)
        const float m2 = fmaxf(m, top), al = exp2_fast(m - m2);
        m = m2;
        l *= al;
#pragma unroll
        for (int d = 0; d < DT; ++d)
          for (int i = 0; i < 16; ++i) o[d][i] *= al;
      }
      s8 pf[NS * 2];
#pragma unroll
      for (int u = 0; u < NS; ++u) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = exp2_fast(__builtin_fmaf(s[u][i], mc, -m));
#pragma unroll
        for (int i = 0; i < 16; i += 4) l += (s[u][i] + s[u][i + 1]) + (s[u][i + 2] + s[u][i + 3]);
#pragma unroll
        for (int q = 0; q < 2; ++q)
          pf[u * 2 + q] = __builtin_bit_cast(s8, u4{pack2<O::kBf16>(s[u][8 * q], s[u][8 * q + 1]), pack2<O::kBf16>(s[u][8 * q + 2], s[u][8 * q + 3]),
                                                    pack2<O::kBf16>(s[u][8 * q + 4], s[u][8 * q + 5]), pack2<O::kBf16>(s[u][8 * q + 6], s[u][8 * q + 7])});
      }
      // V^T: columns 32 d + lane % 32, the keys of score order: 16 q + 4 half + 0 .. 3, and 8 further
      const int v_key = 4 * half + ((lane & 15) >> 2), v_c = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
#pragma unroll
      for (int q = 0; q < NS * 2; ++q)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EMBER_LDS(s4)*)(vl + v_at<CH, false>(16 * q + v_key, 4 * d + v_c) + (lane & 1) * 8));
          const s4 z = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EMBER_LDS(s4)*)(vl + v_at<CH, false>(16 * q + 8 + v_key, 4 * d + v_c) + (lane & 1) * 8));
          o[d] = mma32<O::kBf16>(s8{y[0], y[1], y[2], y[3], z[0], z[1], z[2], z[3]}, pf[q], o[d]);
        }
      lds_ahead<NS * 2 * DT, 2, 4>();
    }
    if (more) store(kt + KT, (n + 1) & 1, in_part(kt + KT), &odd_keys[(n + 1) & 3]);
    __syncthreads();
  }

  if (!ok) return;  // (no barrier follows)
  l = sum_lanes32(l);
  // column 32 d + 8 (i / 4) + 4 half + i % 4 of this lane's row
  if (parts.o) {
    const int64_t row = (int64_t)(part0 + split) * parts.rows + (int64_t)(first + tok) * a.H + h;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      for (int i = 0; i < 16; i += 4) {
        const int col = d * 32 + 2 * i + 4 * half;
        if (col < c.D) *reinterpret_cast<f4*>(parts.o + row * c.D + col) = f4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
      }
    if (half == 0) {
      parts.ml[row * 2] = m;
      parts.ml[row * 2 + 1] = l;
    }
  } else {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* const out = static_cast<uint16_t*>(a.out) + (int64_t)(first + tok) * a.out_stride + (int64_t)h * c.D;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      for (int i = 0; i < 16; i += 4) {
        const int col = d * 32 + 2 * i + 4 * half;
        const u2 y = {pack2<IO == EMBER_TYPE_BF16>(o[d][i] * inv, o[d][i + 1] * inv), pack2<IO == EMBER_TYPE_BF16>(o[d][i + 2] * inv, o[d][i + 3] * inv)};
        if (col < c.D) *reinterpret_cast<u2*>(out + col) = y;
      }
  }
}

template <int T, int IO, int DP, bool SHARED>
int launch_wide(const AttnArgs& a, const Parts& p, const WideCall& w, hipStream_t st) {
  const int64_t rows = (int64_t)(SHARED ? a.c.n_tokens : a.c.max_q) * a.G, tiles = (rows + kWideRows - 1) / kWideRows;
  const dim3 grid((unsigned)(tiles * w.splits * a.c.n_kv), SHARED ? 1 : a.c.n_seqs);
  constexpr size_t lds = WideLds<DP>::kBytes;
  static_assert(lds <= 65536, "no attribute needed");
  auto go = [&](auto* kernel) { kernel<<<grid, kWideThreads, lds, st>>>(a, p, w.part0, (int)tiles, w.splits, w.chunk, w.begin, w.end); };
  const bool gen = a.softcap > 0.0f || a.slopes;
  if (a.c.D == DP) gen ? go(attn_wide_kernel<T, IO, DP, true, SHARED, true>) : go(attn_wide_kernel<T, IO, DP, false, SHARED, true>);
  else gen ? go(attn_wide_kernel<T, IO, DP, true, SHARED, false>) : go(attn_wide_kernel<T, IO, DP, false, SHARED, false>);
  return hipGetLastError() == hipSuccess ? EMBER_OK : EMBER_ERR_LAUNCH;
}

template <int T, int IO>
int launch_wide_type(const AttnArgs& a, const Parts& p, const WideCall& w, hipStream_t st) {
  if (w.end) {  // the shared pages
    if (a.c.D <= 64) return launch_wide<T, IO, 64, true>(a, p, w, st);
    if (a.c.D <= 128) return launch_wide<T, IO, 128, true>(a, p, w, st);
    return launch_wide<T, IO, 256, true>(a, p, w, st);
  }
  if (a.c.D <= 64) return launch_wide<T, IO, 64, false>(a, p, w, st);
  if (a.c.D <= 128) return launch_wide<T, IO, 128, false>(a, p, w, st);
  return launch_wide<T, IO, 256, false>(a, p, w, st);
}

}  // namespace ember_attn_impl
