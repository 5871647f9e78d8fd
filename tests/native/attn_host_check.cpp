// Checks on the CPU what keeps the cache and attention kernels inside their buffers: the place of a token whatever the device arrays
// hold, and that an attention plan's parts cover every key within the scratch that is asked for. Prints "ok" and the cases, or the case that failed.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../ember.cpp_amd/csrc/attn_internal.hpp"

using namespace ember_attn_impl;

static long cases = 0;
#define CHECK(ok, ...)                   \
  do {                                   \
    ++cases;                             \
    if (!(ok)) {                         \
      std::printf("line %d: ", __LINE__); \
      std::printf(__VA_ARGS__);          \
      std::printf("\n");                 \
      return 1;                          \
    }                                    \
  } while (0)

int main() {
  std::mt19937_64 rng(7);
  auto upto = [&](int64_t lo, int64_t hi) { return lo + (int64_t)(rng() % (uint64_t)(hi - lo + 1)); };
  auto spread = [&](int64_t hi) { return upto(0, std::max<int64_t>(1, hi >> upto(0, 30))); };  // small ones as often as large ones

  // quotients: next to multiples, and anywhere below 2^31
  for (uint32_t d : {1u, 2u, 3u, 5u, 7u, 12u, 16u, 48u, 100u, 127u, 128u, 129u, 1000u, 8192u, 65535u, 65537u, (1u << 29) - 1, 1u << 29, (1u << 30) + 1, 0x7fffffffu}) {
    const FastDiv f = fast_div(d);
    for (int i = 0; i < 3000; ++i) {
      const int64_t m = (int64_t)d * (spread(0x7fffffff) / d);
      for (int64_t n : {m - 1, m, m + 1, (int64_t)spread(0x7fffffff), (int64_t)0x7fffffff - i})
        if (n >= 0 && n < (1ll << 31)) CHECK(div_by((uint32_t)n, f) == n / d, "%lld / %u", (long long)n, d);
    }
  }

  // places: page ids, starts and lengths of any value
  for (int run = 0; run < 4000; ++run) {
    ember_kv_cache kc{};
    kc.type = EMBER_TYPE_F16, kc.n_kv = (int)upto(1, 8), kc.head_dim = 64, kc.page = (int)(1 + spread(5000)), kc.n_pages = (int)upto(1, 12);
    ember_kv_batch kb{};
    const bool paged = rng() % 3 != 0;
    kb.n_seqs = (int)upto(1, paged ? 6 : std::min(6, kc.n_pages));
    kb.max_pages = (int)upto(1, 5), kb.n_tokens = (int)upto(1, 40), kb.max_q = (int)upto(1, 50), kb.max_kv = (int)spread(kc.page * 6);
    auto any = [&](int64_t hi) { return (int32_t)(rng() % 4 ? upto(-2, hi) : (int64_t)(int32_t)rng()); };
    std::vector<int32_t> starts(kb.n_seqs + 1), lens(kb.n_seqs), table(kb.n_seqs * kb.max_pages);
    for (auto& x : starts) x = any(kb.n_tokens + 2);
    for (auto& x : lens) x = any((int64_t)kc.page * 6);
    for (auto& x : table) x = any(kc.n_pages + 1);
    kb.q_start = rng() % 4 ? starts.data() : nullptr, kb.kv_len = lens.data(), kb.pages = paged ? table.data() : nullptr;
    CacheArgs c{};
    make_cache_args(&kc, &kb, &c);
    CHECK(c.cap <= kb.max_kv && c.cap <= (int64_t)kc.page * (paged ? kb.max_pages : 1) && c.max_q >= 1, "cap %d max_q %d", c.cap, c.max_q);
    for (int b = 0; b < kb.n_seqs; ++b) {
      int first, count;
      if (kb.q_start || b < kb.n_tokens) {
        seq_rows(c, b, first, count);
        CHECK(count == 0 || (count > 0 && first >= 0 && (int64_t)first + count <= kb.n_tokens), "rows %d + %d of %d", first, count, kb.n_tokens);
      }
      CHECK(length(c, lens[b]) >= 0 && length(c, lens[b]) <= c.cap, "length %d", lens[b]);
      for (int t = 0; t < 20; ++t) {
        const int i = any(kb.n_tokens + 3), f = kb.q_start ? starts[b] : i, e = kb.q_start ? starts[b + 1] : i + (i < 0x7fffffff);
        const int64_t p = place_of(c, b, f, e, lens[b], i);
        if (p < 0) {
          CHECK(p == kNoSeq || p == kNoPage, "place %lld", (long long)p);
          continue;
        }
        // by the definition
        const int64_t pos = (int64_t)std::max(0, std::min(lens[b], c.cap)) - ((int64_t)e - f) + (i - f);
        const int64_t pid = paged ? table[b * kb.max_pages + pos / kc.page] : b;
        CHECK(i >= 0 && i < kb.n_tokens && f >= 0 && i >= f && pos >= 0 && pos < c.cap && pos / kc.page < (paged ? kb.max_pages : 1), "token %d at %lld", i, (long long)pos);
        CHECK(pid >= 0 && pid < kc.n_pages && p == pid * kc.n_kv * kc.page + pos % kc.page, "token %d: row %lld", i, (long long)p);
      }
    }
  }

  // plans
  for (int run = 0; run < 200000; ++run) {
    ember_kv_cache kc{};
    const int types[3] = {EMBER_TYPE_F16, EMBER_TYPE_BF16, EMBER_TYPE_Q8_0};
    kc.type = types[rng() % 3], kc.n_kv = 1 << upto(0, 8), kc.head_dim = 32 * (int)upto(1, 8), kc.page = (int)(1 + spread(1000));
    kc.n_pages = 100;
    ember_kv_batch kb{};
    int32_t dummy = 0;
    kb.n_seqs = (int)(1 + spread(65534)), kb.n_tokens = (int)(kb.n_seqs + spread(1 << 22)), kb.max_q = (int)(1 + spread(1 << 22));
    kb.max_kv = (int)spread(1 << 29), kb.pages = &dummy, kb.kv_len = &dummy, kb.q_start = rng() % 2 ? &dummy : nullptr;
    kb.max_pages = (int)(1 + spread((1 << 29) / kc.page));
    kb.shared = rng() % 2 ? kc.page * (int)upto(0, kb.max_pages) : 0;
    AttnArgs a{};
    make_cache_args(&kc, &kb, &a.c);
    a.G = (int)upto(1, 128), a.H = a.G * kc.n_kv, a.window = rng() % 2 ? (int)spread(0x7fffffff) : 0, a.prefix = rng() % 3 ? nullptr : &dummy, a.shared = kb.shared;
    const AttnPlan p = attn_plan(a);
    CHECK(p.splits >= 1 && p.splits <= 256 && p.shared_splits >= 0 && p.shared_splits <= 256 && p.chunk > 0, "splits %d %d", p.splits, p.shared_splits);
    CHECK(p.begin >= 0 && p.begin <= a.c.cap && (p.begin > 0) == (p.shared_splits > 0), "begin %d", p.begin);
    // the keys that the rows of a sequence can see, from wherever they begin in a tile on, and the shared ones
    int64_t keys = a.c.cap - p.begin;
    if (a.window && !a.prefix) keys = std::min<int64_t>(keys, (int64_t)a.window + a.c.max_q - 1);
    CHECK((int64_t)p.splits * p.chunk >= keys + (a.window ? 63 : 0) || (int64_t)p.splits * p.chunk >= a.c.cap - p.begin + 63, "%d parts of %d for %lld keys", p.splits, p.chunk, (long long)keys);
    CHECK((int64_t)p.splits * p.chunk < (1ll << 31) && p.chunk % 64 == 0, "parts of %d", p.chunk);
    if (p.begin) CHECK((int64_t)p.shared_splits * p.shared_chunk >= p.begin && p.shared_chunk % 64 == 0, "shared parts");
    CHECK(p.parts == (p.splits + p.shared_splits > 1 ? p.splits + p.shared_splits : 0), "parts %d", p.parts);
    CHECK(attn_scratch(a) == (size_t)p.parts * a.c.n_tokens * a.H * (a.c.D + 2) * 4, "scratch");
    CHECK(p.step == ((int64_t)a.c.max_q * a.G <= 64), "step");
  }
  std::printf("ok %ld\n", cases);
  return 0;
}
