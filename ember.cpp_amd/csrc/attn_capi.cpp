// C ABI of the cache and the attention (include/ember_attn.h): argument checks and launches.
#include <algorithm>

#include "attn_internal.hpp"

namespace ember_attn_impl {

namespace {
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int half_bytes(int type) { return type == EMBER_TYPE_F32 ? 4 : 2; }

int check_cache(const ember_kv_cache* c) {
  if (!c) return EMBER_ERR_NULL;
  if (c->type != EMBER_TYPE_F16 && c->type != EMBER_TYPE_BF16 && c->type != EMBER_TYPE_Q8_0) return EMBER_ERR_TYPE;
  if (c->head_dim < 32 || c->head_dim > 256 || c->head_dim % 32 || c->n_kv < 1 || c->n_kv > 256 || c->page < 1 || c->n_pages < 1)
    return EMBER_ERR_SHAPE;
  // rows of one head are numbered by 32 bits
  if ((double)c->n_pages * c->page * c->n_kv >= 4294967295.0) return EMBER_ERR_SHAPE;
  const bool q8 = c->type == EMBER_TYPE_Q8_0;
  if (!c->k || !c->v || (q8 && (!c->k_scale || !c->v_scale))) return EMBER_ERR_NULL;
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || (q8 && (!aligned(c->k_scale, 16) || !aligned(c->v_scale, 16)))) return EMBER_ERR_ALIGN;
  return EMBER_OK;
}

int check_batch(const ember_kv_cache* c, const ember_kv_batch* b) {
  if (!b) return EMBER_ERR_NULL;
  if (b->n_seqs < 0 || b->n_seqs > 65535 || b->n_tokens < 0 || b->max_q < 1 || b->max_kv < 0 || b->max_kv > (1 << 29) || b->shared < 0)
    return EMBER_ERR_SHAPE;
  if (!b->q_start && b->n_tokens < b->n_seqs) return EMBER_ERR_SHAPE;
  if (b->pages ? b->max_pages < 1 : (b->n_seqs > c->n_pages || b->shared)) return EMBER_ERR_SHAPE;
  if (b->shared % c->page || (b->pages && b->shared / c->page > b->max_pages)) return EMBER_ERR_SHAPE;
  if (b->n_seqs && !b->kv_len) return EMBER_ERR_NULL;
  if (!aligned(b->kv_len, 4) || !aligned(b->q_start, 4) || !aligned(b->pages, 4)) return EMBER_ERR_ALIGN;
  return EMBER_OK;
}

int check_rows(const void* p, int64_t stride, int width, int type) {
  if (!p) return EMBER_ERR_NULL;
  if (stride < width || stride > (int64_t)1 << 40) return EMBER_ERR_SHAPE;
  if (!aligned(p, 16) || stride * half_bytes(type) % 16) return EMBER_ERR_ALIGN;
  return EMBER_OK;
}

int check_kv_call(const ember_kv_cache* c, const ember_kv_batch* b, const void* k, int64_t ks, const void* v, int64_t vs, int type) {
  int s;
  if ((s = check_cache(c)) || (s = check_batch(c, b))) return s;
  if (type != EMBER_TYPE_F32 && type != EMBER_TYPE_F16 && type != EMBER_TYPE_BF16) return EMBER_ERR_TYPE;
  if (b->n_seqs == 0 || b->n_tokens == 0) return EMBER_OK;
  const int width = c->n_kv * c->head_dim;
  if ((s = check_rows(k, ks, width, type))) return s;
  return check_rows(v, vs, width, type);
}

int check_attn(const ember_attn_opts* a, const ember_kv_cache* c, const ember_kv_batch* b) {
  int s;
  if (!a) return EMBER_ERR_NULL;
  if ((s = check_cache(c)) || (s = check_batch(c, b))) return s;
  if (a->n_heads < 1 || a->n_heads % c->n_kv || a->n_heads / c->n_kv > 128) return EMBER_ERR_SHAPE;
  if (!(a->scale > 0.0f) || !(a->scale < 1e30f) || !(a->softcap >= 0.0f) || !(a->softcap < 1e30f) || a->window < 0) return EMBER_ERR_SHAPE;
  if (a->softcap > 0.0f && !(a->scale / a->softcap < 1e30f)) return EMBER_ERR_SHAPE;  // (a quotient that the kernels multiply by)
  if (!aligned(a->slopes, 4) || !aligned(a->prefix, 4)) return EMBER_ERR_ALIGN;
  return EMBER_OK;
}

AttnArgs attn_args(const ember_attn_opts* a, const ember_kv_cache* c, const ember_kv_batch* b) {
  AttnArgs r{};
  make_cache_args(c, b, &r.c);
  r.H = a->n_heads;
  r.G = a->n_heads / c->n_kv;
  r.scale = a->scale;
  r.softcap = a->softcap;
  r.window = a->window;
  r.slopes = a->slopes;
  r.prefix = a->prefix;
  r.shared = b->shared;
  return r;
}
}  // namespace

int make_cache_args(const ember_kv_cache* c, const ember_kv_batch* b, CacheArgs* out) {
  CacheArgs& r = *out;
  r.k = c->k;
  r.v = c->v;
  r.ks = static_cast<_Float16*>(c->k_scale);
  r.vs = static_cast<_Float16*>(c->v_scale);
  r.type = c->type;
  r.n_kv = c->n_kv;
  r.D = c->head_dim;
  r.n_pages = c->n_pages;
  r.page = fast_div((uint32_t)c->page);
  r.n_seqs = b->n_seqs;
  r.n_tokens = b->n_tokens;
  r.max_q = b->q_start ? std::min(b->max_q, std::max(b->n_tokens, 1)) : 1;
  r.max_pages = b->max_pages;
  r.cap = (int)std::min<int64_t>(b->max_kv, (int64_t)c->page * (b->pages ? b->max_pages : 1));
  r.q_start = b->q_start;
  r.kv_len = b->kv_len;
  r.pages = b->pages;
  return EMBER_OK;
}

}  // namespace ember_attn_impl

using namespace ember_attn_impl;

extern "C" {

int ember_kv_store(const ember_kv_cache* c, const ember_kv_batch* b, const void* k, int64_t k_stride, const void* v,
                   int64_t v_stride, int type, hipStream_t stream) {
  if (int s = check_kv_call(c, b, k, k_stride, v, v_stride, type)) return s;
  if (b->n_seqs == 0 || b->n_tokens == 0) return EMBER_OK;
  CacheArgs a;
  make_cache_args(c, b, &a);
  return launch_kv_store(a, k, k_stride, v, v_stride, type, stream);
}

int ember_kv_load(const ember_kv_cache* c, const ember_kv_batch* b, void* k, int64_t k_stride, void* v, int64_t v_stride,
                  int type, hipStream_t stream) {
  if (int s = check_kv_call(c, b, k, k_stride, v, v_stride, type)) return s;
  if (b->n_seqs == 0 || b->n_tokens == 0) return EMBER_OK;
  CacheArgs a;
  make_cache_args(c, b, &a);
  return launch_kv_load(a, k, k_stride, v, v_stride, type, stream);
}

size_t ember_attn_scratch_bytes(const ember_attn_opts* a, const ember_kv_cache* c, const ember_kv_batch* b) {
  if (check_attn(a, c, b) || b->n_seqs == 0 || b->n_tokens == 0) return 0;
  return attn_scratch(attn_args(a, c, b));
}

int ember_attn(const ember_attn_opts* a, const ember_kv_cache* c, const ember_kv_batch* b, const void* q, int64_t q_stride,
               void* out, int64_t out_stride, int type, void* scratch, size_t scratch_bytes, hipStream_t stream) {
  if (int s = check_attn(a, c, b)) return s;
  if (type != EMBER_TYPE_F16 && type != EMBER_TYPE_BF16) return EMBER_ERR_TYPE;
  if (c->type != EMBER_TYPE_Q8_0 && type != c->type) return EMBER_ERR_TYPE;
  if (b->n_seqs == 0 || b->n_tokens == 0) return EMBER_OK;
  const int width = a->n_heads * c->head_dim;
  if (int s = check_rows(q, q_stride, width, type)) return s;
  if (int s = check_rows(out, out_stride, width, type)) return s;
  const size_t need = ember_attn_scratch_bytes(a, c, b);
  if (need && (!scratch || scratch_bytes < need)) return EMBER_ERR_SCRATCH;
  if (need && !aligned(scratch, 256)) return EMBER_ERR_ALIGN;
  AttnArgs r = attn_args(a, c, b);
  r.q = q;
  r.out = out;
  r.q_stride = q_stride;
  r.out_stride = out_stride;
  r.type = type;
  return launch_attn(r, scratch, stream);
}

}  // extern "C"
