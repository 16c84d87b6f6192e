// The entry points of include/awq_infer.h for several requests at once: argument checks around the launchers of batch.hpp, and
// the rotary tables.
#include "batch.hpp"

#include <math.h>

static bool sixteen_bits(int32_t dtype) { return dtype == AWQ_DTYPE_BFLOAT16 || dtype == AWQ_DTYPE_FLOAT16; }
static bool aligned(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; }
static bool cache_heads(int kv_heads, int dim) { return kv_heads >= 1 && kv_heads <= 65536 && page_dim(dim); }
static bool query_heads(int heads, int kv_heads) { return heads >= 1 && heads <= 65536 && heads % kv_heads == 0; }
static bool page_count(int n_pages) { return n_pages >= 0 && n_pages < (1 << 25); }

extern "C" int64_t awq_page_bytes(int32_t kv_heads, int32_t dim) { return cache_heads(kv_heads, dim) ? kv_heads * page_head_bytes(dim) : 0; }

extern "C" int awq_page_plan(const awq_page_plan_args* a, void* stream) {
  AWQ_REQUIRE(a != nullptr, "args is NULL");
  AWQ_REQUIRE(a->n_requests >= 0 && a->max_pages >= 0 && a->max_pages < (1 << 25) && page_count(a->n_pages), "requests or pages out of range");
  AWQ_REQUIRE(a->n_requests * (64ll * a->max_pages + 1) < (1ll << 31), "too many requests and pages");
  AWQ_REQUIRE(a->max_tokens >= 0 && a->max_tokens < (1ll << 31), "max_tokens out of range");
  AWQ_REQUIRE(a->free_in && a->free_out && a->starts, "NULL pointer");
  AWQ_REQUIRE(a->n_requests == 0 || (a->cached && a->fresh && a->table && a->lengths), "NULL pointer");
  AWQ_REQUIRE(a->n_pages == 0 || a->free_pages, "NULL pointer");
  AWQ_REQUIRE(a->max_tokens == 0 || (a->positions && a->slots), "NULL pointer");
  return launch_page_plan(*a, (hipStream_t)stream);
}

extern "C" int awq_rotary_tables(const awq_rotary_spec* s, int64_t max_pos, float* cosines, float* sines) {
  AWQ_REQUIRE(s != nullptr && cosines && sines, "NULL pointer");
  const bool bands = s->kind == AWQ_ROTARY_BANDS || s->kind == AWQ_ROTARY_TURNS;
  AWQ_REQUIRE(bands || (s->kind >= AWQ_ROTARY_PLAIN && s->kind <= AWQ_ROTARY_BASE), "unknown kind");
  AWQ_REQUIRE(s->rot >= 2 && s->rot % 2 == 0 && s->rot <= 65536 && max_pos >= 0, "rot or max_pos out of range");
  AWQ_REQUIRE(s->base > 1.0 && isfinite(s->base), "base must be above 1");
  AWQ_REQUIRE(s->kind == AWQ_ROTARY_PLAIN || (s->factor >= 1.0 && isfinite(s->factor)), "factor must be at least 1");
  AWQ_REQUIRE(s->kind != AWQ_ROTARY_BASE || s->rot > 2, "one pair alone has no lowest frequency to divide");
  AWQ_REQUIRE(!bands || (s->original > 0.0 && s->slow > 0.0 && s->fast > s->slow && isfinite(s->original) && isfinite(s->fast)),
              "bands need original > 0 and 0 < slow < fast");
  const int half = s->rot / 2;
  const double base = s->kind == AWQ_ROTARY_BASE ? s->base * pow(s->factor, (double)s->rot / (s->rot - 2)) : s->base;
  const double amplitude = bands ? 0.1 * log(s->factor) + 1.0 : 1.0;
  // the index at which a frequency makes `turns` turns in `original` positions: original base^(-2 i / rot) = 2 pi turns
  const auto index_of = [&](double turns) { return s->rot * log(s->original / (2.0 * M_PI * turns)) / (2.0 * log(s->base)); };
  for (int i = 0; i < half; ++i) {
    double f = pow(base, -2.0 * i / s->rot);
    if (s->kind == AWQ_ROTARY_LINEAR) f /= s->factor;
    if (bands) {
      const double first = index_of(s->fast), last = index_of(s->slow), turns = s->original * f / (2.0 * M_PI);
      const double at = s->kind == AWQ_ROTARY_BANDS ? (i - first) / (last - first) : (s->fast - turns) / (s->fast - s->slow);
      const double share = fmin(fmax(at, 0.0), 1.0);  // of the divided frequency
      f = f * (1.0 - share) + f / s->factor * share;
    }
    for (int64_t p = 0; p < max_pos; ++p) {
      cosines[p * half + i] = (float)(amplitude * cos(f * (double)p));
      sines[p * half + i] = (float)(amplitude * sin(f * (double)p));
    }
  }
  return AWQ_OK;
}

extern "C" int awq_paged_append(const awq_paged_append_args* a, int32_t dtype, void* stream) {
  AWQ_REQUIRE(a != nullptr, "args is NULL");
  AWQ_REQUIRE(sixteen_bits(dtype), "bfloat16 or binary16 only");
  AWQ_REQUIRE(cache_heads(a->kv_heads, a->dim), "heads of 64, 128 or 256 only");
  AWQ_REQUIRE(a->n_tokens >= 0 && a->n_tokens < (1ll << 31) && a->max_pos >= 0 && a->max_pos < (1ll << 31) && page_count(a->n_pages),
              "tokens, positions or pages out of range");
  AWQ_REQUIRE(a->rot >= 0 && a->rot <= a->dim && a->rot % 16 == 0, "rot is a multiple of 16, at most dim");
  if (a->n_tokens == 0) return AWQ_OK;
  AWQ_REQUIRE(a->positions && (a->rot == 0 || (a->cosines && a->sines)), "NULL pointer");
  AWQ_REQUIRE((((uintptr_t)a->cosines | (uintptr_t)a->sines) & 15) == 0, "the tables are 16-byte aligned");
  if (a->q) {
    AWQ_REQUIRE(query_heads(a->heads, a->kv_heads), "heads is a multiple of kv_heads");
    AWQ_REQUIRE(a->q_out && aligned(a->q, a->ldq) && aligned(a->q_out, a->ldq_out), "q: 16-byte aligned rows in and out");
    AWQ_REQUIRE(a->ldq >= (int64_t)a->heads * a->dim && a->ldq_out >= (int64_t)a->heads * a->dim, "rows of q overlap");
    AWQ_REQUIRE(a->q != a->q_out || a->ldq == a->ldq_out, "in place with one stride");
  }
  if (a->k) {
    AWQ_REQUIRE(aligned(a->k, a->ldk) && a->ldk >= (int64_t)a->kv_heads * a->dim, "k: 16-byte aligned rows that do not overlap");
    AWQ_REQUIRE(!a->k_out || (aligned(a->k_out, a->ldk_out) && a->ldk_out >= (int64_t)a->kv_heads * a->dim), "k_out: 16-byte aligned rows that do not overlap");
    AWQ_REQUIRE(a->k != a->k_out || a->ldk == a->ldk_out, "in place with one stride");
  }
  if (a->cache) {
    AWQ_REQUIRE(a->k && a->v && a->slots, "an append needs k, v and slots");
    AWQ_REQUIRE(aligned(a->v, a->ldv) && a->ldv >= (int64_t)a->kv_heads * a->dim, "v: 16-byte aligned rows that do not overlap");
    AWQ_REQUIRE(aligned(a->cache, 0), "the cache is 16-byte aligned");
  }
  return launch_paged_append(*a, dtype == AWQ_DTYPE_BFLOAT16, (hipStream_t)stream);
}

extern "C" int awq_paged_rows(const awq_paged_rows_args* a, int32_t dtype, void* stream) {
  AWQ_REQUIRE(a != nullptr, "args is NULL");
  AWQ_REQUIRE(sixteen_bits(dtype), "bfloat16 or binary16 only");
  AWQ_REQUIRE(cache_heads(a->kv_heads, a->dim), "heads of 64, 128 or 256 only");
  AWQ_REQUIRE(a->n_requests >= 0 && a->max_pages >= 0 && a->max_pages < (1 << 25) && page_count(a->n_pages) && a->n_rows >= 0 && a->n_rows < (1ll << 31),
              "requests, pages or rows out of range");
  if (a->n_requests == 0 || a->n_rows == 0) return AWQ_OK;
  AWQ_REQUIRE(a->cache && a->table && a->lengths && a->starts && aligned(a->cache, 0), "NULL pointer, or a cache that is not 16-byte aligned");
  AWQ_REQUIRE(aligned(a->k, a->ldk) && aligned(a->v, a->ldv), "k and v: 16-byte aligned rows");
  AWQ_REQUIRE((!a->k || a->ldk >= (int64_t)a->kv_heads * a->dim) && (!a->v || a->ldv >= (int64_t)a->kv_heads * a->dim), "rows overlap");
  return launch_paged_rows(*a, dtype == AWQ_DTYPE_BFLOAT16, (hipStream_t)stream);
}

static bool paged_shape(int32_t n_requests, int32_t heads, int32_t kv_heads, int32_t dim, int32_t max_pages) {
  return n_requests >= 0 && max_pages >= 0 && max_pages < (1 << 25) && cache_heads(kv_heads, dim) && query_heads(heads, kv_heads) &&
         (int64_t)n_requests * max_pages < (1ll << 31) && (int64_t)n_requests * heads < (1ll << 31);
}

extern "C" int64_t awq_paged_workspace_bytes(int32_t n_requests, int32_t heads, int32_t kv_heads, int32_t dim, int32_t max_pages) {
  return paged_shape(n_requests, heads, kv_heads, dim, max_pages) ? paged_workspace_bytes(n_requests, heads, kv_heads, dim, max_pages) : 0;
}

extern "C" int awq_paged_attention(const awq_paged_attention_args* a, int32_t dtype, void* stream) {
  AWQ_REQUIRE(a != nullptr, "args is NULL");
  AWQ_REQUIRE(sixteen_bits(dtype), "bfloat16 or binary16 only");
  AWQ_REQUIRE(paged_shape(a->n_requests, a->heads, a->kv_heads, a->dim, a->max_pages) && page_count(a->n_pages),
              "heads of 64, 128 or 256, a multiple of kv_heads of them; requests and pages in range");
  AWQ_REQUIRE(isfinite(a->scale), "scale is a number");
  if (a->n_requests == 0) return AWQ_OK;
  AWQ_REQUIRE(a->q && a->ctx && a->lengths && a->workspace, "NULL pointer");
  AWQ_REQUIRE((a->cache && a->table) || a->max_pages == 0, "NULL pointer");
  AWQ_REQUIRE(aligned(a->q, a->ldq) && aligned(a->ctx, a->ldc) && aligned(a->cache, 0) && aligned(a->workspace, 0), "16-byte aligned rows, cache and workspace");
  AWQ_REQUIRE(a->ldq >= (int64_t)a->heads * a->dim && a->ldc >= (int64_t)a->heads * a->dim, "rows overlap");
  AWQ_REQUIRE(a->workspace_bytes >= paged_workspace_bytes(a->n_requests, a->heads, a->kv_heads, a->dim, a->max_pages), "the workspace is too small");
  return launch_paged_attention(*a, dtype == AWQ_DTYPE_BFLOAT16, (hipStream_t)stream);
}

extern "C" int awq_packed_attention(const awq_packed_attention_args* a, int32_t dtype, void* stream) {
  AWQ_REQUIRE(a != nullptr, "args is NULL");
  AWQ_REQUIRE(sixteen_bits(dtype), "bfloat16 or binary16 only");
  AWQ_REQUIRE(cache_heads(a->kv_heads, a->dim) && query_heads(a->heads, a->kv_heads), "heads of 64, 128 or 256, a multiple of kv_heads of them");
  AWQ_REQUIRE(a->n_requests >= 0 && a->n_tokens >= 0 && a->n_tokens < (1ll << 31) && a->n_keys >= 0 && a->n_keys < (1ll << 31), "requests or rows out of range");
  AWQ_REQUIRE(isfinite(a->scale), "scale is a number");
  AWQ_REQUIRE(a->k_starts || a->n_keys >= a->n_tokens, "keys without starts of their own have the queries'");
  if (a->n_requests == 0 || a->n_tokens == 0) return AWQ_OK;
  AWQ_REQUIRE(a->q && a->ctx && a->q_starts && ((a->k && a->v) || a->n_keys == 0), "NULL pointer");
  AWQ_REQUIRE(aligned(a->q, a->ldq) && aligned(a->k, a->ldk) && aligned(a->v, a->ldv) && aligned(a->ctx, a->ldc), "16-byte aligned rows");
  AWQ_REQUIRE(a->ldq >= (int64_t)a->heads * a->dim && a->ldc >= (int64_t)a->heads * a->dim && a->ldk >= (int64_t)a->kv_heads * a->dim &&
                  a->ldv >= (int64_t)a->kv_heads * a->dim,
              "rows overlap");
  AWQ_REQUIRE(a->ldk <= 1 << 25 && a->ldv <= 1 << 25, "rows of k and v at most 2^25 values apart");
  return launch_packed_attention(*a, dtype == AWQ_DTYPE_BFLOAT16, (hipStream_t)stream);
}

static bool sample_shape(int64_t n_rows, int64_t vocab) { return n_rows >= 0 && n_rows < (1 << 25) && vocab >= 1 && vocab <= 524288; }

extern "C" int64_t awq_sample_workspace_bytes(int64_t n_rows, int64_t vocab) {
  return sample_shape(n_rows, vocab) ? sample_workspace_bytes(n_rows, vocab) : 0;
}

extern "C" int awq_sample(const awq_sample_args* a, int32_t dtype, void* stream) {
  AWQ_REQUIRE(a != nullptr, "args is NULL");
  AWQ_REQUIRE(sixteen_bits(dtype) || dtype == AWQ_DTYPE_FLOAT32, "unknown dtype");
  AWQ_REQUIRE(sample_shape(a->n_rows, a->vocab), "rows or vocab out of range");
  if (a->n_rows == 0) return AWQ_OK;
  AWQ_REQUIRE(a->logits && a->uniform && a->ids && a->workspace, "NULL pointer");
  AWQ_REQUIRE(((uintptr_t)a->workspace & 15) == 0 && ((uintptr_t)a->logits & (dtype == AWQ_DTYPE_FLOAT32 ? 3 : 1)) == 0, "misaligned logits or workspace");
  AWQ_REQUIRE(a->ld >= a->vocab, "rows overlap");
  AWQ_REQUIRE(a->workspace_bytes >= sample_workspace_bytes(a->n_rows, a->vocab), "the workspace is too small");
  return launch_sample(*a, dtype, (hipStream_t)stream);
}
