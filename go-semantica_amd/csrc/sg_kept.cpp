// sg_kept.cpp -- C ABI of the operators over kept keys and values: a cache, rows into it and
// out of it, attention of a batch that shares long prefixes.  A cache is plain memory to the
// calls, which keep no state, allocate nothing, take no lock and may be captured.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <new>

#include "sg_checks.h"
#include "sg_kernels.h"
#include "sg_kv_cache.h"

struct sg_kv_cache {
  int device = 0, dtype = 0, heads = 0, hd = 0, D = 0;
  bool q8 = false;
  int32_t slots = 0;
  int64_t tile_bytes = 0, head_bytes = 0;
  char* data = nullptr;
};

using namespace sgi;

namespace {

int rows_call(sg_ctx* ctx, const sg_kv_cache* c, void* k, int64_t ldk, void* v, int64_t ldv, int32_t rows,
              const int32_t* d_off, int32_t n_seq, const int32_t* d_starts, void* stream, bool write) {
  if (!ctx || !c || !d_starts || (rows > 0 && (!k || !v))) return fail(SG_ERR_INVALID, "NULL argument");
  SG_TRY(check_batch(d_off, rows, n_seq));
  if (c->device != ctx_device(ctx)) return fail(SG_ERR_INVALID, "the cache lies on another device");
  if (rows == 0) return SG_OK;
  if (sgk::kv_rows_threads(rows, c->heads, c->dtype, c->q8) > sgk::kMostThreads)
    return fail(SG_ERR_INVALID, "%d rows of %d heads are more than one launch takes", rows, c->heads);
  const int cols = c->heads * c->hd;
  const Span sk{k, ldk, rows, cols, c->dtype}, sv{v, ldv, rows, cols, c->dtype};
  SG_TRY(check_pieces("k", sk));
  SG_TRY(check_pieces("v", sv));
  if (!write && sk.overlaps(sv)) return fail(SG_ERR_INVALID, "k overlaps v");
  OnDevice on;
  SG_TRY(on.enter(c->device));
  sg_kv_rows_args a{};
  a.cache = c->data;
  a.head_bytes = c->head_bytes;
  a.tile_bytes = c->tile_bytes;
  a.slots = c->slots;
  a.k = k;
  a.v = v;
  a.ldk = ldk;
  a.ldv = ldv;
  a.off = d_off;
  a.starts = d_starts;
  a.rows = rows;
  a.n_seq = n_seq;
  a.heads = c->heads;
  a.hd = c->hd;
  a.D = c->D;
  hipStream_t s = ctx_stream(ctx, stream);
  SG_HIP(write ? sgk::kv_write(a, c->dtype, c->q8, s) : sgk::kv_read(a, c->dtype, c->q8, s));
  return SG_OK;
}

}  // namespace

extern "C" {

int sg_kv_cache_create(sg_ctx* ctx, int32_t slots, int32_t n_kv_heads, int32_t head_dim, int32_t dtype, int32_t bits,
                       void* stream, sg_kv_cache** out) {
  if (!ctx || !out) return fail(SG_ERR_INVALID, "NULL argument");
  *out = nullptr;
  SG_TRY(check_dtype(dtype));
  if (bits != 0 && bits != 8) return fail(SG_ERR_INVALID, "bits %d: 8, or 0 for the type itself, are kept", bits);
  if (slots <= 0 || slots > kMostRows) return fail(SG_ERR_INVALID, "slots %d out of range (1..%d)", slots, kMostRows);
  if (n_kv_heads <= 0 || n_kv_heads > 65535) return fail(SG_ERR_INVALID, "%d key heads", n_kv_heads);
  if (head_dim <= 0 || head_dim > 256 || head_dim % 8)
    return fail(SG_ERR_INVALID, "head_dim %d: a multiple of 8 up to 256 is needed", head_dim);
  const int D = sgc::pad_dim(head_dim);
  const int64_t tile = sgc::tile_bytes(D, bits == 8 ? 1 : elem_bytes(dtype));
  const int64_t head = ((int64_t)slots + sgc::kTile - 1) / sgc::kTile * tile;
  OnDevice on;
  SG_TRY(on.enter(ctx_device(ctx)));
  sg_kv_cache* c = new (std::nothrow) sg_kv_cache;
  if (!c) return fail(SG_ERR_NOMEM, "out of host memory");
  c->device = ctx_device(ctx);
  c->dtype = dtype;
  c->heads = n_kv_heads;
  c->hd = head_dim;
  c->D = D;
  c->q8 = bits == 8;
  c->slots = slots;
  c->tile_bytes = tile;
  c->head_bytes = head;
  const size_t bytes = (size_t)head * n_kv_heads;
  hipStream_t s = ctx_stream(ctx, stream);
  int r = SG_OK;
  if (hipMalloc(reinterpret_cast<void**>(&c->data), bytes) != hipSuccess) {
    c->data = nullptr;
    r = fail(SG_ERR_NOMEM, "hipMalloc failed (cache: %zu bytes)", bytes);
  } else {
    // Zeros: dims of padding stay so, and a slot that was never written reads as zeros.
    hipError_t e = hipMemsetAsync(c->data, 0, bytes, s);
    if (e == hipSuccess) e = hipStreamSynchronize(s);
    if (e != hipSuccess) r = fail(SG_ERR_DEVICE, "clearing the cache: %s", hipGetErrorString(e));
  }
  if (r != SG_OK) {
    sg_kv_cache_free(c);
    (void)hipGetLastError();  // reported here, and to no later call's check
    return r;
  }
  *out = c;
  return SG_OK;
}

void sg_kv_cache_free(sg_kv_cache* c) {
  if (!c) return;
  OnDevice on;
  (void)on.enter(c->device);
  if (c->data) {
    (void)hipDeviceSynchronize();
    (void)hipFree(c->data);
  }
  delete c;
}

int sg_kv_cache_bytes(const sg_kv_cache* c, size_t* bytes) {
  if (!c || !bytes) return fail(SG_ERR_INVALID, "NULL argument");
  *bytes = (size_t)c->head_bytes * c->heads;
  return SG_OK;
}

int sg_kv_cache_write(sg_ctx* ctx, sg_kv_cache* cache, const void* k, int64_t ldk, const void* v, int64_t ldv,
                      int32_t rows, const int32_t* d_off, int32_t n_seq, const int32_t* d_starts, void* stream) {
  return rows_call(ctx, cache, const_cast<void*>(k), ldk, const_cast<void*>(v), ldv, rows, d_off, n_seq, d_starts, stream, true);
}

int sg_kv_cache_read(sg_ctx* ctx, const sg_kv_cache* cache, void* k, int64_t ldk, void* v, int64_t ldv, int32_t rows,
                     const int32_t* d_off, int32_t n_seq, const int32_t* d_starts, void* stream) {
  return rows_call(ctx, cache, k, ldk, v, ldv, rows, d_off, n_seq, d_starts, stream, false);
}

static int check_attention(const sg_kv_cache* c, int32_t n_heads, int32_t rows, int32_t n_seq, int32_t n_prefix) {
  if (n_heads <= 0 || n_heads % c->heads || n_heads > 65535)
    return fail(SG_ERR_INVALID, "%d query heads over %d key heads", n_heads, c->heads);
  if (rows < 0 || rows > kMostRows) return fail(SG_ERR_INVALID, "rows %d out of range (0..%d)", rows, kMostRows);
  if (n_seq < 0 || n_seq > (1 << 30) || n_prefix < 0 || n_prefix > (1 << 30))
    return fail(SG_ERR_INVALID, "n_seq %d, n_prefix %d out of range (0..2^30)", n_seq, n_prefix);
  if ((int64_t)rows * n_heads > (int64_t(1) << 25)) return fail(SG_ERR_INVALID, "%d rows of %d heads are more than 2^25", rows, n_heads);
  return SG_OK;
}

int sg_attention_shared_work_bytes(const sg_kv_cache* cache, int32_t n_heads, int32_t rows, int32_t n_seq,
                                   int32_t n_prefix, size_t* bytes) {
  if (!cache || !bytes) return fail(SG_ERR_INVALID, "NULL argument");
  SG_TRY(check_attention(cache, n_heads, rows, n_seq, n_prefix));
  *bytes = sgk::attn_shared_work_bytes(cache->dtype, cache->q8, rows, n_heads, cache->heads, cache->D, n_seq, n_prefix);
  return SG_OK;
}

int sg_attention_shared(sg_ctx* ctx, void* out, int64_t ldo, const void* q, int64_t ldq, const sg_kv_cache* cache,
                        int32_t n_heads, int32_t rows, const int32_t* d_off, int32_t n_seq, const sg_shared_keys* keys,
                        void* work, size_t work_bytes, void* stream) {
  if (!ctx || !cache || !keys || (rows > 0 && (!out || !q))) return fail(SG_ERR_INVALID, "NULL argument");
  if (!keys->starts || !keys->lengths) return fail(SG_ERR_INVALID, "starts and lengths are needed");
  SG_TRY(check_batch(d_off, rows, n_seq));
  SG_TRY(check_attention(cache, n_heads, rows, n_seq, keys->n_prefix));
  if (keys->n_prefix > 0 && (!keys->shared || !keys->prefix_starts || !keys->prefix_lengths))
    return fail(SG_ERR_INVALID, "prefixes need shared, prefix_starts and prefix_lengths");
  if (cache->device != ctx_device(ctx)) return fail(SG_ERR_INVALID, "the cache lies on another device");
  const float scale = keys->scale != 0.0f ? keys->scale : 1.0f / std::sqrt((float)cache->hd), cap = keys->softcap;
  // (So that products of them are numbers.)
  if (!(std::fabs(scale) >= 1e-15f && std::fabs(scale) <= 1e15f) || !(cap == 0.0f || (cap >= 1e-15f && cap <= 1e15f)))
    return fail(SG_ERR_INVALID, "scale and softcap must be 0 or within 1e-15 .. 1e15, softcap not negative");
  if (keys->window < 0) return fail(SG_ERR_INVALID, "window < 0");
  if (rows == 0) return SG_OK;
  const int cols = n_heads * cache->hd;
  const Span so{out, ldo, rows, cols, cache->dtype}, sq{q, ldq, rows, cols, cache->dtype};
  SG_TRY(check_pieces("out", so));
  SG_TRY(check_pieces("q", sq));
  if (so.overlaps(sq)) return fail(SG_ERR_INVALID, "out overlaps q");
  const size_t need = sgk::attn_shared_work_bytes(cache->dtype, cache->q8, rows, n_heads, cache->heads, cache->D, n_seq, keys->n_prefix);
  if (!work || work_bytes < need || reinterpret_cast<uintptr_t>(work) % 16)
    return fail(SG_ERR_INVALID, "work: %zu bytes, 16-byte aligned, are needed (%zu given)", need, work ? work_bytes : 0);
  const uintptr_t w0 = reinterpret_cast<uintptr_t>(work), w1 = w0 + need;
  for (const Span* t : {&so, &sq})
    if (w0 < t->hi() && t->lo() < w1) return fail(SG_ERR_INVALID, "work overlaps out or q");
  OnDevice on;
  SG_TRY(on.enter(cache->device));
  constexpr float kLog2e = 1.44269504088896340736f;
  sg_attn_shared_args a{};
  a.out = out;
  a.q = q;
  a.cache = cache->data;
  a.ldo = ldo;
  a.ldq = ldq;
  a.head_bytes = cache->head_bytes;
  a.tile_bytes = cache->tile_bytes;
  a.scale = cap != 0.0f ? 1.0f : std::fabs(scale) * kLog2e;
  a.cap = cap * kLog2e;
  a.to_cap = cap != 0.0f ? std::fabs(scale) / cap : 0.0f;
  a.negative = scale < 0.0f;
  a.causal = keys->causal != 0;
  a.window = keys->window;
  a.rows = rows;
  a.heads = n_heads;
  a.kv_heads = cache->heads;
  a.group = n_heads / cache->heads;
  a.hd = cache->hd;
  sg_attn_batch b{};
  b.off = d_off;
  b.starts = keys->starts;
  b.lengths = keys->lengths;
  b.shared = keys->shared;
  b.prefix_starts = keys->prefix_starts;
  b.prefix_lengths = keys->prefix_lengths;
  b.slots = cache->slots;
  b.n_seq = n_seq;
  b.n_prefix = keys->n_prefix;
  SG_HIP(sgk::attn_shared(a, b, cache->dtype, cache->q8, cache->D, work, ctx_stream(ctx, stream)));
  return SG_OK;
}

}  // extern "C"
