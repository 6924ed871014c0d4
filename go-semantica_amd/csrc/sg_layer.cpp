// sg_layer.cpp -- C ABI of the operators over device-resident offsets: masked
// attention, block norms, request adapters.  They keep no state in the context and
// allocate nothing, so they take no lock and may be captured into a graph.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>

#include "sg_internal.h"
#include "sg_kernels.h"

struct sg_adapter_bank {
  int device = 0, dtype = 0, n = 0, rank_pad = 0, in_dim = 0, out_dim = 0;
  void *a = nullptr, *b = nullptr;
  float* scales = nullptr;
};

namespace {

using sgi::fail;

// The context's device for the duration of a call, the caller's afterwards.
struct OnDevice {
  int before = -1;
  int enter(int device) {
    SG_HIP(hipGetDevice(&before));
    if (before == device) {
      before = -1;
      return SG_OK;
    }
    SG_HIP(hipSetDevice(device));
    return SG_OK;
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

constexpr int32_t kMostRows = INT32_MAX - (1 << 16);  // a row index and a tile's length beyond it fit 32 bits

int elem_bytes(int dtype) { return dtype == SG_F32 ? 4 : 2; }

int check_dtype(int dtype) {
  if (dtype != SG_F32 && dtype != SG_F16 && dtype != SG_BF16) return fail(SG_ERR_INVALID, "unknown element type %d", dtype);
  return SG_OK;
}

// [rows][cols] at p with a row stride of ld elements.
struct Span {
  const void* p;
  int64_t ld;
  int rows, cols, dtype;
  uintptr_t lo() const { return reinterpret_cast<uintptr_t>(p); }
  uintptr_t hi() const { return lo() + ((uintptr_t)(rows - 1) * ld + cols) * elem_bytes(dtype); }
  bool overlaps(const Span& o) const {
    if (lo() >= o.hi() || o.lo() >= hi()) return false;
    const uintptr_t step = (uintptr_t)ld * elem_bytes(dtype);
    if (ld != o.ld || dtype != o.dtype || step == 0) return true;
    // Columns of one wide tensor: where o's rows begin within (or before) this one's.
    const uintptr_t at = o.lo() >= lo() ? (o.lo() - lo()) % step : (step - (lo() - o.lo()) % step) % step;
    return at < (uintptr_t)cols * elem_bytes(dtype) || at + (uintptr_t)o.cols * elem_bytes(dtype) > step;
  }
  bool same(const Span& o) const { return p == o.p && ld == o.ld; }
};

// Whole elements, and a stride that holds a row and whose tensor stays within the address space.
int check_span(const char* name, const Span& t) {
  if (t.lo() % elem_bytes(t.dtype)) return fail(SG_ERR_INVALID, "%s is not aligned to its elements", name);
  if (t.ld < t.cols || t.ld > (int64_t(1) << 28))
    return fail(SG_ERR_INVALID, "%s: row stride %lld for rows of %d", name, (long long)t.ld, t.cols);
  return SG_OK;
}
int check_pieces(const char* name, const Span& t) {
  SG_TRY(check_span(name, t));
  if (t.lo() % 16 || t.ld * elem_bytes(t.dtype) % 16)
    return fail(SG_ERR_INVALID, "%s must be 16-byte aligned, its row stride whole 16 bytes", name);
  return SG_OK;
}

int check_batch(const int32_t* d_off, int rows, int n_seq) {
  if (rows < 0 || rows > kMostRows) return fail(SG_ERR_INVALID, "rows %d out of range (0..%d)", rows, kMostRows);
  if (!d_off || n_seq <= 0) return fail(SG_ERR_INVALID, "seq_offsets must describe at least one sequence");
  if (n_seq > (1 << 30)) return fail(SG_ERR_INVALID, "n_seq %d above 2^30", n_seq);
  return SG_OK;
}

}  // namespace

extern "C" {

int sg_attention_masked(sg_ctx* ctx, void* out, int64_t ldo, const void* q, int64_t ldq, const void* k, int64_t ldk,
                        const void* v, int64_t ldv, int32_t dtype, int32_t n_heads, int32_t n_kv_heads,
                        int32_t head_dim, int32_t rows, const int32_t* d_off, int32_t n_seq, const sg_attn_mask* mask,
                        void* stream) {
  if (!ctx || (rows > 0 && (!out || !q || !k || !v))) return fail(SG_ERR_INVALID, "NULL argument");
  SG_TRY(check_dtype(dtype));
  if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || n_heads > 65535)
    return fail(SG_ERR_INVALID, "%d query heads over %d key heads", n_heads, n_kv_heads);
  if (head_dim <= 0 || head_dim > 256 || head_dim % 8)
    return fail(SG_ERR_INVALID, "head_dim %d: a multiple of 8 up to 256 is needed", head_dim);
  SG_TRY(check_batch(d_off, rows, n_seq));
  static const sg_attn_mask kPlain{};
  const sg_attn_mask& m = mask ? *mask : kPlain;
  if (!std::isfinite(m.scale) || !std::isfinite(m.softcap) || m.softcap < 0)
    return fail(SG_ERR_INVALID, "scale must be finite, softcap finite and not negative");
  if (m.window < 0) return fail(SG_ERR_INVALID, "window < 0");
  if (m.prefix && !m.causal) return fail(SG_ERR_INVALID, "a prefix needs causal");
  if (rows == 0) return SG_OK;
  if ((int64_t)n_heads * head_dim > INT32_MAX) return fail(SG_ERR_INVALID, "rows of more than 2^31 elements");
  if (sgk::attention_masked_threads(dtype, rows, n_heads) > sgk::kMostThreads)
    return fail(SG_ERR_INVALID, "%d rows of %d heads are more than one launch takes", rows, n_heads);
  const int qd = n_heads * head_dim, kd = n_kv_heads * head_dim;
  const Span so{out, ldo, rows, qd, dtype}, sq{q, ldq, rows, qd, dtype}, sk{k, ldk, rows, kd, dtype},
      sv{v, ldv, rows, kd, dtype};
  SG_TRY(check_pieces("out", so));
  SG_TRY(check_pieces("q", sq));
  SG_TRY(check_pieces("k", sk));
  SG_TRY(check_pieces("v", sv));
  // A tile of keys is addressed with 32 bits from its first row.
  if (ldk > (1 << 22) || ldv > (1 << 22)) return fail(SG_ERR_INVALID, "k and v: row stride above 2^22");
  if (so.overlaps(sq) || so.overlaps(sk) || so.overlaps(sv)) return fail(SG_ERR_INVALID, "out overlaps q, k or v");
  OnDevice on;
  SG_TRY(on.enter(sgi::ctx_device(ctx)));
  sg_attn_masked_args a{};
  a.out = out;
  a.q = q;
  a.k = k;
  a.v = v;
  a.ldo = ldo;
  a.ldq = ldq;
  a.ldk = ldk;
  a.ldv = ldv;
  a.off = d_off;
  a.slopes = m.slopes;
  a.docs = m.doc_ids;
  a.prefix = m.prefix;
  a.scale = m.scale != 0.0f ? m.scale : 1.0f / std::sqrt((float)head_dim);
  a.softcap = m.softcap;
  a.rows = rows;
  a.n_seq = n_seq;
  a.heads = n_heads;
  a.kv_heads = n_kv_heads;
  a.hd = head_dim;
  a.causal = m.causal != 0;
  a.window = m.window;
  SG_HIP(sgk::attention_masked(a, dtype, sgi::ctx_stream(ctx, stream)));
  return SG_OK;
}

int sg_block_norm(sg_ctx* ctx, void* xn, int64_t ldxn, void* sum, int64_t lds, const void* x, int64_t ldx,
                  const void* h, int64_t ldh, int32_t dtype, int32_t rows, int32_t cols, const float* w_post,
                  const float* w_pre, float eps, const float* gate, float scale, const int32_t* d_off, int32_t n_seq,
                  void* stream) {
  if (!ctx || (rows > 0 && (!sum || !x || !h))) return fail(SG_ERR_INVALID, "NULL argument");
  SG_TRY(check_dtype(dtype));
  if (xn && !w_pre) return fail(SG_ERR_INVALID, "xn needs w_pre");
  if (!xn && w_pre && rows > 0) return fail(SG_ERR_INVALID, "w_pre needs xn");
  if (cols <= 0 || cols > sgk::kBlockNormCols)
    return fail(SG_ERR_INVALID, "cols %d out of range (1..%d)", cols, sgk::kBlockNormCols);
  if (!(eps >= 0.0f) || !std::isfinite(eps) || !std::isfinite(scale))
    return fail(SG_ERR_INVALID, "eps must be finite and not negative, scale finite");
  if (rows < 0 || rows > kMostRows) return fail(SG_ERR_INVALID, "rows %d out of range (0..%d)", rows, kMostRows);
  if (d_off) SG_TRY(check_batch(d_off, rows, n_seq));
  if (!d_off && n_seq != 0) return fail(SG_ERR_INVALID, "n_seq %d without seq_offsets", n_seq);
  if (rows == 0) return SG_OK;
  const Span ss{sum, lds, rows, cols, dtype}, sx{x, ldx, rows, cols, dtype}, sh{h, ldh, rows, cols, dtype},
      sn{xn, ldxn, rows, cols, dtype};
  SG_TRY(check_span("sum", ss));
  SG_TRY(check_span("x", sx));
  SG_TRY(check_span("h", sh));
  if (xn) SG_TRY(check_span("xn", sn));
  auto clash = [](const Span& o, const Span& i) { return o.overlaps(i) && !o.same(i); };
  if (clash(ss, sx) || clash(ss, sh) || (xn && (clash(sn, sx) || clash(sn, sh) || sn.overlaps(ss))))
    return fail(SG_ERR_INVALID, "an output overlaps another tensor");
  OnDevice on;
  SG_TRY(on.enter(sgi::ctx_device(ctx)));
  sg_block_norm_args a{};
  a.xn = xn;
  a.sum = sum;
  a.x = x;
  a.h = h;
  a.ldxn = ldxn;
  a.lds = lds;
  a.ldx = ldx;
  a.ldh = ldh;
  a.w_post = w_post;
  a.w_pre = w_pre;
  a.gate = gate;
  a.off = d_off;
  a.eps = eps;
  a.scale = scale;
  a.rows = rows;
  a.cols = cols;
  a.n_seq = n_seq;
  SG_HIP(sgk::block_norm(a, dtype, sgi::ctx_stream(ctx, stream)));
  return SG_OK;
}

int sg_adapter_bank_create(sg_ctx* ctx, const void* d_a, const void* d_b, const float* d_scales, int32_t dtype,
                           int32_t n_adapters, int32_t rank, int32_t in_dim, int32_t out_dim, void* stream,
                           sg_adapter_bank** out) {
  if (!ctx || !d_a || !d_b || !d_scales || !out) return fail(SG_ERR_INVALID, "NULL argument");
  *out = nullptr;
  SG_TRY(check_dtype(dtype));
  if (n_adapters <= 0) return fail(SG_ERR_INVALID, "n_adapters must be positive");
  if (rank <= 0 || rank > sgk::kAdapterMaxRank)
    return fail(SG_ERR_INVALID, "rank %d out of range (1..%d)", rank, sgk::kAdapterMaxRank);
  if (in_dim <= 0 || in_dim % 8 || out_dim <= 0 || out_dim % 8 || in_dim > (1 << 24) || out_dim > (1 << 24))
    return fail(SG_ERR_INVALID, "in_dim and out_dim must be positive multiples of 8 (up to 2^24)");
  // (Ahead of the sizes, which would leave 64 bits.)
  if ((double)n_adapters * sgk::adapters_rank_pad(rank) * std::max(in_dim, out_dim) > 0x1p48)
    return fail(SG_ERR_INVALID, "%d adapters: too many for one bank", n_adapters);
  const size_t na = sgk::adapters_a_bytes(dtype, n_adapters, rank, in_dim);
  const size_t nb = sgk::adapters_b_bytes(dtype, n_adapters, rank, out_dim);
  OnDevice on;
  SG_TRY(on.enter(sgi::ctx_device(ctx)));
  sg_adapter_bank* b = new (std::nothrow) sg_adapter_bank;
  if (!b) return fail(SG_ERR_NOMEM, "out of host memory");
  b->device = sgi::ctx_device(ctx);
  b->dtype = dtype;
  b->n = n_adapters;
  b->rank_pad = sgk::adapters_rank_pad(rank);
  b->in_dim = in_dim;
  b->out_dim = out_dim;
  hipStream_t s = sgi::ctx_stream(ctx, stream);
  int r = SG_OK;
  if (hipMalloc(&b->a, na) != hipSuccess || hipMalloc(&b->b, nb) != hipSuccess ||
      hipMalloc(&b->scales, sizeof(float) * (size_t)n_adapters) != hipSuccess)
    r = fail(SG_ERR_NOMEM, "hipMalloc failed (adapters: %zu bytes)", na + nb);
  if (r == SG_OK) {
    hipError_t e = sgk::adapters_pack(dtype, d_a, d_b, n_adapters, rank, in_dim, out_dim, b->a, b->b, s);
    if (e == hipSuccess)
      e = hipMemcpyAsync(b->scales, d_scales, sizeof(float) * (size_t)n_adapters, hipMemcpyDeviceToDevice, s);
    if (e == hipSuccess) e = hipStreamSynchronize(s);
    if (e != hipSuccess) r = fail(SG_ERR_DEVICE, "packing the adapters: %s", hipGetErrorString(e));
  }
  if (r != SG_OK) {
    sg_adapter_bank_free(b);
    (void)hipGetLastError();  // reported here, and to no later call's check
    return r;
  }
  *out = b;
  return SG_OK;
}

void sg_adapter_bank_free(sg_adapter_bank* b) {
  if (!b) return;
  OnDevice on;
  (void)on.enter(b->device);
  (void)hipDeviceSynchronize();
  if (b->a) (void)hipFree(b->a);
  if (b->b) (void)hipFree(b->b);
  if (b->scales) (void)hipFree(b->scales);
  delete b;
}

int sg_adapters_work_bytes(const sg_adapter_bank* bank, int32_t rows, size_t* bytes) {
  if (!bank || !bytes) return fail(SG_ERR_INVALID, "NULL argument");
  if (rows < 0 || rows > kMostRows) return fail(SG_ERR_INVALID, "rows %d out of range (0..%d)", rows, kMostRows);
  *bytes = sgk::adapters_work_bytes(bank->dtype, rows, bank->in_dim, bank->rank_pad);
  return SG_OK;
}

int sg_adapters_apply(sg_ctx* ctx, void* dst, int64_t ldd, const void* base, int64_t ldb, const sg_adapter_bank* bank,
                      const void* x, int64_t ldx, int32_t rows, const int32_t* d_off, int32_t n_seq,
                      const int32_t* d_adapter_ids, void* work, size_t work_bytes, void* stream) {
  if (!ctx || !bank || !d_adapter_ids || (rows > 0 && (!dst || !base || !x))) return fail(SG_ERR_INVALID, "NULL argument");
  SG_TRY(check_batch(d_off, rows, n_seq));
  if (bank->device != sgi::ctx_device(ctx)) return fail(SG_ERR_INVALID, "the adapters lie on another device");
  if (rows == 0) return SG_OK;
  if (sgk::adapters_threads(rows, bank->out_dim, bank->rank_pad) > sgk::kMostThreads)
    return fail(SG_ERR_INVALID, "%d rows of %d columns are more than one launch takes", rows, bank->out_dim);
  const Span sd{dst, ldd, rows, bank->out_dim, bank->dtype}, sb{base, ldb, rows, bank->out_dim, bank->dtype},
      sx{x, ldx, rows, bank->in_dim, bank->dtype};
  SG_TRY(check_pieces("dst", sd));
  SG_TRY(check_pieces("base", sb));
  SG_TRY(check_pieces("x", sx));
  if (sd.overlaps(sx) || (sd.overlaps(sb) && !sd.same(sb))) return fail(SG_ERR_INVALID, "dst overlaps x or base");
  const size_t need = sgk::adapters_work_bytes(bank->dtype, rows, bank->in_dim, bank->rank_pad);
  if (!work || work_bytes < need || reinterpret_cast<uintptr_t>(work) % 16)
    return fail(SG_ERR_INVALID, "work: %zu bytes, 16-byte aligned, are needed (%zu given)", need, work ? work_bytes : 0);
  const uintptr_t w0 = reinterpret_cast<uintptr_t>(work), w1 = w0 + need;
  for (const Span* t : {&sd, &sb, &sx})
    if (w0 < t->hi() && t->lo() < w1) return fail(SG_ERR_INVALID, "work overlaps dst, base or x");
  OnDevice on;
  SG_TRY(on.enter(sgi::ctx_device(ctx)));
  sg_adapters_args a{};
  a.dst = dst;
  a.base = base;
  a.x = x;
  a.ldd = ldd;
  a.ldb = ldb;
  a.ldx = ldx;
  a.wa = bank->a;
  a.wb = bank->b;
  a.scales = bank->scales;
  a.off = d_off;
  a.ids = d_adapter_ids;
  a.u = static_cast<float*>(work);
  a.rows = rows;
  a.n_seq = n_seq;
  a.n_adapters = bank->n;
  a.in_dim = bank->in_dim;
  a.out_dim = bank->out_dim;
  a.rank_pad = bank->rank_pad;
  SG_HIP(sgk::adapters_apply(a, bank->dtype, sgi::ctx_stream(ctx, stream)));
  return SG_OK;
}

}  // extern "C"
