// sg_q4.cpp -- C ABI of matrices of 4-bit weights with group scales and of their products.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <new>

#include "sg_checks.h"
#include "sg_kernels.h"

struct sg_q4_weight {
  int device = 0, out_dim = 0, in_dim = 0, group = 0;
  bool scales_f32 = false;
  uint32_t* w = nullptr;
  void* scales = nullptr;
  uint8_t* zeros = nullptr;
};

using namespace sgi;

namespace {

int check_shape(int32_t out_dim, int32_t in_dim, int32_t group) {
  if (group != 32 && group != 64 && group != 128) return fail(SG_ERR_INVALID, "group %d: 32, 64 or 128 is needed", group);
  if (out_dim <= 0 || in_dim <= 0 || in_dim % group || out_dim > (1 << 24) || in_dim > (1 << 24))
    return fail(SG_ERR_INVALID, "out_dim must be positive, in_dim whole groups of %d (up to 2^24 each)", group);
  return SG_OK;
}

// The handle and its device memory.
int make(sg_ctx* ctx, int32_t out_dim, int32_t in_dim, int32_t group, bool scales_f32, bool zeros, sg_q4_weight** out) {
  sg_q4_weight* q = new (std::nothrow) sg_q4_weight;
  if (!q) return fail(SG_ERR_NOMEM, "out of host memory");
  q->device = ctx_device(ctx);
  q->out_dim = out_dim;
  q->in_dim = in_dim;
  q->group = group;
  q->scales_f32 = scales_f32;
  const size_t blocks = (size_t)sgk::q4_blocks(out_dim, in_dim), scales = blocks * 16 * (128 / group);
  if (hipMalloc(reinterpret_cast<void**>(&q->w), blocks * 1024) != hipSuccess ||
      hipMalloc(&q->scales, scales * (scales_f32 ? 4 : 2)) != hipSuccess ||
      (zeros && hipMalloc(reinterpret_cast<void**>(&q->zeros), scales) != hipSuccess)) {
    sg_q4_weight_free(q);
    (void)hipGetLastError();
    return fail(SG_ERR_NOMEM, "hipMalloc failed (4-bit weights: %zu bytes)", blocks * 1024);
  }
  *out = q;
  return SG_OK;
}

int finish(sg_q4_weight* q, hipError_t e, hipStream_t s, sg_q4_weight** out) {
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  if (e != hipSuccess) {
    const int r = fail(SG_ERR_DEVICE, "packing 4-bit weights: %s", hipGetErrorString(e));
    sg_q4_weight_free(q);
    (void)hipGetLastError();  // reported here, and to no later call's check
    return r;
  }
  *out = q;
  return SG_OK;
}

}  // namespace

extern "C" {

int sg_q4_weight_create(sg_ctx* ctx, const uint8_t* d_codes, const void* d_scales, int32_t scale_dtype,
                        const uint8_t* d_zeros, int32_t out_dim, int32_t in_dim, int32_t group, void* stream,
                        sg_q4_weight** out) {
  if (!ctx || !d_codes || !d_scales || !out) return fail(SG_ERR_INVALID, "NULL argument");
  *out = nullptr;
  SG_TRY(check_dtype(scale_dtype));
  SG_TRY(check_shape(out_dim, in_dim, group));
  if (reinterpret_cast<uintptr_t>(d_scales) % elem_bytes(scale_dtype))
    return fail(SG_ERR_INVALID, "scales are not aligned to their elements");
  OnDevice on;
  SG_TRY(on.enter(ctx_device(ctx)));
  sg_q4_weight* q = nullptr;
  SG_TRY(make(ctx, out_dim, in_dim, group, scale_dtype != SG_F16, d_zeros != nullptr, &q));
  hipStream_t s = ctx_stream(ctx, stream);
  return finish(q, sgk::q4_pack(d_codes, d_scales, scale_dtype, d_zeros, out_dim, in_dim, group, q->w, q->scales, q->zeros, s), s,
                out);
}

int sg_q4_weight_create_q4_0(sg_ctx* ctx, const void* raw, int32_t out_dim, int32_t in_dim, sg_q4_weight** out) {
  if (!ctx || !raw || !out) return fail(SG_ERR_INVALID, "NULL argument");
  *out = nullptr;
  SG_TRY(check_shape(out_dim, in_dim, 32));
  OnDevice on;
  SG_TRY(on.enter(ctx_device(ctx)));
  sg_q4_weight* q = nullptr;
  SG_TRY(make(ctx, out_dim, in_dim, 32, false, false, &q));
  hipStream_t s = ctx_stream(ctx, nullptr);
  const size_t bytes = (size_t)out_dim * (in_dim / 32) * 18;
  uint8_t* d = nullptr;
  if (hipMalloc(reinterpret_cast<void**>(&d), bytes) != hipSuccess) {
    (void)hipGetLastError();
    sg_q4_weight_free(q);
    return fail(SG_ERR_NOMEM, "hipMalloc failed (4-bit weights: %zu bytes)", bytes);
  }
  hipError_t e = hipMemcpy(d, raw, bytes, hipMemcpyHostToDevice);
  if (e == hipSuccess) e = sgk::q4_pack_q4_0(d, out_dim, in_dim, q->w, q->scales, s);
  const int r = finish(q, e, s, out);
  (void)hipFree(d);
  return r;
}

void sg_q4_weight_free(sg_q4_weight* q) {
  if (!q) return;
  OnDevice on;
  (void)on.enter(q->device);
  if (q->w) (void)hipDeviceSynchronize();
  if (q->w) (void)hipFree(q->w);
  if (q->scales) (void)hipFree(q->scales);
  if (q->zeros) (void)hipFree(q->zeros);
  delete q;
}

int sg_matmul_q4(sg_ctx* ctx, void* dst, int64_t ldd, const sg_q4_weight* w, const void* x, int64_t ldx, int32_t dtype,
                 int32_t rows, void* stream) {
  if (!ctx || !w || (rows > 0 && (!dst || !x))) return fail(SG_ERR_INVALID, "NULL argument");
  SG_TRY(check_dtype(dtype));
  if (rows < 0 || rows > kMostRows) return fail(SG_ERR_INVALID, "rows %d out of range (0..%d)", rows, kMostRows);
  if (w->device != ctx_device(ctx)) return fail(SG_ERR_INVALID, "the weights lie on another device");
  if (rows == 0) return SG_OK;
  if (sgk::q4_threads(rows, w->out_dim) > sgk::kMostThreads)
    return fail(SG_ERR_INVALID, "%d rows of %d outputs are more than one launch takes", rows, w->out_dim);
  const Span sd{dst, ldd, rows, w->out_dim, dtype}, sx{x, ldx, rows, w->in_dim, dtype};
  SG_TRY(check_span("dst", sd));
  SG_TRY(check_pieces("x", sx));
  if (sd.overlaps(sx)) return fail(SG_ERR_INVALID, "dst overlaps x");
  OnDevice on;
  SG_TRY(on.enter(w->device));
  sg_q4_args a{};
  a.dst = dst;
  a.x = x;
  a.ldd = ldd;
  a.ldx = ldx;
  a.w = w->w;
  a.scales = w->scales;
  a.zeros = w->zeros;
  a.rows = rows;
  a.out_dim = w->out_dim;
  a.in_dim = w->in_dim;
  a.group = w->group;
  a.scales_f32 = w->scales_f32;
  SG_HIP(sgk::matmul_q4(a, dtype, ctx_stream(ctx, stream)));
  return SG_OK;
}

}  // extern "C"
