// sg_checks.h -- what the operators over device-resident offsets check of their arguments.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sg_internal.h"

namespace sgi {

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

inline int elem_bytes(int dtype) { return dtype == SG_F32 ? 4 : 2; }

inline int check_dtype(int dtype) {
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
inline int check_span(const char* name, const Span& t) {
  if (t.lo() % elem_bytes(t.dtype)) return fail(SG_ERR_INVALID, "%s is not aligned to its elements", name);
  if (t.ld < t.cols || t.ld > (int64_t(1) << 28))
    return fail(SG_ERR_INVALID, "%s: row stride %lld for rows of %d", name, (long long)t.ld, t.cols);
  return SG_OK;
}
inline int check_pieces(const char* name, const Span& t) {
  SG_TRY(check_span(name, t));
  if (t.lo() % 16 || t.ld * elem_bytes(t.dtype) % 16)
    return fail(SG_ERR_INVALID, "%s must be 16-byte aligned, its row stride whole 16 bytes", name);
  return SG_OK;
}

inline int check_batch(const int32_t* d_off, int rows, int n_seq) {
  if (rows < 0 || rows > kMostRows) return fail(SG_ERR_INVALID, "rows %d out of range (0..%d)", rows, kMostRows);
  if (!d_off || n_seq <= 0) return fail(SG_ERR_INVALID, "seq_offsets must describe at least one sequence");
  if (n_seq > (1 << 30)) return fail(SG_ERR_INVALID, "n_seq %d above 2^30", n_seq);
  return SG_OK;
}

}  // namespace sgi
