// sg_packed.h -- device helpers of the operators that read a packed batch's CSR
// offsets from device memory, and their element types.
#pragma once
#include "sg_device.h"

namespace sgp {

// bf16 as its bits; float, _Float16 and bf16_t are the operators' element types.
struct bf16_t {
  uint16_t u;
};
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

template <typename T>
struct elem;
template <>
struct elem<float> {
  static constexpr int vec = 4;  // elements of 16 bytes
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <>
struct elem<_Float16> {
  static constexpr int vec = 8;
  static __device__ __forceinline__ float to(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 from(float v) { return (_Float16)v; }
};
template <>
struct elem<bf16_t> {
  static constexpr int vec = 8;
  static __device__ __forceinline__ float to(bf16_t v) { return __uint_as_float((uint32_t)v.u << 16); }
  static __device__ __forceinline__ bf16_t from(float v) { return bf16_t{__builtin_bit_cast(uint16_t, (__bf16)v)}; }
};

// 16 bytes of T.
template <typename T>
struct alignas(16) chunk {
  T v[elem<T>::vec];
};

// A launch that answers for itself: hipGetLastError would report what an earlier call of the
// thread left behind, and a launch that fails leaves nothing for the next caller's check.
template <typename T>
struct as_is {
  typedef T type;
};
template <typename... P>
hipError_t run_kernel(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t s, typename as_is<P>::type... p) {
  void* at[] = {&p...};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, at, lds, s);
  if (e != hipSuccess) (void)hipGetLastError();
  return e;
}

// Offsets come from device memory, so no host check has seen them: whatever
// they hold, an index formed from one is clamped to the tensors' rows.
__device__ __forceinline__ int clamp_row(int v, int rows) { return min(max(v, 0), rows); }

// The largest i in [0, n) with off[i] <= row (the sequence that holds the row,
// unless the row is behind it; empty sequences are passed over), -1 if there is
// none.  Called by a whole wave with a uniform row: 64 candidates a step, so
// 4096 sequences take two dependent loads where a lane's bisection takes twelve.
__device__ __forceinline__ int find_seq(const int32_t* __restrict__ off, int n, int row, int lane) {
  int lo = 0, len = n;
  while (true) {
    const int step = (len + 63) >> 6;
    const int64_t at = (int64_t)lane * step;
    const bool le = at < len && off[lo + (int)at] <= row;
    const int c = __popcll(__ballot(le));
    if (c == 0) return -1;  // only in the first step of ascending offsets
    lo += (c - 1) * step;
    len = min(step, len - (c - 1) * step);
    if (step <= 1) return __builtin_amdgcn_readfirstlane(lo);
  }
}

// The sequence of each lane's row, the wave's rows being row0 .. last: an index in
// [0, n) and its offsets, whatever the offsets hold; a row of no sequence gets one
// that does not contain it.  A step narrows both ends 64-fold, and one more load
// serves all lanes unless 63 sequences or more share the rows: the dependent loads
// are what this costs (a lane's own bisection of 256 offsets is eight of them).
__device__ __forceinline__ void row_seq(const int32_t* __restrict__ off, int n, int row0, int last, int row, int lane,
                                        int& seq, int& s0, int& s1) {
  int i0 = 0, i1 = 0, span = n;  // row0's is in [i0, i0 + span), last's in [i1, i1 + span)
  while (span >= SG_WAVE) {
    const int step = (span + 63) >> 6, at = lane * step;
    const bool le0 = at < span && i0 + at < n && off[min(i0 + at, n)] <= row0;
    const bool le1 = at < span && i1 + at < n && off[min(i1 + at, n)] <= last;
    i0 += max((int)__popcll(__ballot(le0)) - 1, 0) * step;
    i1 += max((int)__popcll(__ballot(le1)) - 1, 0) * step;
    span = step;
  }
  const int count = max(min(n - i0, i1 - i0 + span), 1);  // candidates from i0 on
  if (count < SG_WAVE) {
    const int o = off[min(i0 + lane, n)];
    int lo = max((int)__popcll(__ballot(lane < count && o <= row0)) - 1, 0);
    int hi = max((int)__popcll(__ballot(lane < count && o <= last)) - 1, lo);
    while (__ballot(lo < hi)) {
      const int mid = lo + (hi - lo + 1) / 2;
      const int v = __shfl(o, mid);
      if (lo < hi) {
        if (v <= row) lo = mid;
        else hi = mid - 1;
      }
    }
    s0 = __shfl(o, lo);
    s1 = __shfl(o, lo + 1);
    seq = i0 + lo;
    return;
  }
  int hi = i0 + count - 1;
  seq = i0;
  while (seq < hi) {
    const int mid = seq + (hi - seq + 1) / 2;
    if (off[mid] <= row) seq = mid;
    else hi = mid - 1;
  }
  s0 = off[seq];
  s1 = off[seq + 1];
}

__device__ __forceinline__ float wave_sum(float a) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) a += __shfl_xor(a, o);
  return a;
}

}  // namespace sgp
