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

__device__ __forceinline__ float wave_sum(float a) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) a += __shfl_xor(a, o);
  return a;
}

}  // namespace sgp
