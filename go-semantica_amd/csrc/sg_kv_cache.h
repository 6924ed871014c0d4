// sg_kv_cache.h -- how a key/value cache lies in memory.
//
// Slots are kept in tiles of 32, a key head's tiles one after another; a tile holds its
// keys, its values and a tail of 256 bytes.  Within a tile both lie as the matrix cores
// take them (16x16 products over 32 keys or dims: a lane has eight elements in a row), so
// attention moves whole kilobytes to registers or LDS and nothing is transposed:
//   keys    fragment half * (D / 32) + dim / 32, half = key / 16:
//           lane key % 16 + 16 * (dim / 8 % 4), element dim % 8
//   values  fragment dim / 16:
//           lane dim % 16 + 16 * (key / 4 % 4), element key / 16 * 4 + key % 4
// (the value's keys stand in the order in which a lane holds a key tile's scores).  A lane
// moves 16 bytes at a time: two fragments of codes, one of a 16-bit type, half a one of
// float32.  Dims up to D (64, 128 or 256) are zeros.
//
// Tail, 8 bits: 32 scales of the keys, 32 of the values.  Otherwise: one word with a bit for
// each slot whose value holds an infinity or a NaN.
#pragma once
#include "sg_packed.h"

namespace sgc {

constexpr int kTile = 32;  // slots
constexpr int kTail = 256;

__host__ __device__ constexpr int pad_dim(int hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }
__host__ __device__ constexpr int64_t tile_bytes(int D, int es) { return (int64_t)2 * kTile * D * es + kTail; }

// A kept element: codes of 8 bits, or T itself.
template <typename T, bool Q8>
struct kept {
  typedef T type;
};
template <typename T>
struct kept<T, true> {
  typedef int8_t type;
};

// Byte offset of element j of a lane's piece of a fragment, ES bytes each.
template <int ES>
__device__ __forceinline__ int place(int frag, int lane, int j) {
  if constexpr (ES == 1) return (frag >> 1) * 1024 + lane * 16 + (frag & 1) * 8 + j;
  if constexpr (ES == 2) return frag * 1024 + lane * 16 + j * 2;
  return frag * 2048 + (j >> 2) * 1024 + lane * 16 + (j & 3) * 4;
}
template <int ES>
__device__ __forceinline__ int key_at(int D, int key, int dim) {
  return place<ES>((key >> 4) * (D >> 5) + (dim >> 5), (key & 15) + ((dim >> 3) & 3) * 16, dim & 7);
}
template <int ES>
__device__ __forceinline__ int value_at(int D, int key, int dim) {
  return kTile * D * ES + place<ES>(dim >> 4, (dim & 15) + ((key >> 2) & 3) * 16, (key >> 4) * 4 + (key & 3));
}

// The places that the query at place pos sees of its prefix (x, y) and of its own keys (z, w,
// counted from the first).
__device__ __forceinline__ int4 places_seen(int64_t pos, int plen, int len, int causal, int window) {
  int64_t lo = 0, hi = (int64_t)plen + len;
  if (causal) hi = min(hi, pos + 1);
  if (window > 0) {
    lo = max(lo, pos - window + 1);
    hi = min(hi, pos + window);
  }
  auto cut = [](int64_t v, int most) { return (int)min(max(v, (int64_t)0), (int64_t)most); };
  return make_int4(cut(lo, plen), cut(hi, plen), cut(lo - plen, len), cut(hi - plen, len));
}

// An output under a maximum that has risen by so much.  An infinity is a value's that was seen, and
// stays one where the factor underflows: its key's weight is small, not zero.
__device__ __forceinline__ float faded(float o, float by) { return fabsf(o) == INFINITY ? o : o * by; }

// a / b of numbers that are not negative; short where both are (64-bit division is a hundred instructions).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

// The largest i in [0, n) with at[i] <= x, for ascending at with at[0] <= x; called by a whole
// wave with a uniform x: 64 candidates a step.
__device__ __forceinline__ int last_at_most(const int64_t* at, int n, int64_t x, int lane) {
  int lo = 0, len = n;
  while (len > 1) {
    const int step = (len + 63) >> 6, j = lane * step;
    const int c = __popcll(__ballot(j < len && at[lo + j] <= x));
    lo += (c - 1) * step;
    len = min(step, len - (c - 1) * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

}  // namespace sgc
