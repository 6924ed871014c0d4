// k_kv_cache.hip -- rows of keys and values into a cache and back out of it
// (sg_kv_cache_write, sg_kv_cache_read):
//   scale = max(fl32(max |x| / 127), 2^-126) over a row's head;  code = the integer nearest
//   to x / scale, halves to even;  x' = fl32(code * scale), rounded to the type
// or, without codes, the values as they are.
//
// A code is exact: q = rint(x / scale) is formed with a reciprocal and put right by the
// residual x - q scale, which fmaf gives without rounding (|q| < 2^8; x is a multiple of
// half a scale's last place where |q| >= 1/2, and then |x - q scale| <= scale, 25 bits that
// end there).
//
// A workgroup takes R rows of the packed batch and one head: 256 / R lanes a row.  Keys go
// to the cache as they were loaded, eight dims of a slot together; values cross LDS, for a
// cache's lane holds one dim of four slots in a row: four rows that fill such a run are
// stored as one, others element by element.
//
// Two sequences may name the same slots: the later one's rows are kept, whole (each
// workgroup looks at the sequences behind its own).
#include <algorithm>

#include "semantica_gpu.h"
#include "sg_kernels.h"
#include "sg_kv_cache.h"

namespace {

using sgc::kTile;
using sgp::chunk;
using sgp::elem;

constexpr int kThreads = 256;

// The code of x for a scale and its reciprocal.
__device__ __forceinline__ float code_of(float x, float scale, float inv) {
  float q = __builtin_rintf(x * inv);
  const float r = __builtin_fmaf(-q, scale, x), half = 0.5f * scale;
  // (half is exact: a scale is no subnormal.  A tie goes to the even code.)
  const bool odd = ((int)q & 1) != 0;
  if (r > half || (r == half && odd)) q += 1.0f;
  if (r < -half || (r == -half && odd)) q -= 1.0f;
  return fminf(fmaxf(q, -127.0f), 127.0f);
}

// The slot of each of the workgroup's rows, in LDS: kNone for a slot outside the cache (or, on
// the way in, one that a later sequence of the call fills as well), kNoRow for a row of no sequence.
constexpr int kNone = -1, kNoRow = -2;

template <int R, bool WRITE>
__device__ __forceinline__ void row_slots(const sg_kv_rows_args& a, int row0, volatile int32_t* slot) {
  __shared__ int32_t span[3];
  const int t = threadIdx.x, lane = t & 63;
  if (t < 64) {
    const int last = min(row0 + R, a.rows) - 1, row = row0 + lane % R;
    int i, s0, s1;
    sgp::row_seq(a.off, a.n_seq, row0, last, min(row, last), lane, i, s0, s1);
    const bool there = row <= last && row >= s0 && row < s1;
    const int start = a.starts[i];
    const int64_t s = (int64_t)start + (row - s0);
    const bool in = there && start >= 0 && s < a.slots;
    if (lane < R) slot[lane] = in ? (int)s : there ? kNone : kNoRow;
    if constexpr (WRITE) {
      // The slots that the rows span, and their first sequence.
      int lo = in ? (int)s : INT32_MAX, hi = in ? (int)s : -1, first = in ? i : INT32_MAX;
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) {
        lo = min(lo, __shfl_xor(lo, o));
        hi = max(hi, __shfl_xor(hi, o));
        first = min(first, __shfl_xor(first, o));
      }
      if (lane == 0) {
        span[0] = lo;
        span[1] = hi;
        span[2] = first;
      }
    }
  }
  __syncthreads();
  if constexpr (WRITE) {
    const int lo = span[0], hi = span[1];
    if (hi < 0) return;  // (alike for all threads)
    for (int j = span[2] + 1 + t; j < a.n_seq; j += kThreads) {
      const int64_t b = a.starts[j];
      const int r0 = sgp::clamp_row(a.off[j], a.rows), r1 = sgp::clamp_row(a.off[j + 1], a.rows);
      if (b < 0 || r1 <= r0 || b > hi || b + (r1 - r0) <= lo) continue;
      for (int r = 0; r < R && row0 + r < r0; r++) {  // rows of sequences before j
        const int s = slot[r];
        if (s >= b && s < b + (r1 - r0)) slot[r] = kNone;
      }
    }
    __syncthreads();
  }
}

// Row r's part in its run of four slots: 4: its rows fill the run and r is the first, 0: r is
// another of them, 1: r stands for itself.
template <int R>
__device__ __forceinline__ int run_of(const volatile int32_t* slot, int r) {
  const int s = slot[r], o = s & 3, f = r - o;
  if (f < 0 || f + 3 >= R) return 1;
  bool whole = true;
#pragma unroll
  for (int q = 0; q < 4; q++) whole &= slot[f + q] == s - o + q;
  return whole ? (o == 0 ? 4 : 0) : 1;
}

// N elements of 1, 2 or 4 bytes as one store.
template <typename E, int N>
struct alignas(sizeof(E) * N) pack {
  E v[N];
};

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
constexpr uint32_t kInf = 0x7f800000u;

template <typename T, bool Q8, int R>
__global__ __launch_bounds__(kThreads) void k_kv_write(sg_kv_rows_args a) {
  typedef typename sgc::kept<T, Q8>::type E;
  constexpr int ES = sizeof(E), VEC = elem<T>::vec, LPR = kThreads / R, NP = (256 / VEC + LPR - 1) / LPR;
  __shared__ int32_t slot[R];
  __shared__ alignas(16) E vl[R * 256];
  const int t = threadIdx.x, r = t / LPR, l = t % LPR, h = blockIdx.y, row0 = (int)blockIdx.x * R;
  const int row = min(row0 + r, a.rows - 1), pieces = a.hd / VEC;
  chunk<T> k[NP], v[NP];
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int at = l + i * LPR;
    if (at < pieces) {
      k[i] = *reinterpret_cast<const chunk<T>*>(static_cast<const T*>(a.k) + row * a.ldk + (int64_t)h * a.hd + at * VEC);
      v[i] = *reinterpret_cast<const chunk<T>*>(static_cast<const T*>(a.v) + row * a.ldv + (int64_t)h * a.hd + at * VEC);
    }
  }
  row_slots<R, true>(a, row0, slot);
  const int s = slot[r];
  char* tile = a.cache + (int64_t)h * a.head_bytes + (int64_t)(max(s, 0) / kTile) * a.tile_bytes;
  const int key = max(s, 0) % kTile;
  // The largest magnitudes as bits: a NaN's are above an infinity's.
  uint32_t km = 0, vm = 0;
#pragma unroll
  for (int i = 0; i < NP; i++)
    if (l + i * LPR < pieces)
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        km = max(km, magnitude(elem<T>::to(k[i].v[j])));
        vm = max(vm, magnitude(elem<T>::to(v[i].v[j])));
      }
#pragma unroll
  for (int o = LPR / 2; o >= 1; o >>= 1) {
    km = max(km, (uint32_t)__shfl_xor((int)km, o));
    vm = max(vm, (uint32_t)__shfl_xor((int)vm, o));
  }
  float ks = 0, vs = 0, ki = 0, vi = 0;
  if constexpr (Q8) {
    ks = km < kInf ? fmaxf(__uint_as_float(km) / 127.0f, 0x1p-126f) : __uint_as_float(0x7fc00000u);
    vs = vm < kInf ? fmaxf(__uint_as_float(vm) / 127.0f, 0x1p-126f) : __uint_as_float(0x7fc00000u);
    ki = 1.0f / ks;
    vi = 1.0f / vs;
  }
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int dim = (l + i * LPR) * VEC;
    if (dim >= a.hd) continue;
    pack<E, VEC> kp, vp;
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      if constexpr (Q8) {
        kp.v[j] = km < kInf ? (E)(int)code_of(elem<T>::to(k[i].v[j]), ks, ki) : (E)0;
        vp.v[j] = vm < kInf ? (E)(int)code_of(elem<T>::to(v[i].v[j]), vs, vi) : (E)0;
      } else {
        kp.v[j] = k[i].v[j];
        vp.v[j] = v[i].v[j];
      }
    }
    *reinterpret_cast<pack<E, VEC>*>(vl + r * 256 + dim) = vp;
    if (s >= 0) *reinterpret_cast<pack<E, VEC>*>(tile + sgc::key_at<ES>(a.D, key, dim)) = kp;
  }
  if (l == 0 && s >= 0) {
    char* tail = tile + a.tile_bytes - sgc::kTail;
    if constexpr (Q8) {
      reinterpret_cast<float*>(tail)[key] = ks;
      reinterpret_cast<float*>(tail)[kTile + key] = vs;
    } else {
      // No other row of the call owns this bit; the others of the word come and go.
      uint32_t* word = reinterpret_cast<uint32_t*>(tail);
      const uint32_t bit = 1u << key;
      const bool set = (__hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & bit) != 0;
      if (vm >= kInf && !set) atomicOr(word, bit);
      if (vm < kInf && set) atomicAnd(word, ~bit);
    }
  }
  __syncthreads();
  for (int q = t >> 6; q < R; q += kThreads / 64) {
    const int p = slot[q];
    const int n = p >= 0 ? run_of<R>(slot, q) : 0;
    if (n == 0) continue;
    char* base = a.cache + (int64_t)h * a.head_bytes + (int64_t)(p / kTile) * a.tile_bytes;
    for (int dim = t & 63; dim < a.hd; dim += 64) {
      char* at = base + sgc::value_at<ES>(a.D, p % kTile, dim);
      if (n == 4) {
        pack<E, 4> x;
#pragma unroll
        for (int j = 0; j < 4; j++) x.v[j] = vl[(q + j) * 256 + dim];
        *reinterpret_cast<pack<E, 4>*>(at) = x;
      } else {
        *reinterpret_cast<E*>(at) = vl[q * 256 + dim];
      }
    }
  }
}

template <typename T, bool Q8, int R>
__global__ __launch_bounds__(kThreads) void k_kv_read(sg_kv_rows_args a) {
  typedef typename sgc::kept<T, Q8>::type E;
  constexpr int ES = sizeof(E), VEC = elem<T>::vec, LPR = kThreads / R, NP = (256 / VEC + LPR - 1) / LPR;
  __shared__ int32_t slot[R];
  __shared__ alignas(16) E vl[R * 256];
  const int t = threadIdx.x, r = t / LPR, l = t % LPR, h = blockIdx.y, row0 = (int)blockIdx.x * R;
  row_slots<R, false>(a, row0, slot);
  const char* head = a.cache + (int64_t)h * a.head_bytes;
  for (int q = t >> 6; q < R; q += kThreads / 64) {
    const int p = slot[q];
    const int n = p >= 0 ? run_of<R>(slot, q) : 0;
    if (n == 0) continue;
    const char* base = head + (int64_t)(p / kTile) * a.tile_bytes;
    for (int dim = t & 63; dim < a.hd; dim += 64) {
      const char* at = base + sgc::value_at<ES>(a.D, p % kTile, dim);
      if (n == 4) {
        const pack<E, 4> x = *reinterpret_cast<const pack<E, 4>*>(at);
#pragma unroll
        for (int j = 0; j < 4; j++) vl[(q + j) * 256 + dim] = x.v[j];
      } else {
        vl[q * 256 + dim] = *reinterpret_cast<const E*>(at);
      }
    }
  }
  const int s = slot[r], row = row0 + r, key = max(s, 0) % kTile;
  const char* tile = head + (int64_t)(max(s, 0) / kTile) * a.tile_bytes;
  const float* tail = reinterpret_cast<const float*>(tile + a.tile_bytes - sgc::kTail);
  float ks = 1.0f, vs = 1.0f;
  if constexpr (Q8) {
    ks = tail[key];
    vs = tail[kTile + key];
  }
  pack<E, VEC> kp[NP];
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int dim = (l + i * LPR) * VEC;
    if (s >= 0 && dim < a.hd) kp[i] = *reinterpret_cast<const pack<E, VEC>*>(tile + sgc::key_at<ES>(a.D, key, dim));
  }
  __syncthreads();
  if (s == kNoRow) return;
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int dim = (l + i * LPR) * VEC;
    if (dim >= a.hd) continue;
    chunk<T> k, v;
    const pack<E, VEC> vp = *reinterpret_cast<const pack<E, VEC>*>(vl + r * 256 + dim);
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      if constexpr (Q8) {
        k.v[j] = elem<T>::from(s >= 0 ? (float)kp[i].v[j] * ks : 0.0f);
        v.v[j] = elem<T>::from(s >= 0 ? (float)vp.v[j] * vs : 0.0f);
      } else {
        k.v[j] = s >= 0 ? kp[i].v[j] : elem<T>::from(0.0f);
        v.v[j] = s >= 0 ? vp.v[j] : elem<T>::from(0.0f);
      }
    }
    *reinterpret_cast<chunk<T>*>(static_cast<T*>(a.k) + row * a.ldk + (int64_t)h * a.hd + dim) = k;
    *reinterpret_cast<chunk<T>*>(static_cast<T*>(a.v) + row * a.ldv + (int64_t)h * a.hd + dim) = v;
  }
}

// Few rows go four to a workgroup, so that a step's new tokens spread over the GPU.
constexpr int kManyRows = 32, kFewRows = 4;
bool few(int rows, int heads) { return (int64_t)((rows + kManyRows - 1) / kManyRows) * heads < 512; }

template <typename T, bool Q8, bool WRITE>
hipError_t run_rows(const sg_kv_rows_args& a, hipStream_t s) {
  if (few(a.rows, a.heads)) {
    const dim3 grid((a.rows + kFewRows - 1) / kFewRows, a.heads);
    return sgp::run_kernel(WRITE ? k_kv_write<T, Q8, kFewRows> : k_kv_read<T, Q8, kFewRows>, grid, dim3(kThreads), 0, s, a);
  }
  const dim3 grid((a.rows + kManyRows - 1) / kManyRows, a.heads);
  return sgp::run_kernel(WRITE ? k_kv_write<T, Q8, kManyRows> : k_kv_read<T, Q8, kManyRows>, grid, dim3(kThreads), 0, s, a);
}

template <bool WRITE>
hipError_t by_type(const sg_kv_rows_args& a, int dtype, bool q8, hipStream_t s) {
  if (dtype == SG_F32) return q8 ? run_rows<float, true, WRITE>(a, s) : run_rows<float, false, WRITE>(a, s);
  if (dtype == SG_F16) return q8 ? run_rows<_Float16, true, WRITE>(a, s) : run_rows<_Float16, false, WRITE>(a, s);
  return q8 ? run_rows<sgp::bf16_t, true, WRITE>(a, s) : run_rows<sgp::bf16_t, false, WRITE>(a, s);
}

}  // namespace

namespace sgk {

int64_t kv_rows_threads(int rows) { return (int64_t)((rows + kManyRows - 1) / kManyRows) * kThreads; }

hipError_t kv_write(const sg_kv_rows_args& a, int dtype, bool q8, hipStream_t s) { return by_type<true>(a, dtype, q8, s); }
hipError_t kv_read(const sg_kv_rows_args& a, int dtype, bool q8, hipStream_t s) { return by_type<false>(a, dtype, q8, s); }

}  // namespace sgk
