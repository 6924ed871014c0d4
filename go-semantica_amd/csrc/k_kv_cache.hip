// k_kv_cache.hip -- rows of keys and values into a cache and back out of it
// (sg_kv_cache_write, sg_kv_cache_read):
//   scale = max(fl32(max |x| / 127), 2^-126) over a row's head;  code = the integer nearest
//   to x / scale, halves to even;  x' = fl32(code * scale), rounded to the type
// or, without codes, the values as they are.
//
// A code is exact: q = rint(x / scale) is formed with a reciprocal and put right by the
// residual x - q scale, which fmaf gives without rounding (|q| <= 127; x is a multiple of
// half a scale's last place where |q| >= 1/2, and then |x - q scale| <= scale, 25 bits that
// end there).  |x| / scale is 127 (1 + 2^-23) at most, so no code is cut.
//
// A workgroup takes blocks of R rows of the packed batch and one head: 256 / R lanes a row.  Keys go
// to the cache as they were loaded, eight dims of a slot together; values cross LDS, for a
// cache's lane holds one dim of four slots in a row: four rows that fill such a run are
// stored as one, others element by element.
//
// Memory bounds them where there are many rows (131072 bf16 rows of 8 heads of 128 from codes: 170 us,
// 4.8 TB/s, as they are in and out 255 and 220; 32768 float32 rows of one head of 256 to codes and back: 23
// and 17 us, 3.6 and 4.8 TB/s, as they are 31 and 29, 4.3 and 4.6: a workgroup of these has one block of
// rows, which it loads whole before it stores), three dependent loads and a round through LDS where there
// are few (64 tokens 6 us in, 4.7 out).  Rows that stand alone in their run of four slots cost four times
// their bytes in values: 32768 single tokens 145 us out.
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
__device__ __forceinline__ int code_of(float x, float scale, float inv) {
  int q = (int)__builtin_rintf(x * inv);
  const float r = __builtin_fmaf(-(float)q, scale, x), half = 0.5f * scale;
  // (half is exact: a scale is no subnormal.  A tie goes to the even code.)
  const int up = r > half || (r == half && (q & 1)), down = r < -half || (r == -half && (q & 1));
  return q + up - down;
}

// Codes of N values, four to a word.  The nearest whole number falls out of the sum with
// 1.5 * 2^23, in its last byte as it is kept; only where some value of the wave lies half a
// scale from it or more is there anything to decide.
template <int N>
__device__ __forceinline__ void codes_of(const float* x, float scale, float inv, uint32_t* words) {
  constexpr float kRound = 12582912.0f;
  uint32_t t[N];
  float off = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float v = __builtin_fmaf(x[i], inv, kRound);
    t[i] = __float_as_uint(v);
    off = fmaxf(off, fabsf(__builtin_fmaf(-(v - kRound), scale, x[i])));
  }
  if (__ballot(off >= 0.5f * scale)) {
    asm volatile("");  // (a branch)
#pragma unroll
    for (int i = 0; i < N; i++) t[i] = (uint32_t)code_of(x[i], scale, inv);
  }
#pragma unroll
  for (int i = 0; i < N / 4; i++) {
    const uint32_t a = __builtin_amdgcn_perm(t[4 * i + 1], t[4 * i], 0x0c0c0400u);
    const uint32_t b = __builtin_amdgcn_perm(t[4 * i + 3], t[4 * i + 2], 0x04000c0cu);
    words[i] = a | b;
  }
}

// The slot of each of the workgroup's rows (up to `count`), in LDS: kNone for a slot outside the
// cache (or, on the way in, one that a later sequence of the call fills as well), kNoRow for a
// row of no sequence.
constexpr int kNone = -1, kNoRow = -2;

template <bool WRITE>
__device__ __forceinline__ void row_slots(const sg_kv_rows_args& a, int row0, int count, int32_t* slot) {
  __shared__ int32_t span[3][kThreads / 64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  int lo = INT32_MAX, hi = -1, first = INT32_MAX;  // the slots that the rows span, and their first sequence
  const int base = row0 + wave * 64;
  if (wave * 64 < count && base < a.rows) {
    const int last = min(min(base + 64, row0 + count), a.rows) - 1, row = base + lane;
    int i, s0, s1;
    sgp::row_seq(a.off, a.n_seq, base, last, min(row, last), lane, i, s0, s1);
    const bool there = row <= last && row >= s0 && row < s1;
    const int start = a.starts[i];
    const int64_t s = (int64_t)start + row - s0;
    const bool in = there && start >= 0 && s >= 0 && s < a.slots;
    if (wave * 64 + lane < count) slot[wave * 64 + lane] = in ? (int)s : there ? kNone : kNoRow;
    if (in) {
      lo = hi = (int)s;
      first = i;
    }
  } else if (t < count) {
    slot[t] = kNoRow;
  }
  if constexpr (WRITE) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      lo = min(lo, __shfl_xor(lo, o));
      hi = max(hi, __shfl_xor(hi, o));
      first = min(first, __shfl_xor(first, o));
    }
    if (lane == 0) {
      span[0][wave] = lo;
      span[1][wave] = hi;
      span[2][wave] = first;
    }
  }
  __syncthreads();
  if constexpr (WRITE) {
    for (int w = 0; w < kThreads / 64; w++) {
      lo = min(lo, span[0][w]);
      hi = max(hi, span[1][w]);
      first = min(first, span[2][w]);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    first = __builtin_amdgcn_readfirstlane(first);
    if (hi < 0) return;  // (alike for all threads)
    for (int j = first + 1 + t; j < a.n_seq; j += kThreads) {
      const int64_t b = a.starts[j];
      const int r0 = sgp::clamp_row(a.off[j], a.rows), r1 = sgp::clamp_row(a.off[j + 1], a.rows);
      if (b < 0 || r1 <= r0 || b > hi || b + (r1 - r0) <= lo) continue;
      for (int r = 0; r < count && row0 + r < r0; r++) {  // rows of sequences before j
        const int s = slot[r];
        if (s >= b && s < b + (r1 - r0)) slot[r] = kNone;
      }
    }
    __syncthreads();
  }
}

// Each row's part in its run of four slots, in LDS: 4: the run's rows stand in its block of R and
// this is the first, 0: another of them, or a row without a slot, 1: a row that stands for itself.
template <int R>
__device__ __forceinline__ void runs_of(const int32_t* slot, int count, int32_t* run) {
  for (int r = threadIdx.x; r < count; r += kThreads) {
    const int s = slot[r], o = s & 3, f = r % R - o;
    bool whole = s >= 0 && f >= 0 && f + 3 < R;
    if (whole)
#pragma unroll
      for (int q = 0; q < 4; q++) whole &= slot[r - o + q] == s - o + q;
    run[r] = s < 0 ? 0 : whole ? (o == 0 ? 4 : 0) : 1;
  }
  __syncthreads();
}

// N elements of 1, 2 or 4 bytes as one store.
template <typename E, int N>
struct alignas(sizeof(E) * N) pack {
  E v[N];
};

// A pack moves as the whole it is (its elements by themselves would be as many instructions).
template <int BYTES>
struct whole;
template <>
struct whole<1> {
  typedef uint8_t type;
};
template <>
struct whole<2> {
  typedef uint16_t type;
};
template <>
struct whole<4> {
  typedef uint32_t type;
};
template <>
struct whole<8> {
  typedef uint32_t type __attribute__((ext_vector_type(2)));
};
template <>
struct whole<16> {
  typedef uint32_t type __attribute__((ext_vector_type(4)));
};
template <typename P>
__device__ __forceinline__ P get(const void* at) {
  return __builtin_bit_cast(P, *static_cast<const typename whole<sizeof(P)>::type*>(at));
}
template <typename P>
__device__ __forceinline__ void put(void* at, const P& p) {
  *static_cast<typename whole<sizeof(P)>::type*>(at) = __builtin_bit_cast(typename whole<sizeof(P)>::type, p);
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
constexpr uint32_t kInf = 0x7f800000u;

// A workgroup's share: `subs` blocks of R rows, `heads` heads of each, one (block, head) after
// another with the next one's loads on their way: finding the rows' slots is three dependent loads,
// and a block's load and store one more each.
// Rows lie 256 bytes' multiples apart and so does a head in them: workgroups of an XCD that went
// over the heads in step would meet in an eighth of its L2's channels, so each begins elsewhere.
struct share {
  int row0, head0, heads, items, turn;
  __device__ __forceinline__ int sub(int item) const { return item / heads; }
  __device__ __forceinline__ int head(int item) const { return head0 + (item + turn) % heads; }
};
template <int R>
__device__ __forceinline__ share share_of(const sg_kv_rows_args& a, int subs, int heads) {
  const int groups = (a.heads + heads - 1) / heads;
  share s;
  s.row0 = (int)(blockIdx.x / groups) * (subs * R);
  s.head0 = (int)(blockIdx.x % groups) * heads;
  s.heads = min(heads, a.heads - s.head0);
  s.turn = blockIdx.x / 8;
  s.items = min(subs, (a.rows - s.row0 + R - 1) / R) * s.heads;
  return s;
}

constexpr int kMostRowsOf = 256;  // a workgroup's, at most

template <typename T, bool Q8, int R>
__global__ __launch_bounds__(kThreads) void k_kv_write(sg_kv_rows_args a, int subs, int heads) {
  typedef typename sgc::kept<T, Q8>::type E;
  constexpr int ES = sizeof(E), VEC = elem<T>::vec, LPR = kThreads / R, NP = (256 / VEC + LPR - 1) / LPR;
  __shared__ int32_t slot[kMostRowsOf], run[kMostRowsOf];
  __shared__ alignas(16) E vl[2][R * 256];
  const int t = threadIdx.x, r = t / LPR, l = t % LPR, pieces = a.hd / VEC;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const share sh = share_of<R>(a, subs, heads);
  chunk<T> k[NP], v[NP];
  auto load = [&](int item) {
    const int row = min(sh.row0 + sh.sub(item) * R + r, a.rows - 1);
    const int64_t col = (int64_t)sh.head(item) * a.hd;
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const int at = l + i * LPR;
      if (at < pieces) {
        k[i] = get<chunk<T>>(static_cast<const T*>(a.k) + row * a.ldk + col + at * VEC);
        v[i] = get<chunk<T>>(static_cast<const T*>(a.v) + row * a.ldv + col + at * VEC);
      }
    }
  };
  load(0);
  row_slots<true>(a, sh.row0, subs * R, slot);
  runs_of<R>(slot, subs * R, run);
  for (int item = 0; item < sh.items; item++) {
    const int sub = sh.sub(item) * R, h = sh.head(item);
    E* vt = vl[item & 1];
    const int s = slot[sub + r], key = max(s, 0) % kTile;
    char* tile = a.cache + (int64_t)h * a.head_bytes + (int64_t)(max(s, 0) / kTile) * a.tile_bytes;
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
      if constexpr (Q8) {
        struct {
          uint32_t w[VEC / 4];
        } kw, vw;
        float x[VEC], y[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          x[j] = km < kInf ? elem<T>::to(k[i].v[j]) : 0.0f;
          y[j] = vm < kInf ? elem<T>::to(v[i].v[j]) : 0.0f;
        }
        codes_of<VEC>(x, ks, ki, kw.w);
        codes_of<VEC>(y, vs, vi, vw.w);
        kp = __builtin_bit_cast(pack<E, VEC>, kw);
        vp = __builtin_bit_cast(pack<E, VEC>, vw);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          kp.v[j] = k[i].v[j];
          vp.v[j] = v[i].v[j];
        }
      }
      put(vt + r * 256 + dim, vp);
      if (s >= 0) put(tile + sgc::key_at<ES>(a.D, key, dim), kp);
    }
    if (item + 1 < sh.items) load(item + 1);
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
    __syncthreads();  // (the other stage was read before it)
    for (int q = wave; q < R; q += kThreads / 64) {
      const int n = __builtin_amdgcn_readfirstlane(run[sub + q]);
      if (n == 0) continue;
      const int p = __builtin_amdgcn_readfirstlane(slot[sub + q]);
      char* base = a.cache + (int64_t)h * a.head_bytes + (int64_t)(p / kTile) * a.tile_bytes;
      for (int dim = t & 63; dim < a.hd; dim += 64) {
        char* at = base + sgc::value_at<ES>(a.D, p % kTile, dim);
        if (n == 4) {
          pack<E, 4> x;
#pragma unroll
          for (int j = 0; j < 4; j++) x.v[j] = vt[(q + j) * 256 + dim];
          put(at, x);
        } else {
          put(at, vt[q * 256 + dim]);
        }
      }
    }
  }
}

template <typename T, bool Q8, int R>
__global__ __launch_bounds__(kThreads) void k_kv_read(sg_kv_rows_args a, int subs, int heads) {
  typedef typename sgc::kept<T, Q8>::type E;
  constexpr int ES = sizeof(E), VEC = elem<T>::vec, LPR = kThreads / R, NP = (256 / VEC + LPR - 1) / LPR;
  constexpr int RW = R / (kThreads / 64);  // rows of a wave in the values' transposition
  __shared__ int32_t slot[kMostRowsOf], run[kMostRowsOf];
  __shared__ alignas(16) E vl[2][R * 256];
  const int t = threadIdx.x, r = t / LPR, l = t % LPR, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const share sh = share_of<R>(a, subs, heads);
  row_slots<false>(a, sh.row0, subs * R, slot);
  runs_of<R>(slot, subs * R, run);
  pack<E, VEC> kp[NP];
  pack<E, 4> vp[RW][4];
  float ks = 1.0f, vs = 1.0f;
  auto load = [&](int item) {
    const int sub = sh.sub(item) * R;
    const char* head = a.cache + (int64_t)sh.head(item) * a.head_bytes;
#pragma unroll
    for (int i = 0; i < RW; i++) {
      const int q = wave * RW + i, n = __builtin_amdgcn_readfirstlane(run[sub + q]);
      if (n == 0) continue;
      const int p = __builtin_amdgcn_readfirstlane(slot[sub + q]);
      const char* base = head + (int64_t)(p / kTile) * a.tile_bytes;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int dim = (t & 63) + e * 64;
        if (e * 64 >= a.hd) break;
        if (dim >= a.hd) continue;
        const char* at = base + sgc::value_at<ES>(a.D, p % kTile, dim);
        if (n == 4) vp[i][e] = get<pack<E, 4>>(at);
        else vp[i][e].v[0] = get<E>(at);
      }
    }
    const int s = slot[sub + r], key = max(s, 0) % kTile;
    const char* tile = head + (int64_t)(max(s, 0) / kTile) * a.tile_bytes;
    if (s >= 0) {
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const int dim = (l + i * LPR) * VEC;
        if (dim < a.hd) kp[i] = get<pack<E, VEC>>(tile + sgc::key_at<ES>(a.D, key, dim));
      }
      if constexpr (Q8) {
        const float* tail = reinterpret_cast<const float*>(tile + a.tile_bytes - sgc::kTail);
        ks = tail[key];
        vs = tail[kTile + key];
      }
    }
  };
  load(0);
  for (int item = 0; item < sh.items; item++) {
    const int sub = sh.sub(item) * R;
    E* vt = vl[item & 1];
#pragma unroll
    for (int i = 0; i < RW; i++) {
      const int q = wave * RW + i, n = __builtin_amdgcn_readfirstlane(run[sub + q]);
      if (n == 0) continue;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int dim = (t & 63) + e * 64;
        if (e * 64 >= a.hd) break;
        if (dim >= a.hd) continue;
        vt[q * 256 + dim] = vp[i][e].v[0];
        if (n == 4)
#pragma unroll
          for (int j = 1; j < 4; j++) vt[(q + j) * 256 + dim] = vp[i][e].v[j];
      }
    }
    const int s = slot[sub + r];
    const int64_t row = sh.row0 + sub + r, col = (int64_t)sh.head(item) * a.hd;
    const float vscale = vs;
    if (s != kNoRow) {
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const int dim = (l + i * LPR) * VEC;
        if (dim >= a.hd) continue;
        chunk<T> k;
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          if constexpr (Q8) k.v[j] = elem<T>::from(s >= 0 ? (float)kp[i].v[j] * ks : 0.0f);
          else k.v[j] = s >= 0 ? kp[i].v[j] : elem<T>::from(0.0f);
        }
        put(static_cast<T*>(a.k) + row * a.ldk + col + dim, k);
      }
    }
    if (item + 1 < sh.items) load(item + 1);
    __syncthreads();  // (the other stage was read before it)
    if (s == kNoRow) continue;
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const int dim = (l + i * LPR) * VEC;
      if (dim >= a.hd) continue;
      chunk<T> v;
      const pack<E, VEC> x = get<pack<E, VEC>>(vt + r * 256 + dim);
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        if constexpr (Q8) v.v[j] = elem<T>::from(s >= 0 ? (float)x.v[j] * vscale : 0.0f);
        else v.v[j] = s >= 0 ? x.v[j] : elem<T>::from(0.0f);
      }
      put(static_cast<T*>(a.v) + row * a.ldv + col + dim, v);
    }
  }
}

// Few rows go four to a workgroup, so that a step's new tokens spread over the GPU; many in
// blocks of 32 (16 of float32 as it is, whose two stages then fit LDS), up to eight (block, head)
// to a workgroup as long as there are workgroups for the GPU.
// (Single tokens, bf16, 8 heads of 128, in and out, us, by 4 and by 32: 64 tokens 10 and 21, 1024 20 and 24,
// 2048 34 and 29, 8192 146 and 81.  131072 rows out: one (block, head) to a workgroup 186 us, two 172,
// eight 170; 512 workgroups are too few for 32768 float32 rows in and out: 52 for 41.)
constexpr int kFewRows = 4;
constexpr int64_t kEnough = 2048;  // workgroups

struct launch_shape {
  int rows, subs, heads;  // of a block; blocks and heads of a workgroup
  int64_t groups;
};
launch_shape shape(int rows, int heads, bool wide) {
  const int many = wide ? 16 : 32;
  launch_shape s{many, 1, 1, 0};
  auto count = [&] { s.groups = ((int64_t)rows + (int64_t)s.rows * s.subs - 1) / (s.rows * s.subs) * ((heads + s.heads - 1) / s.heads); };
  count();
  if (s.groups < 512) {
    s.rows = kFewRows;
    count();
    return s;
  }
  while (s.heads * s.subs < 8 && s.groups >= 2 * kEnough) {
    if (s.heads * 2 <= heads) s.heads *= 2;
    else s.subs *= 2;
    count();
  }
  return s;
}

constexpr bool is_wide(bool f32, bool q8) { return f32 && !q8; }

template <typename T, bool Q8, bool WRITE>
hipError_t run_rows(const sg_kv_rows_args& a, hipStream_t s) {
  constexpr int MANY = is_wide(sizeof(T) == 4, Q8) ? 16 : 32;
  const launch_shape f = shape(a.rows, a.heads, MANY == 16);
  const dim3 grid((unsigned)f.groups);
  if (f.rows == kFewRows)
    return sgp::run_kernel(WRITE ? k_kv_write<T, Q8, kFewRows> : k_kv_read<T, Q8, kFewRows>, grid, dim3(kThreads), 0, s, a, f.subs, f.heads);
  return sgp::run_kernel(WRITE ? k_kv_write<T, Q8, MANY> : k_kv_read<T, Q8, MANY>, grid, dim3(kThreads), 0, s, a, f.subs, f.heads);
}

template <bool WRITE>
hipError_t by_type(const sg_kv_rows_args& a, int dtype, bool q8, hipStream_t s) {
  if (dtype == SG_F32) return q8 ? run_rows<float, true, WRITE>(a, s) : run_rows<float, false, WRITE>(a, s);
  if (dtype == SG_F16) return q8 ? run_rows<_Float16, true, WRITE>(a, s) : run_rows<_Float16, false, WRITE>(a, s);
  return q8 ? run_rows<sgp::bf16_t, true, WRITE>(a, s) : run_rows<sgp::bf16_t, false, WRITE>(a, s);
}

}  // namespace

namespace sgk {

int64_t kv_rows_threads(int rows, int heads, int dtype, bool q8) {
  return shape(rows, heads, is_wide(dtype == SG_F32, q8)).groups * kThreads;
}

hipError_t kv_write(const sg_kv_rows_args& a, int dtype, bool q8, hipStream_t s) { return by_type<true>(a, dtype, q8, s); }
hipError_t kv_read(const sg_kv_rows_args& a, int dtype, bool q8, hipStream_t s) { return by_type<false>(a, dtype, q8, s); }

}  // namespace sgk
