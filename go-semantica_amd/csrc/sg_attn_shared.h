// sg_attn_shared.h -- attention of a batch's queries over kept keys and values
// (sg_attention_shared): the kernels, shared by the files that instantiate them.
// k_attn_shared.hip has the plan and the join.
//
// A query's keys are places 0 .. plen - 1, its prefix, and plen .. plen + len - 1, its
// sequence's own.  Query rows times the query heads of a key head are pairs; a job is M
// consecutive pairs of one group -- all sequences behind one prefix, over that prefix, or one
// sequence, over its own keys -- and a list of jobs is laid end to end in units (a tile of 32
// slots) and dealt to workers in equal shares, whatever the lengths: a worker ends in the
// middle of a job and the next one goes on there.  So a long prefix is split over the GPU
// when there are few queries and read once for all of them when there are many, and nothing
// about the lengths is needed on the host.  What a worker has of a job -- running maximum m,
// sum l and output O, unnormalised -- goes to the workspace, and k_attn_join adds up.
//
// Scores are formed transposed, S^T = K Q^T on 16x16 tiles: a lane has one pair's scores of
// four keys in a row, twice for 32 keys, and these eight are, as they stand, its part of the
// B operand of O^T += V^T P^T, for values are kept in that order (sg_kv_cache.h).
//
// Codes of 8 bits are whole numbers, exact in the type: the keys' scale multiplies the
// score, the values' the weight.  float32 queries and weights go over codes as three bf16 parts, 24
// bits (48 cycles of 32 products of 16 and 16 where float32's own take 256); over float32 keys and
// values it goes through float32 matrix products.
//
// 16-bit types round the weights once, for the second product: to the type itself over keys
// and values as they are (their sum is taken of the rounded ones), and over codes, with the value's
// scale in them, to bf16 with bf16 queries; with fp16 queries that product would leave fp16's range, so
// they are split into two bf16 halves (2^-17 of each, exponents of float32) and the codes taken
// as bf16.  This is as large as the rounding of the result: the error against 64 bits is 2.3e-3 in
// bf16 for 1.66e-3 with weights of float32's precision, in fp16 2.8e-4 for 2.1e-4.  Two halves everywhere
// would give that, for another second product (us, rounded and in halves): 32 x 512 bf16 behind 8192 2250
// and 3140, 600 bf16 rows of 256 dims behind 20000 146 and 177, over codes 64 tokens behind 8192 68 and
// 72, 27 rows behind 131072 133 and 154.
//
// What bounds them (MI355X): a wide workgroup of bf16 takes each fragment of a tile from LDS for two
// products, and a pair and lane has eight exponentials of 16 cycles; vector and matrix
// instructions of a SIMD overlap little, and two waves a SIMD hide the rest.
//   bf16, 16384 rows of 32 heads over 8 of 128 dims behind 8192 places: 2.2 ms, 1020 TFLOP/s of the 1214
//   that a large product reaches.
//   bf16 over codes, 27 rows of 32 heads over 8 behind 131072 places: 112 us, 2.5 TB/s: decoding and
//   the softmax of a tile stand between its load and the next barrier.
//   float32, 10476 rows of 3 heads over 1 of 256 dims, window 512: 198 us, 83 of 152 TFLOP/s: two
//   waves a SIMD, products that wait for fragments.
//   one float32 query of 3 heads over 1 of 256 dims behind 1536 places (narrow): 12 us, one tile a
//   wave, its loads' latency and 256 products in a row.
#pragma once
#include <atomic>

#include "semantica_gpu.h"
#include "sg_kernels.h"
#include "sg_kv_cache.h"

namespace sga {

using sgc::kTail;
using sgc::kTile;
using sgp::bf16_t;
using sgp::elem;

typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
constexpr float kLog2e = 1.44269504088896340736f;

// Eight elements in a row of a matrix core operand.
template <typename T>
struct frag {
  typedef s16x8_t type;
};
struct f32x8_t {
  f32x4_t v[2];
};
template <>
struct frag<float> {
  typedef f32x8_t type;
};

__device__ __forceinline__ f32x4_t mma(_Float16, s16x8_t a, s16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mma(bf16_t, s16x8_t a, s16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(sgp::bf16x8_t, a), __builtin_bit_cast(sgp::bf16x8_t, b), c,
                                                 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mma(float, const f32x8_t& a, const f32x8_t& b, f32x4_t c) {
#pragma unroll
  for (int j = 0; j < 8; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j >> 2][j & 3], b.v[j >> 2][j & 3], c, 0, 0, 0);
  return c;
}
// A part of a score.  (float32: 32 products by themselves, then added: shorter sums are nearer, and
// do not wait for each other, which few waves gain by; many lose 7 %.)
template <typename K, typename F>
__device__ __forceinline__ f32x4_t add_score(const F& a, const F& b, f32x4_t c) {
  if constexpr (__is_same(K, float)) return c + mma(K{}, a, b, f32x4_t{0, 0, 0, 0});
  else return mma(K{}, a, b, c);
}

// Eight codes (two words) as M.
template <typename M>
__device__ __forceinline__ typename frag<M>::type decode(uint32_t lo, uint32_t hi) {
  const uint32_t w[2] = {lo, hi};
  if constexpr (__is_same(M, float)) {
    f32x8_t x;
#pragma unroll
    for (int j = 0; j < 8; j++) x.v[j >> 2][j & 3] = (float)(int8_t)(w[j >> 2] >> ((j & 3) * 8));
    return x;
  } else if constexpr (__is_same(M, _Float16)) {
    // 0x6400 + u is fp16's 1024 + u: bytes c + 128 behind 0x64, less 1152.
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    u32x4_t x;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const uint32_t u = w[i] ^ 0x80808080u;
      const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
      x[2 * i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off);
      x[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off);
    }
    return __builtin_bit_cast(s16x8_t, x);
  } else {
    // A float's upper half is the bf16: whole numbers below 2^8 have nothing in the lower.
    u32x4_t x;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t v = w[i >> 1] >> ((i & 1) * 16);
      const float a = (float)(int8_t)v, b = (float)(int8_t)(v >> 8);
      x[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    }
    return __builtin_bit_cast(s16x8_t, x);
  }
}

template <typename M>
__device__ __forceinline__ typename frag<M>::type load_frag(const char* base, int f, int lane) {
  if constexpr (__is_same(M, float)) {
    f32x8_t x;
    x.v[0] = *reinterpret_cast<const f32x4_t*>(base + f * 2048 + lane * 16);
    x.v[1] = *reinterpret_cast<const f32x4_t*>(base + f * 2048 + 1024 + lane * 16);
    return x;
  } else {
    return *reinterpret_cast<const s16x8_t*>(base + f * 1024 + lane * 16);
  }
}

template <typename M>
__device__ __forceinline__ void store_frag(char* base, int f, int lane, const typename frag<M>::type& x) {
  if constexpr (__is_same(M, float)) {
    *reinterpret_cast<f32x4_t*>(base + f * 2048 + lane * 16) = x.v[0];
    *reinterpret_cast<f32x4_t*>(base + f * 2048 + 1024 + lane * 16) = x.v[1];
  } else {
    *reinterpret_cast<s16x8_t*>(base + f * 1024 + lane * 16) = x;
  }
}

// 2^x, -infinity to 0.
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh: x P(x^2) below 1/2 (9e-8 relative), 1 - 2 / (1 + e^2x) above.
__device__ __forceinline__ float tanh_of(float x) {
  const float z = x * x, ax = fabsf(x);
  float p = __builtin_fmaf(z, -0.00661201408f, 0.021273822f);
  p = __builtin_fmaf(z, p, -0.0538932246f);
  p = __builtin_fmaf(z, p, 0.133329003f);
  p = __builtin_fmaf(z, p, -0.333333241f);
  p = __builtin_fmaf(z, p, 1.0f) * x;
  const float e = exp2_of(2.0f * kLog2e * ax);
  const float far = __builtin_copysignf(1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f), x);
  return ax < 0.5f ? p : far;  // (a NaN is far's)
}

// The largest over the four lanes that share a pair: lane, lane ^ 16, ^ 32, ^ 48.
__device__ __forceinline__ float pair_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float pair_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// The type that a kernel's values and weights are multiplied in, and the weights' halves.
template <typename T, bool Q8>
struct weight {
  typedef T type;
  static constexpr int parts = 1;
};
template <>
struct weight<_Float16, true> {
  typedef bf16_t type;
  static constexpr int parts = 2;
};
template <>
struct weight<bf16_t, true> {
  typedef bf16_t type;
  static constexpr int parts = 1;
};
template <>
struct weight<float, true> {
  typedef bf16_t type;
  static constexpr int parts = 3;
};
// The same of keys and queries.
template <typename T, bool Q8>
struct query {
  typedef T type;
  static constexpr int parts = 1;
};
template <>
struct query<float, true> {
  typedef bf16_t type;
  static constexpr int parts = 3;
};
// fp16 weights are multiplied by 2^6, so that they keep their bits down to 2^-20; sums and outputs
// alike, so it leaves by itself.
template <typename T, bool Q8>
constexpr float kShift = __is_same(T, _Float16) && !Q8 ? 6.0f : 0.0f;
// A tile's sum of weights from which on a pair's maximum is raised (and its sums rescaled): far
// above 32 weights of 1, within the weights' type.
template <typename T, bool Q8>
constexpr float kMost = __is_same(T, _Float16) && !Q8 ? 0x1p14f : 0x1p10f;

// Sums of weights by the matrix core: 16-bit types whose weights are multiplied as they are.
template <typename T, bool Q8>
constexpr bool kSumByProduct = !Q8 && sizeof(T) == 2;

// What a wave has of its QT * 16 pairs: queries, running maxima and sums, outputs.
template <typename T, bool Q8, int D, int QT>
struct state {
  typename frag<typename query<T, Q8>::type>::type q[QT][D / 32][query<T, Q8>::parts];
  f32x4_t o[QT][D / 16];
  float m[QT], l[QT];
  float base[QT], most[QT];  // what scores are taken against: m, shifted; the sum that raises it
  int lo[QT], hi[QT];  // visible keys of the lane's pairs, counted from the job's first
  int all_lo, all_hi;  // keys that every pair of the wave sees
};

// Eight weights as operands of the second product.
template <typename T, bool Q8>
__device__ __forceinline__ void pack_weights(const float* p, typename frag<typename weight<T, Q8>::type>::type* w) {
  typedef typename query<T, Q8>::type K;
  typedef typename weight<T, Q8>::type M;
  if constexpr (__is_same(M, float)) {
#pragma unroll
    for (int j = 0; j < 8; j++) w[0].v[j >> 2][j & 3] = p[j];
  } else if constexpr (__is_same(M, _Float16)) {
    half8_t x;
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = (_Float16)p[j];
    w[0] = __builtin_bit_cast(s16x8_t, x);
  } else {
    sgp::bf16x8_t x;
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = (__bf16)p[j];
    w[0] = __builtin_bit_cast(s16x8_t, x);
    if constexpr (weight<T, Q8>::parts >= 2) {
      sgp::bf16x8_t y, z;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float rest = p[j] - (float)x[j];
        y[j] = (__bf16)rest;
        z[j] = (__bf16)(rest - (float)y[j]);
      }
      w[1] = __builtin_bit_cast(s16x8_t, y);
      if constexpr (weight<T, Q8>::parts == 3) w[2] = __builtin_bit_cast(s16x8_t, z);
    }
  }
}

// A tile's products become weights.  first: the place of the tile's first slot among the keys
// that lo and hi count (negative where the tile begins before them); tail: the tile's, in LDS or
// memory.  Weights are 2^(s c - m) of scores s as they come: c > 0 holds the scale (queries are
// negated for a negative one), so one fma does the rest.  m need not be the maximum: it is that of
// the tile that a pair saw first, and raised when a tile's weights add up to kMost or more, which
// the sum tells that is taken anyway.
template <typename T, bool Q8, int D, int QT>
__device__ __forceinline__ void weigh(const sg_attn_shared_args& a, state<T, Q8, D, QT>& st, f32x4_t (&s)[2][QT], int first,
                                      const float* tail, int lane,
                                      typename frag<typename weight<T, Q8>::type>::type (&w)[QT][weight<T, Q8>::parts]) {
  const int g = lane >> 4;
  float vs[8], p[QT][8];
  if constexpr (Q8) {
    f32x4_t ks[2], v[2];
#pragma unroll
    for (int half = 0; half < 2; half++) {
      ks[half] = *reinterpret_cast<const f32x4_t*>(tail + half * 16 + g * 4);
      v[half] = *reinterpret_cast<const f32x4_t*>(tail + kTile + half * 16 + g * 4);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      vs[j] = v[j >> 2][j & 3];
#pragma unroll
      for (int t = 0; t < QT; t++) p[t][j] = s[j >> 2][t][j & 3] * ks[j >> 2][j & 3];
    }
  } else {
#pragma unroll
    for (int t = 0; t < QT; t++)
#pragma unroll
      for (int j = 0; j < 8; j++) p[t][j] = s[j >> 2][t][j & 3];
  }
  if (a.cap != 0.0f) {
#pragma unroll
    for (int t = 0; t < QT; t++)
#pragma unroll
      for (int j = 0; j < 8; j++) p[t][j] = a.cap * tanh_of(p[t][j] * a.to_cap);
  }
  const bool part = first < st.all_lo || first + kTile > st.all_hi;
  if (part) {
#pragma unroll
    for (int t = 0; t < QT; t++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int key = first + (j >> 2) * 16 + g * 4 + (j & 3);
        p[t][j] = key >= st.lo[t] && key < st.hi[t] ? p[t][j] : -INFINITY;
      }
  }
  // A hidden key's scale may be NaN, and one's whose score is -infinity: it has no weight.
  bool skip = part;
  if constexpr (Q8) {
    const float any = ((vs[0] + vs[1]) + (vs[2] + vs[3])) + ((vs[4] + vs[5]) + (vs[6] + vs[7]));
    skip |= __ballot(any != any) != 0;
  }
#pragma unroll
  for (int t = 0; t < QT; t++) {
    float e[8], sum;
    auto form = [&](bool far) {
#pragma unroll
      for (int j = 0; j < 8; j++)
        e[j] = exp2_of(far ? p[t][j] * a.scale - st.m[t] + kShift<T, Q8> : __builtin_fmaf(p[t][j], a.scale, -st.base[t]));
      if constexpr (kSumByProduct<T, Q8>) {
        // The packed weights' sum by a product with ones: a sixteenth of the second product's work
        // in place of eight additions a lane, and the sum of the weights as they are multiplied.
        pack_weights<T, Q8>(e, w[t]);
        const short one = __builtin_bit_cast(short, elem<T>::from(1.0f));
        const s16x8_t ones = {one, one, one, one, one, one, one, one};
        sum = mma(T{}, ones, w[t][0], f32x4_t{0, 0, 0, 0})[0];
      } else {
        sum = ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
      }
    };
    form(false);
    if (__ballot(sum > st.most[t])) {
      float top = fmaxf(fmaxf(fmaxf(p[t][0], p[t][1]), fmaxf(p[t][2], p[t][3])),
                        fmaxf(fmaxf(p[t][4], p[t][5]), fmaxf(p[t][6], p[t][7]))) * a.scale;
      top = fmaxf(pair_max(top), st.m[t]);
      const float by = top > st.m[t] ? exp2_of(st.m[t] - top) : 1.0f;  // (m may be -infinity: 0)
      st.m[t] = top;
      st.base[t] = (top == -INFINITY ? 0.0f : top) - kShift<T, Q8>;
      // (A maximum of 2^24 or more is rounded by one or more: there the products are rounded as it was,
      // tile by tile, so that the largest weight is 1 and not two to that rounding.)
      const bool far = fabsf(top) >= 0x1p24f && top != -INFINITY;
      st.most[t] = top == -INFINITY || far ? -1.0f : kMost<T, Q8>;
      st.l[t] *= by;
#pragma unroll
      for (int f = 0; f < D / 16; f++) {
        if constexpr (Q8) {
          st.o[t][f] *= by;
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++) st.o[t][f][i] = sgc::faded(st.o[t][f][i], by);
        }
      }
      form(far);
    }
    st.l[t] += sum;
    if constexpr (Q8) {
#pragma unroll
      for (int j = 0; j < 8; j++) e[j] *= vs[j];
      if (skip) {
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = p[t][j] == -INFINITY ? 0.0f : e[j];
      }
    }
    if constexpr (!kSumByProduct<T, Q8>) pack_weights<T, Q8>(e, w[t]);
  }
}

// Values that are not finite, in a tile that may be hidden in part: a zero weight times one is a
// NaN.  So they are zeros in the product (clean), and which pairs see an infinity or a NaN of a
// dim is counted by products of ones behind it (mark_bad): exact, and no business of the weights',
// not of later ones either (sgc::faded).
template <typename M>
__device__ __forceinline__ void set_elem(typename frag<M>::type& x, int j, float v) {
  if constexpr (__is_same(M, float)) x.v[j >> 2][j & 3] = v;
  else x[j] = __builtin_bit_cast(short, elem<M>::from(v));
}
template <typename M>
__device__ __forceinline__ float get_elem(const typename frag<M>::type& x, int j) {
  if constexpr (__is_same(M, float)) return x.v[j >> 2][j & 3];
  else return elem<M>::to(__builtin_bit_cast(M, (short)x[j]));
}
template <typename T>
__device__ __forceinline__ typename frag<T>::type clean(typename frag<T>::type x) {
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float v = get_elem<T>(x, j);
    set_elem<T>(x, j, fabsf(v) < INFINITY ? v : 0.0f);
  }
  return x;
}
template <typename T, bool Q8, int D, int QT>
__device__ __forceinline__ void mark_bad(state<T, Q8, D, QT>& st, int first, const char* vals, int lane) {
  typedef typename frag<T>::type X;
  X sees[QT];
#pragma unroll
  for (int t = 0; t < QT; t++)
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int key = first + (j >> 2) * 16 + (lane >> 4) * 4 + (j & 3);
      set_elem<T>(sees[t], j, key >= st.lo[t] && key < st.hi[t] ? 1.0f : 0.0f);
    }
#pragma unroll
  for (int f = 0; f < D / 16; f++) {
    const X x = load_frag<T>(vals, f, lane);
    X one[3];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float v = get_elem<T>(x, j);
      set_elem<T>(one[0], j, v == INFINITY ? 1.0f : 0.0f);
      set_elem<T>(one[1], j, v == -INFINITY ? 1.0f : 0.0f);
      set_elem<T>(one[2], j, v != v ? 1.0f : 0.0f);
    }
#pragma unroll
    for (int t = 0; t < QT; t++) {
      const f32x4_t none = {0, 0, 0, 0};
      const f32x4_t up = mma(T{}, one[0], sees[t], none), down = mma(T{}, one[1], sees[t], none),
                    nan = mma(T{}, one[2], sees[t], none);
      f32x4_t add;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float a = (up[i] != 0.0f ? INFINITY : 0.0f) - (down[i] != 0.0f ? INFINITY : 0.0f);
        add[i] = nan[i] != 0.0f ? __builtin_nanf("") : a;
      }
      st.o[t][f] += add;
    }
    asm volatile("" ::: "memory");  // (one fragment at a time: registers)
  }
}

// Worker index of a workgroup: workgroups go round the eight XCDs, and neighbouring workers, which
// read the same head's tiles, stay on one.
__device__ __forceinline__ int spread(int block, int blocks) { return (block & 7) * (blocks >> 3) + (block >> 3); }

// Which (job, units) a worker has: the list laid out head by head, `per` units a worker.
struct share {
  int head, job;
  int64_t at, left;  // unit within the head's, units to do
};

__device__ __forceinline__ share first_share(const sg_attn_list& list, int64_t worker, int heads, int lane) {
  share s{0, 0, 0, 0};
  const int64_t units = list.plan->units, per = list.plan->per, total = units * heads;
  const int64_t begin = worker * per;
  if (begin >= total) return s;
  s.left = min(per, total - begin);
  s.head = (int)sgc::quotient(begin, units);
  s.at = begin - s.head * units;
  // The last job that begins at or before the unit: it is not empty.
  s.job = sgc::last_at_most(list.cum, list.plan->jobs, s.at, lane);
  return s;
}

// Loads the queries of the wave's pairs of a job.
template <typename T, bool Q8, int D, int QT>
__device__ __forceinline__ void begin_job(const sg_attn_shared_args& a, state<T, Q8, D, QT>& st, const sg_attn_job& job, int head,
                                          int pair0, int lane) {
#pragma unroll
  for (int t = 0; t < QT; t++) {
    const int pair = pair0 + t * 16 + (lane & 15);
    const bool in = pair < job.rows * a.group;
    const int r = in ? pair / a.group : 0, h = head * a.group + (in ? pair - r * a.group : 0);
    const T* q = static_cast<const T*>(a.q) + (int64_t)(job.row0 + r) * a.ldq + (int64_t)h * a.hd;
#pragma unroll
    for (int d = 0; d < D / 32; d++) {
      const int dim = d * 32 + (lane >> 4) * 8;
      typename frag<T>::type x{};
      if (in && dim < a.hd) {
        if constexpr (__is_same(T, float)) {
          x.v[0] = *reinterpret_cast<const f32x4_t*>(q + dim);
          x.v[1] = *reinterpret_cast<const f32x4_t*>(q + dim + 4);
        } else {
          x = *reinterpret_cast<const s16x8_t*>(q + dim);
        }
      }
      if (a.negative) {
        if constexpr (__is_same(T, float)) {
          x.v[0] = -x.v[0];
          x.v[1] = -x.v[1];
        } else {
          x ^= (short)0x8000;
        }
      }
      if constexpr (query<T, Q8>::parts == 3) {
        // Cut off, not rounded: eight bits each, and their sum is the query.
        s16x8_t part[3];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const uint32_t u = __float_as_uint(x.v[j >> 2][j & 3]), hi = u & 0xffff0000u;
          // (An infinity less itself would be a NaN: it has no further parts.  A NaN whose first part is cut to
          // an infinity has a quiet one for its second, as any difference with it is.)
          const float rest = (u & 0x7fffffffu) == 0x7f800000u ? 0.0f : __uint_as_float(u) - __uint_as_float(hi);
          const uint32_t mid = __float_as_uint(rest) & 0xffff0000u;
          part[0][j] = (short)(hi >> 16);
          part[1][j] = (short)(mid >> 16);
          part[2][j] = (short)(__float_as_uint(rest - __uint_as_float(mid)) >> 16);
        }
#pragma unroll
        for (int h = 0; h < 3; h++) st.q[t][d][h] = part[h];
      } else {
        st.q[t][d][0] = x;
      }
    }
    st.m[t] = -INFINITY;
    st.l[t] = 0.0f;
    st.base[t] = -kShift<T, Q8>;
    st.most[t] = -1.0f;  // (any sum)
#pragma unroll
    for (int f = 0; f < D / 16; f++) st.o[t][f] = f32x4_t{0, 0, 0, 0};
  }
}

// Which keys of the prefix (own 0) or of their own the wave's pairs see.
template <typename T, bool Q8, int D, int QT>
__device__ __forceinline__ void begin_keys(const sg_attn_shared_args& a, state<T, Q8, D, QT>& st, const sg_attn_job& job,
                                           int pair0, int own, int lane) {
  int all_lo = 0, all_hi = INT32_MAX;
#pragma unroll
  for (int t = 0; t < QT; t++) {
    const int pair = pair0 + t * 16 + (lane & 15);
    const bool in = pair < job.rows * a.group;
    const int r = in ? pair / a.group : 0;
    int lo, hi;
    if (job.kind == kPrefixKeys) {
      const int2 seen = a.seen[job.row0 + r];
      lo = seen.x;
      hi = seen.y;
    } else {
      const int4 seen = sgc::places_seen((int64_t)job.plen + job.len - job.rows + r, job.plen, job.len, a.causal, a.window);
      lo = own ? seen.z : seen.x;
      hi = own ? seen.w : seen.y;
    }
    st.lo[t] = in ? lo : 0;
    st.hi[t] = in ? hi : 0;
    if (in) {
      all_lo = max(all_lo, st.lo[t]);
      all_hi = min(all_hi, st.hi[t]);
    }
  }
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) {  // (lanes 16 apart have the same pairs)
    all_lo = max(all_lo, __shfl_xor(all_lo, o));
    all_hi = min(all_hi, __shfl_xor(all_hi, o));
  }
  st.all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  st.all_hi = __builtin_amdgcn_readfirstlane(all_hi);
}

// What a wave has of a job.  A worker that did the whole of it writes the output, if the job has
// all keys of its rows, or the pairs' own places; otherwise it is the worker's first piece
// (`later`: of a job that another worker began) or its last.
template <typename T, bool Q8, int D, int QT>
__device__ __forceinline__ void end_job(const sg_attn_shared_args& a, const sg_attn_list& list, state<T, Q8, D, QT>& st,
                                        const sg_attn_job& job, int head, int pair0, int in_job, int64_t worker, bool whole,
                                        bool later, int lane) {
  const int g = lane >> 4;
#pragma unroll
  for (int t = 0; t < QT; t++) {
    const float l = kSumByProduct<T, Q8> ? st.l[t] : pair_sum(st.l[t]);
    const int pair = pair0 + t * 16 + (lane & 15);
    if (pair >= job.rows * a.group) continue;
    const int r = pair / a.group, h = head * a.group + pair - r * a.group;
    if (whole && job.kind == kAllKeys) {
      T* out = static_cast<T*>(a.out) + (int64_t)(job.row0 + r) * a.ldo + (int64_t)h * a.hd;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      struct alignas(4 * sizeof(T)) four {
        T v[4];
      };
#pragma unroll
      for (int f = 0; f < D / 16; f++) {
        four y;
#pragma unroll
        for (int i = 0; i < 4; i++) y.v[i] = elem<T>::from(l == 0.0f ? 0.0f : st.o[t][f][i] * inv);
        if (f * 16 + g * 4 < a.hd) *reinterpret_cast<four*>(out + f * 16 + g * 4) = y;
      }
      continue;
    }
    const int64_t at = whole ? ((int64_t)(job.kind == kOwnKeys ? a.rows : 0) + job.row0 + r) * a.heads + h
                             : list.piece0 + (worker * 2 + (later ? 0 : 1)) * list.piece_pairs + in_job + t * 16 + (lane & 15);
    float* o = a.part_o + at * D;
#pragma unroll
    for (int f = 0; f < D / 16; f++) *reinterpret_cast<f32x4_t*>(o + f * 16 + g * 4) = st.o[t][f];
    if (g == 0) a.part_ml[at] = make_float2(st.m[t], l);
  }
}

// A worker's part of a job: units [from, to) of it, all of its tiles if whole.  The list's cost of
// a job (in tiles: queries, first tile, results) stands before its tiles and is no work.
struct part {
  int64_t from, to, all;
  bool whole, later;
  bool work;  // a job that has all keys and no tiles has zeros for its rows
};
__device__ __forceinline__ part part_of(const sg_attn_list& list, const sg_attn_job& job, int64_t at, int64_t left, int64_t c0,
                                        int64_t c1) {
  part p;
  p.all = (int64_t)job.tiles[0] + job.tiles[1];
  p.from = max(at - c0 - list.job_cost, (int64_t)0);
  p.to = max(min(at + left, c1) - c0 - list.job_cost, (int64_t)0);
  p.whole = p.from == 0 && p.to == p.all;
  p.later = p.from > 0;
  p.work = p.from < p.to || (p.all == 0 && job.kind == kAllKeys);
  return p;
}

// Few pairs: every wave is a worker and takes fragments from memory, no barrier anywhere.
template <typename T, bool Q8, int D>
__global__ __launch_bounds__(256, __is_same(T, float) ? 1 : 2) void k_attn_narrow(sg_attn_shared_args a, sg_attn_list list) {
  typedef typename query<T, Q8>::type K;
  typedef typename weight<T, Q8>::type M;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t worker = (int64_t)spread(blockIdx.x, gridDim.x) * 4 + wave;
  share sh = first_share(list, worker, a.kv_heads, lane);
  state<T, Q8, D, 1> st;
  while (sh.left > 0) {
    const int64_t c0 = list.cum[sh.job], c1 = list.cum[sh.job + 1], n = min(c1 - sh.at, sh.left);
    if (n > 0) {
      const sg_attn_job job = list.jobs[sh.job];
      const part pt = part_of(list, job, sh.at, sh.left, c0, c1);
      const int pair0 = job.tile * 16;
      if (pt.work) begin_job(a, st, job, sh.head, pair0, lane);
#pragma unroll 1
      for (int seg = 0; seg < 2; seg++) {
        const int64_t t0 = seg ? job.tiles[0] : 0, u0 = max(pt.from, t0), u1 = min(pt.to, t0 + (seg ? job.tiles[1] : job.tiles[0]));
        if (u0 >= u1) continue;
        begin_keys(a, st, job, pair0, job.kind == kOwnKeys || seg, lane);
        const int64_t tile = (seg ? job.slot_tile[1] : job.slot_tile[0]) + (u0 - t0);
        int first = (int)(tile * kTile - (seg ? job.key0[1] : job.key0[0]));
        const char* at = a.cache + (int64_t)sh.head * a.head_bytes + tile * a.tile_bytes;
        for (int left = (int)(u1 - u0); left > 0; left--, first += kTile, at += a.tile_bytes) {
          const char* vals = at + (int64_t)kTile * D * sizeof(typename sgc::kept<T, Q8>::type);
          const char* tail = at + a.tile_bytes - kTail;
          f32x4_t s[2][1] = {};
          typename frag<M>::type w[1][weight<T, Q8>::parts];
          if constexpr (Q8) {
            constexpr int NU = D / 32;  // kilobytes of the keys, and of the values
            u32x4_t kc[NU], vc[NU];
#pragma unroll
            for (int i = 0; i < NU; i++) kc[i] = *reinterpret_cast<const u32x4_t*>(at + i * 1024 + lane * 16);
#pragma unroll
            for (int i = 0; i < NU; i++) vc[i] = *reinterpret_cast<const u32x4_t*>(vals + i * 1024 + lane * 16);
#pragma unroll
            for (int i = 0; i < NU; i++)
#pragma unroll
              for (int e = 0; e < 2; e++) {
                const int f = i * 2 + e, half = f / (D / 32), d = f % (D / 32);
                const typename frag<K>::type x = decode<K>(kc[i][e * 2], kc[i][e * 2 + 1]);
#pragma unroll
                for (int h = query<T, Q8>::parts - 1; h >= 0; h--) s[half][0] = add_score<K>(x, st.q[0][d][h], s[half][0]);
              }
            weigh<T, Q8, D, 1>(a, st, s, first, reinterpret_cast<const float*>(tail), lane, w);
#pragma unroll
            for (int i = 0; i < NU; i++)
#pragma unroll
              for (int e = 0; e < 2; e++) {
                const typename frag<M>::type x = decode<M>(vc[i][e * 2], vc[i][e * 2 + 1]);
#pragma unroll
                for (int h = weight<T, Q8>::parts - 1; h >= 0; h--) st.o[0][i * 2 + e] = mma(M{}, x, w[0][h], st.o[0][i * 2 + e]);
              }
          } else {
            const bool bad = *reinterpret_cast<const uint32_t*>(tail) != 0;
#pragma unroll
            for (int half = 0; half < 2; half++)
#pragma unroll
              for (int d = 0; d < D / 32; d++)
                s[half][0] = add_score<T>(load_frag<T>(at, half * (D / 32) + d, lane), st.q[0][d][0], s[half][0]);
            weigh<T, Q8, D, 1>(a, st, s, first, nullptr, lane, w);
#pragma unroll
            for (int f = 0; f < D / 16; f++) {
              typename frag<T>::type x = load_frag<T>(vals, f, lane);
              if (bad) x = clean<T>(x);
              st.o[0][f] = mma(M{}, x, w[0][0], st.o[0][f]);
            }
            if (bad) mark_bad(st, first, vals, lane);
          }
        }
      }
      if (pt.work) end_job(a, list, st, job, sh.head, pair0, 0, worker, pt.whole, pt.later, lane);
      sh.left -= n;
      sh.at += n;
    }
    if (++sh.job >= list.plan->jobs) {  // the next head's first job
      sh.job = 0;
      sh.at = 0;
      sh.head++;
    }
  }
}

// Many pairs: a workgroup is a worker, its NW waves have QT * 16 pairs each and share the tiles
// in LDS, two stages.  Types go there by direct copies; codes through registers, and lie there
// as the type that multiplies them.  Codes of up to 128 dims go to LDS as they
// are first, kRing tiles of them, each wave its own part (and the scales): a tile of codes is
// 8 KB, and one or two a CU in flight reach half of the memory's rate (27 rows behind 131072 places: 133 us
// without the ring, 110 with it).  At 256 dims the stages leave no room for it.
constexpr int kRing = 4;
template <typename T, bool Q8, int D, int NW>
struct wide_lds {
  static constexpr int KB = kTile * D * (int)sizeof(typename query<T, Q8>::type);  // keys of a tile
  static constexpr bool ring = Q8 && D <= 128;
  static constexpr int stage = 2 * KB + (Q8 && !ring ? kTail : 0);
  static constexpr int part = D / 16 * 1024 / NW + kTail;  // a wave's part of a tile of codes
  static constexpr int bytes = 2 * stage + (ring ? kRing * NW * part : 0);
};
template <typename T, bool Q8, int D, int QT, int NW, int PER_CU>
__global__ __launch_bounds__(64 * NW, PER_CU * NW / 4) void k_attn_wide(sg_attn_shared_args a, sg_attn_list list) {
  typedef typename query<T, Q8>::type K;
  typedef typename weight<T, Q8>::type M;
  typedef wide_lds<T, Q8, D, NW> L;
  constexpr int KB = L::KB, STAGE = L::stage;
  constexpr bool RING = L::ring;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t worker = spread(blockIdx.x, gridDim.x);
  share sh = first_share(list, worker, a.kv_heads, lane);
  state<T, Q8, D, QT> st;
  while (sh.left > 0) {
    const int64_t c0 = list.cum[sh.job], c1 = list.cum[sh.job + 1], n = min(c1 - sh.at, sh.left);
    if (n > 0) {
      const sg_attn_job job = list.jobs[sh.job];
      const part pt = part_of(list, job, sh.at, sh.left, c0, c1);
      const int in_job = wave * QT * 16, pair0 = job.tile * (16 * NW * QT) + in_job;
      constexpr int NU = Q8 ? D / 16 / NW : 2 * KB / 1024 / NW;  // kilobytes of a tile for each wave
      u32x4_t codes[Q8 ? NU : 1];
      float tail_of = 0.0f;
      uint32_t bad_next = 0;
      const int mine = 2 * STAGE + wave * L::part;  // the wave's part of a ring slot
      auto ring_at = [&](int u) { return mine + u % kRing * (NW * L::part); };
      auto fetch = [&](const char* from, int stage, int u) {
        if constexpr (RING) {
          const i32x4_t rsrc = sg_raw_rsrc(from);
#pragma unroll
          for (int i = 0; i < NU; i++) sg_lds_copy16((uint32_t)(ring_at(u) + i * 1024), lane * 16, rsrc, (wave * NU + i) * 1024);
          sg_lds_copy4((uint32_t)(ring_at(u) + NU * 1024), lane * 4, rsrc, (uint32_t)(2 * kTile * D));
        } else if constexpr (Q8) {
#pragma unroll
          for (int i = 0; i < NU; i++) codes[i] = *reinterpret_cast<const u32x4_t*>(from + (wave * NU + i) * 1024 + lane * 16);
          if (wave == 0) tail_of = *reinterpret_cast<const float*>(from + a.tile_bytes - kTail + lane * 4);
        } else {
          bad_next = *reinterpret_cast<const uint32_t*>(from + a.tile_bytes - kTail);
          const i32x4_t rsrc = sg_raw_rsrc(from);
#pragma unroll
          for (int i = 0; i < NU; i++) {
            const uint32_t u = wave * NU + i;
            sg_lds_copy16((uint32_t)(stage * STAGE + u * 1024), lane * 16, rsrc, u * 1024);
          }
        }
      };
      auto put = [&](int stage, int u, int n) {
        if constexpr (RING) {  // (the two tiles behind it stay in flight)
          if (u + 2 < n) sg_wait_vmcnt<2 * (NU + 1)>();
          else sg_wait_vmcnt<0>();
#pragma unroll
          for (int i = 0; i < NU; i++) codes[i] = *reinterpret_cast<const u32x4_t*>(lds + ring_at(u) + i * 1024 + lane * 16);
        }
        if constexpr (Q8) {
          char* to = lds + stage * STAGE;
#pragma unroll
          for (int i = 0; i < NU; i++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const int k = wave * NU + i, f = k * 2 + e;  // fragment of keys, then of values
              if (k < D / 32) store_frag<K>(to, f, lane, decode<K>(codes[i][e * 2], codes[i][e * 2 + 1]));
              else store_frag<M>(to + KB, f - D / 16, lane, decode<M>(codes[i][e * 2], codes[i][e * 2 + 1]));
            }
          if (!RING && wave == 0) *reinterpret_cast<float*>(to + 2 * KB + lane * 4) = tail_of;
        }
      };
      if (pt.work) begin_job(a, st, job, sh.head, pair0, lane);
#pragma unroll 1
      for (int seg = 0; seg < 2; seg++) {
        const int64_t t0 = seg ? job.tiles[0] : 0, u0 = max(pt.from, t0), u1 = min(pt.to, t0 + (seg ? job.tiles[1] : job.tiles[0]));
        if (u0 >= u1) continue;
        const int64_t tile = (seg ? job.slot_tile[1] : job.slot_tile[0]) + (u0 - t0);
        int first = (int)(tile * kTile - (seg ? job.key0[1] : job.key0[0]));
        const char* at = a.cache + (int64_t)sh.head * a.head_bytes + tile * a.tile_bytes;
        const int tiles = (int)(u1 - u0);
        __syncthreads();  // the stages have been read
        fetch(at, 0, 0);
        if constexpr (RING) {
          if (1 < tiles) fetch(at + a.tile_bytes, 0, 1);
          if (2 < tiles) fetch(at + 2 * a.tile_bytes, 0, 2);
        }
        begin_keys(a, st, job, pair0, job.kind == kOwnKeys || seg, lane);
        put(0, 0, tiles);
        for (int u = 0; u < tiles; u++, first += kTile) {
          const int stage = u & 1;
          if constexpr (!Q8) sg_wait_vmcnt<0>();
          __syncthreads();
          // (Taken here, where nothing is in flight: waiting for it later would wait for the next tile.)
          uint32_t bad = __builtin_amdgcn_readfirstlane(bad_next);
          asm volatile("" : "+s"(bad));
          at += a.tile_bytes;
          if constexpr (RING) {
            if (u + 3 < tiles) fetch(at + 2 * a.tile_bytes, 0, u + 3);
          } else {
            if (u + 1 < tiles) fetch(at, stage ^ 1, u + 1);
          }
          const char* keys = lds + stage * STAGE;
          const char* vals = keys + KB;
          if constexpr (!Q8) {
            if (bad) {  // (alike for the workgroup)
              char* own = lds + stage * STAGE + KB;
              for (int f = wave; f < D / 16; f += NW) store_frag<T>(own, f, lane, clean<T>(load_frag<T>(own, f, lane)));
              __syncthreads();
            }
          }
          // Fragments come from LDS NB at a time, a batch ahead of its products (the first values
          // ahead of the softmax): one by one they would cost their latency each.
          constexpr int NF = D / 16, NB = sizeof(K) == 2 ? 8 : 2, NBATCH = (NF + NB - 1) / NB, N0 = NF < NB ? NF : NB;
          typename frag<K>::type kx[2][N0];
          typename frag<M>::type vx[2][N0];
          auto load_keys = [&](int i) {
#pragma unroll
            for (int e = 0; e < N0; e++) kx[i & 1][e] = load_frag<K>(keys, i * N0 + e, lane);
          };
          auto load_vals = [&](int i) {
#pragma unroll
            for (int e = 0; e < N0; e++) vx[i & 1][e] = load_frag<M>(vals, i * N0 + e, lane);
          };
          f32x4_t s[2][QT] = {};
          load_keys(0);
#pragma unroll
          for (int i = 0; i < NBATCH; i++) {
            if (i + 1 < NBATCH) load_keys(i + 1);
            else load_vals(0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < N0; e++) {
              const int f = i * N0 + e, half = f / (D / 32), d = f % (D / 32);
#pragma unroll
              for (int t = 0; t < QT; t++)
#pragma unroll
                for (int h = query<T, Q8>::parts - 1; h >= 0; h--) s[half][t] = mma(K{}, kx[i & 1][e], st.q[t][d][h], s[half][t]);
            }
          }
          if (RING && u + 1 < tiles) put(stage ^ 1, u + 1, tiles);  // (while the scores come)
          typename frag<M>::type w[QT][weight<T, Q8>::parts];
          weigh<T, Q8, D, QT>(a, st, s, first,
                              reinterpret_cast<const float*>(RING ? lds + ring_at(u) + NU * 1024 : keys + 2 * KB), lane, w);
#pragma unroll
          for (int i = 0; i < NBATCH; i++) {
            if (i + 1 < NBATCH) {
              load_vals(i + 1);
              __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int e = 0; e < N0; e++)
#pragma unroll
              for (int t = 0; t < QT; t++)
#pragma unroll
                for (int h = weight<T, Q8>::parts - 1; h >= 0; h--)
                  st.o[t][i * N0 + e] = mma(M{}, vx[i & 1][e], w[t][h], st.o[t][i * N0 + e]);
          }
          if constexpr (!Q8)
            if (bad) mark_bad(st, first, at - a.tile_bytes + KB, lane);
          if (!RING && u + 1 < tiles) put(stage ^ 1, u + 1, tiles);
        }
      }
      if (pt.work) end_job(a, list, st, job, sh.head, pair0, in_job, worker, pt.whole, pt.later, lane);
      sh.left -= n;
      sh.at += n;
    }
    if (++sh.job >= list.plan->jobs) {
      sh.job = 0;
      sh.at = 0;
      sh.head++;
    }
  }
}

// Waves of a workgroup, pairs of each, workgroups of a CU.  Outputs, queries and two batches of fragments
// fill the registers: 32 pairs a wave up to 128 dims, 16 at 256 or in three parts.  (bf16 over codes at
// 128 dims with eight waves of 16 pairs: 110 us for 107.  256 dims with four waves of 32 pairs, one to a
// SIMD: 40 passages of float32 257 us, with eight of 16 190.)
template <typename T, bool Q8, int D>
struct wide_form {
  static constexpr bool F32 = __is_same(T, float);
  static constexpr int NW = (F32 && Q8 ? D == 128 : D == 256) ? 8 : 4;
  static constexpr int QT = sgk::attn_wide_pairs(D, F32, Q8) / (16 * NW);
  static constexpr int PER_CU = D == 256 || (F32 && D == 128) ? 1 : 2;
};

template <typename T, bool Q8, int D>
hipError_t launch_list(const sg_attn_shared_args& a, const sg_attn_list& list, hipStream_t s) {
  if (!list.wide) return sgp::run_kernel(k_attn_narrow<T, Q8, D>, dim3(list.blocks), dim3(256), 0, s, a, list);
  typedef wide_form<T, Q8, D> W;
  constexpr size_t lds = wide_lds<T, Q8, D, W::NW>::bytes;
  auto kernel = k_attn_wide<T, Q8, D, W::QT, W::NW, W::PER_CU>;
  // More than 64 KB has to be asked for, on every device.
  static std::atomic<uint64_t> asked{0};
  int device = 0;
  hipError_t e = hipGetDevice(&device);
  if (e != hipSuccess) return e;
  if (device >= 64 || !(asked.load(std::memory_order_relaxed) >> device & 1)) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) {
      (void)hipGetLastError();
      return e;
    }
    if (device < 64) asked.fetch_or(uint64_t(1) << device, std::memory_order_relaxed);
  }
  return sgp::run_kernel(kernel, dim3(list.blocks), dim3(64 * W::NW), lds, s, a, list);
}

template <typename T>
hipError_t launch_type(const sg_attn_shared_args& a, const sg_attn_list& list, bool q8, int D, hipStream_t s) {
  if (q8) {
    if (D == 64) return launch_list<T, true, 64>(a, list, s);
    if (D == 128) return launch_list<T, true, 128>(a, list, s);
    return launch_list<T, true, 256>(a, list, s);
  }
  if (D == 64) return launch_list<T, false, 64>(a, list, s);
  if (D == 128) return launch_list<T, false, 128>(a, list, s);
  return launch_list<T, false, 256>(a, list, s);
}

}  // namespace sga
