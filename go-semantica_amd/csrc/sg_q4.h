// sg_q4.h -- a few rows times a matrix of 4-bit weights with group scales (sg_matmul_q4): the
// kernels, shared by the files that instantiate them.
//   y[m][n] = sum over groups g of scale[n][g] * sum over k in g of (code[n][k] - zero[n][g]) x[m][k]
//
// Codes less their zeros are whole numbers of -15 .. 15, exact in any type, so the inner sum is
// one matrix product of the codes as they are and its result is scaled in float32: weights are
// never rounded.  fp16 and bf16 rows multiply as they are; float32 rows as three bf16 parts of
// eight bits each, cut off and not rounded, whose sum is x, bit for bit.
//
// Packed weights, 16 outputs and 128 inputs to a block of a kilobyte: a lane's 16 bytes are its
// eight inputs (lane / 16) of each of four products of 32, for output lane % 16, so a wave
// moves a block with one load and shuffles nothing.  Within eight, even inputs lie in the lower
// half of the word and odd ones in the upper: masks give pairs.  Scales follow in the order
// in which lanes hold a product's results.
//
// A workgroup has OT * 16 outputs and MT * 16 rows; its eight waves split the inputs, block by
// block, and are joined through LDS (four waves read too little ahead, sixteen have too few registers:
// both slower).  Few rows: the weights' bytes bound it, 8192 x 8192 and one fp16 row 14.4 us, 2.6 TB/s,
// out of memory (16 such weights in turn; 10 us, 3.8 TB/s, where the 256 MB cache behind the L2s holds
// them); 16 bf16 rows of 4096 to 16384 with zeros 14.9 and 12.9 us, 2.4 and 2.8 TB/s: two dozen vector
// instructions decode a lane's eight codes of a product.  One float32 row of 768 to 2304: 4 us, a chain of
// two loads, the products and the join.
// Many rows: weights are decoded again for every 16 or 32 of them, so that a dense bf16 product of
// the same size takes over (4096 to 8192, groups of 32, 128, dense: 32 rows 13.5, 12.6 and 15 us, 64 23.9,
// 16.1 and 16.2, 512 171, 107 and 37).
#pragma once
#include "semantica_gpu.h"
#include "sg_kernels.h"
#include "sg_packed.h"

namespace sgq {

using sgp::bf16_t;
using sgp::elem;

typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

constexpr int kBlockK = 128, kWaves = 8;

// Eight codes less their zero, as fp16 or bf16.
template <typename M>
struct offset;  // a group's zero, as decode takes it off
template <>
struct offset<_Float16> {
  half2_t v;
  __device__ explicit offset(int zero) {
    const _Float16 z = (_Float16)(float)(1024 + zero);
    v = half2_t{z, z};
  }
};
template <>
struct offset<bf16_t> {
  float v;
  __device__ explicit offset(int zero) : v((float)zero) {}
};
__device__ __forceinline__ s16x8_t decode(uint32_t w, const offset<_Float16>& zero) {
  // 0x6400 + c is fp16's 1024 + c.
  u32x4_t x;
#pragma unroll
  for (int i = 0; i < 4; i++)
    x[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, (w >> (4 * i) & 0x000f000fu) | 0x64006400u) - zero.v);
  return __builtin_bit_cast(s16x8_t, x);
}
__device__ __forceinline__ s16x8_t decode(uint32_t w, const offset<bf16_t>& zero) {
  // A whole number below 2^8 is a bf16 in its float's upper half.
  const uint32_t even = w & 0x0f0f0f0fu, odd = w >> 4 & 0x0f0f0f0fu;  // nibbles 0 2 4 6, 1 3 5 7
  u32x4_t x;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t from = i & 1 ? odd : even;
    const float a = (float)(from >> (i >> 1) * 8 & 0xff) - zero.v, b = (float)(from >> (16 + (i >> 1) * 8) & 0xff) - zero.v;
    x[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  }
  return __builtin_bit_cast(s16x8_t, x);
}

__device__ __forceinline__ f32x4_t mma(_Float16, s16x8_t a, s16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mma(bf16_t, s16x8_t a, s16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(sgp::bf16x8_t, a), __builtin_bit_cast(sgp::bf16x8_t, b), c,
                                                 0, 0, 0);
}

// How rows of T are multiplied: type and parts.
template <typename T>
struct mul {
  typedef T type;
  static constexpr int parts = 1;
};
template <>
struct mul<float> {
  typedef bf16_t type;
  static constexpr int parts = 3;
};

// Eight inputs of a row: one 16-bit piece, or two of float32.
template <typename T>
struct raw8 {
  u32x4_t v[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ void split(const raw8<T>& r, s16x8_t (&p)[mul<T>::parts]) {
  if constexpr (mul<T>::parts == 1) {
    p[0] = __builtin_bit_cast(s16x8_t, r.v[0]);
  } else {
    u32x4_t a, b, c;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      uint32_t hi[2], mid[2], lo[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const uint32_t x = r.v[(2 * i + e) >> 2][(2 * i + e) & 3];
        hi[e] = x & 0xffff0000u;
        // (An infinity less itself would be a NaN: it has no further parts.  A NaN whose first part is cut to
        // an infinity has a quiet one for its second, as any difference with it is.)
        const float rest = (x & 0x7fffffffu) == 0x7f800000u ? 0.0f : __uint_as_float(x) - __uint_as_float(hi[e]);
        mid[e] = __float_as_uint(rest) & 0xffff0000u;
        lo[e] = __float_as_uint(rest - __uint_as_float(mid[e]));
      }
      a[i] = __builtin_amdgcn_perm(hi[1], hi[0], 0x07060302u);
      b[i] = __builtin_amdgcn_perm(mid[1], mid[0], 0x07060302u);
      c[i] = __builtin_amdgcn_perm(lo[1], lo[0], 0x07060302u);
    }
    p[0] = __builtin_bit_cast(s16x8_t, c);  // the smallest first
    p[1] = __builtin_bit_cast(s16x8_t, b);
    p[2] = __builtin_bit_cast(s16x8_t, a);
  }
}

// The scales of a lane's four results, of each of the block's groups.
template <typename S, int PER>
struct alignas(PER * 4 * sizeof(S) < 16 ? 8 : 16) four {
  S v[PER][4];
};

// What a wave loads of a block, as it lies in memory.
template <typename S, int PER, int OT>
struct loaded {
  u32x4_t w[OT];
  four<S, PER> scale[OT];
  uint32_t zero[OT];  // a byte for each group
};

template <typename T, typename S, bool ZEROS, int GROUP, int OT, int MT>
__global__ __launch_bounds__(64 * kWaves) void k_q4(sg_q4_args a) {
  typedef typename mul<T>::type M;
  constexpr int PER = kBlockK / GROUP;  // groups of a block
  typedef loaded<S, PER, OT> L;
  __shared__ f32x4_t red[kWaves][OT * MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  const int tiles = (a.out_dim + 15) / 16, kb = (a.in_dim + kBlockK - 1) / kBlockK;
  const int groups_of_tiles = (tiles + OT - 1) / OT;
  const int tile0 = (int)(blockIdx.x % groups_of_tiles) * OT;
  const int64_t row0 = (int64_t)(blockIdx.x / groups_of_tiles) * (MT * 16);
  f32x4_t acc[OT][MT] = {};
  const T* x[MT];
  bool there[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    const int64_t row = row0 + m * 16 + (lane & 15);
    there[m] = row < a.rows;
    x[m] = static_cast<const T*>(a.x) + (there[m] ? row : 0) * a.ldx + g * 8;
  }
  auto load = [&](int b, L& l) {
#pragma unroll
    for (int o = 0; o < OT; o++) {
      const int64_t block = (int64_t)min(tile0 + o, tiles - 1) * kb + b;
      l.w[o] = *reinterpret_cast<const u32x4_t*>(a.w + block * 256 + lane * 4);
      l.scale[o] = *reinterpret_cast<const four<S, PER>*>(static_cast<const S*>(a.scales) + block * (16 * PER) + g * PER * 4);
      if constexpr (ZEROS) {
        const uint8_t* z = a.zeros + block * (16 * PER) + (lane & 15) * PER;
        if constexpr (PER == 4) l.zero[o] = *reinterpret_cast<const uint32_t*>(z);
        if constexpr (PER == 2) l.zero[o] = *reinterpret_cast<const uint16_t*>(z);
        if constexpr (PER == 1) l.zero[o] = *z;
      }
    }
  };
  raw8<T> r[MT][4];
  // (A lane of no row holds anything: its column of the product is no one's.)
  auto load_rows = [&](int b, int s) {
    const int k = b * kBlockK + s * 32;
#pragma unroll
    for (int m = 0; m < MT; m++)
      if (there[m])
#pragma unroll
        for (int e = 0; e < (int)sizeof(T) / 2; e++)
          r[m][s].v[e] = k < a.in_dim ? *reinterpret_cast<const u32x4_t*>(x[m] + k + e * (16 / (int)sizeof(T))) : u32x4_t{0, 0, 0, 0};
  };
  // The next block's weights are on their way while a block is multiplied, and its rows from the
  // moment that a product has taken this one's.
  L l, next;
  if (wave < kb) {
    load(wave, l);
#pragma unroll
    for (int s = 0; s < 4; s++) load_rows(wave, s);
  }
  for (int b = wave; b < kb; b += kWaves) {
    const bool more = b + kWaves < kb;
    if (more) load(b + kWaves, next);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s0 = 0; s0 < PER; s0++) {
      f32x4_t sum[OT][MT] = {};
#pragma unroll
      for (int i = 0; i < 4 / PER; i++) {
        const int s = s0 * (4 / PER) + i;
        s16x8_t p[MT][mul<T>::parts];
#pragma unroll
        for (int m = 0; m < MT; m++) split<T>(r[m][s], p[m]);
#pragma unroll
        for (int o = 0; o < OT; o++) {
          const s16x8_t c = decode(l.w[o][s], offset<M>(ZEROS ? (int)(l.zero[o] >> s0 * 8 & 0xff) : 8));
#pragma unroll
          for (int m = 0; m < MT; m++)
#pragma unroll
            for (int e = 0; e < mul<T>::parts; e++) sum[o][m] = mma(M{}, c, p[m][e], sum[o][m]);
        }
        if (more) load_rows(b + kWaves, s);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int o = 0; o < OT; o++)
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int i = 0; i < 4; i++) acc[o][m][i] = __builtin_fmaf((float)l.scale[o].v[s0][i], sum[o][m][i], acc[o][m][i]);
      __builtin_amdgcn_sched_barrier(0);
    }
    l = next;
  }
#pragma unroll
  for (int o = 0; o < OT; o++)
#pragma unroll
    for (int m = 0; m < MT; m++) red[wave][o * MT + m][lane] = acc[o][m];
  __syncthreads();
  for (int i = threadIdx.x; i < OT * MT * 64; i += 64 * kWaves) {
    f32x4_t v = red[0][i >> 6][i & 63];
#pragma unroll
    for (int q = 1; q < kWaves; q++) v += red[q][i >> 6][i & 63];
    const int o = (i >> 6) / MT, m = (i >> 6) % MT;
    const int64_t row = row0 + m * 16 + (i & 15);
    const int n = (tile0 + o) * 16 + ((i >> 4) & 3) * 4;
    if (row >= a.rows) continue;
    T* dst = static_cast<T*>(a.dst) + row * a.ldd + n;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (n + e < a.out_dim) dst[e] = elem<T>::from(v[e]);
  }
}

template <typename T, typename S, bool ZEROS, int GROUP, int OT, int MT>
hipError_t launch(const sg_q4_args& a, hipStream_t s) {
  const int64_t tiles = (a.out_dim + 15) / 16, blocks = (tiles + OT - 1) / OT * (((int64_t)a.rows + MT * 16 - 1) / (MT * 16));
  return sgp::run_kernel(k_q4<T, S, ZEROS, GROUP, OT, MT>, dim3((unsigned)blocks), dim3(64 * kWaves), 0, s, a);
}

// More outputs and rows to a workgroup as there are more blocks of 16 and 16 than fill the GPU: what
// is loaded or decoded once then serves several products.  Measured with 4096 inputs (us; OT x MT, fp16
// scales; * is taken):
//   bf16, group 64    512 blocks   1x1 11.4  2x1 9.4*            (16 rows; 1 row 8.4* and 8.9)
//                    1024, 16 rows 1x1 19.9  2x1 14.7  4x1 14.5*  (1 row, group 32: 15.2  14.3*  15.0)
//                    1024, 64 rows           2x1 13.8  4x1 12.9  2x2 11.5*  4x2 15.2
//                    2048, 64 rows 1x1 35    2x1 24    4x1 24    2x2 21     4x2 15.8*
//   group 32, 2048, 64 rows 1x1 37  2x1 26  4x1 26  2x2 23.5*  4x2 31
//   float32, group 64, 512 blocks  1x1 20.4  2x1 13.9*
//                    2048, 64 rows 1x1 64    2x1 39    4x1 33*   2x2 40     4x2 34
//   float32, group 128, 2048, 64 rows        2x1 40    4x1 34    2x2 40     4x2 26*
template <typename T, typename S, bool ZEROS, int GROUP>
hipError_t by_size(const sg_q4_args& a, hipStream_t s) {
  const int64_t tiles = (a.out_dim + 15) / 16, blocks = tiles * ((a.rows + 15) / 16);
  if (tiles >= 16) {  // (a workgroup's last outputs may be none)
    // (With shorter groups its scales and sums are more than registers hold.)
    if constexpr (GROUP > (sizeof(T) == 2 ? 32 : 64))
      if (a.rows > 16 && blocks >= 2048) return launch<T, S, ZEROS, GROUP, 4, 2>(a, s);
    if constexpr (sizeof(T) == 2) {
      if (a.rows > 16 && blocks >= 1024) return launch<T, S, ZEROS, GROUP, 2, 2>(a, s);
      if (a.rows > 2 && blocks >= 1024) return launch<T, S, ZEROS, GROUP, 4, 1>(a, s);
      if (blocks >= (a.rows > 2 ? 512 : 1024)) return launch<T, S, ZEROS, GROUP, 2, 1>(a, s);
    } else {
      if (blocks >= 1024) return launch<T, S, ZEROS, GROUP, 4, 1>(a, s);
      if (blocks >= 512) return launch<T, S, ZEROS, GROUP, 2, 1>(a, s);
    }
  }
  return launch<T, S, ZEROS, GROUP, 1, 1>(a, s);
}

template <typename T, typename S, bool ZEROS>
hipError_t by_group(const sg_q4_args& a, hipStream_t s) {
  if (a.group == 32) return by_size<T, S, ZEROS, 32>(a, s);
  if (a.group == 64) return by_size<T, S, ZEROS, 64>(a, s);
  return by_size<T, S, ZEROS, 128>(a, s);
}

template <typename T>
hipError_t by_weight(const sg_q4_args& a, hipStream_t s) {
  if (a.scales_f32) return a.zeros ? by_group<T, float, true>(a, s) : by_group<T, float, false>(a, s);
  return a.zeros ? by_group<T, _Float16, true>(a, s) : by_group<T, _Float16, false>(a, s);
}

}  // namespace sgq
