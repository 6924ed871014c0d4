// k_q4.hip -- a few rows times a matrix of 4-bit weights with group scales (sg_matmul_q4):
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
// block, and are joined through LDS.
#include <algorithm>

#include "semantica_gpu.h"
#include "sg_kernels.h"
#include "sg_packed.h"

namespace {

using sgp::bf16_t;
using sgp::elem;

typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

constexpr int kBlockK = 128, kWaves = 8;

// ---- packing ----------------------------------------------------------------------

// Code and scale sources: plain arrays, or GGUF's Q4_0 blocks (a half and 16 bytes: the lower
// nibbles are the block's first 16 inputs, the upper ones the others).
struct plain_src {
  const uint8_t* codes;
  const void* scales;
  const uint8_t* zeros;
  int scale_dtype, in, groups, group;
  __device__ int code(int n, int k) const { return codes[(int64_t)n * (in / 2) + k / 2] >> (k & 1) * 4 & 15; }
  __device__ int zero(int n, int g) const { return zeros ? zeros[(int64_t)n * groups + g] & 15 : 8; }
  __device__ float scale(int n, int g) const {
    const int64_t at = (int64_t)n * groups + g;
    if (scale_dtype == SG_F32) return static_cast<const float*>(scales)[at];
    if (scale_dtype == SG_F16) return (float)static_cast<const _Float16*>(scales)[at];
    return elem<bf16_t>::to(static_cast<const bf16_t*>(scales)[at]);
  }
};
struct q4_0_src {
  const uint8_t* raw;
  int groups, group;
  __device__ const uint8_t* block(int n, int g) const { return raw + ((int64_t)n * groups + g) * 18; }
  __device__ int code(int n, int k) const {
    const uint8_t b = block(n, k / 32)[2 + k % 16];
    return k % 32 < 16 ? b & 15 : b >> 4;
  }
  __device__ int zero(int, int) const { return 8; }
  __device__ float scale(int n, int g) const {
    const uint8_t* b = block(n, g);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(b[0] | b[1] << 8));
  }
};

template <typename S>
__global__ __launch_bounds__(256) void k_q4_pack(S src, int out_dim, int in_dim, int64_t blocks, uint32_t* w, void* scales,
                                                 int scales_f32, uint8_t* zeros) {
  const int kb = (in_dim + kBlockK - 1) / kBlockK, per = kBlockK / src.group;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < blocks * 256; i += (int64_t)gridDim.x * 256) {
    const int64_t block = i >> 8;
    const int lane = (int)(i >> 2) & 63, sub = (int)i & 3, tile = (int)(block / kb), b = (int)(block % kb);
    const int n = tile * 16 + (lane & 15), k0 = b * kBlockK + sub * 32 + (lane >> 4) * 8;
    uint32_t word = 0;
    for (int j = 0; j < 8; j++) {
      const int k = k0 + j;
      const int c = n < out_dim && k < in_dim ? src.code(n, k) : 0;
      word |= (uint32_t)c << ((j >> 1) * 4 + (j & 1) * 16);
    }
    w[i] = word;
    // The block's scales [lane / 16][group of the block][4 outputs], zeros [output][group].
    if ((int)(i & 255) < 16 * per) {
      const int e = (int)(i & 255), q = e / (per * 4), s = e / 4 % per, o = tile * 16 + q * 4 + e % 4, g = b * per + s;
      const bool in = o < out_dim && g * src.group < in_dim;
      const float v = in ? src.scale(o, g) : 0.0f;
      const int64_t at = block * 16 * per + e;
      if (scales_f32) static_cast<float*>(scales)[at] = v;
      else static_cast<_Float16*>(scales)[at] = (_Float16)v;
      if (zeros) {
        const int zo = tile * 16 + e / per, zg = b * per + e % per;
        zeros[at] = zo < out_dim && zg * src.group < in_dim ? (uint8_t)src.zero(zo, zg) : 0;
      }
    }
  }
}

// ---- products ---------------------------------------------------------------------

// Eight codes less their zero, as fp16 or bf16.
template <typename M>
__device__ __forceinline__ s16x8_t decode(uint32_t w, float zero) {
  u32x4_t x;
  if constexpr (__is_same(M, _Float16)) {
    // 0x6400 + c is fp16's 1024 + c.
    const _Float16 z = (_Float16)(1024.0f + zero);
    const half2_t off = {z, z};
#pragma unroll
    for (int i = 0; i < 4; i++)
      x[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, (w >> (4 * i) & 0x000f000fu) | 0x64006400u) - off);
  } else {
    // A whole number below 2^8 is a bf16 in its float's upper half.
    const uint32_t even = w & 0x0f0f0f0fu, odd = w >> 4 & 0x0f0f0f0fu;  // nibbles 0 2 4 6, 1 3 5 7
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t from = i & 1 ? odd : even;
      const float a = (float)(from >> (i >> 1) * 8 & 0xff) - zero, b = (float)(from >> (16 + (i >> 1) * 8) & 0xff) - zero;
      x[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    }
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
        // (An infinity less itself would be a NaN: it has no further parts.)
        const float rest = (x & 0x7f800000u) == 0x7f800000u ? 0.0f : __uint_as_float(x) - __uint_as_float(hi[e]);
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

template <typename T, int GROUP, int OT, int MT>
__global__ __launch_bounds__(64 * kWaves) void k_q4(sg_q4_args a) {
  typedef typename mul<T>::type M;
  constexpr int PER = kBlockK / GROUP;  // groups of a block
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
    x[m] = static_cast<const T*>(a.x) + (there[m] ? row : 0) * a.ldx;
  }
  for (int b = wave; b < kb; b += kWaves) {
    u32x4_t w[OT];
    f32x4_t scale[OT][PER];
    float zero[OT][PER];
#pragma unroll
    for (int o = 0; o < OT; o++) {
      const int64_t block = (int64_t)min(tile0 + o, tiles - 1) * kb + b;
      w[o] = *reinterpret_cast<const u32x4_t*>(a.w + block * 256 + lane * 4);
#pragma unroll
      for (int s = 0; s < PER; s++) {
        const int64_t at = block * (16 * PER) + (g * PER + s) * 4;
        if (a.scales_f32) {
          scale[o][s] = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(a.scales) + at);
        } else {
          const half4_t h = *reinterpret_cast<const half4_t*>(static_cast<const _Float16*>(a.scales) + at);
          scale[o][s] = f32x4_t{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
        }
        zero[o][s] = a.zeros ? (float)a.zeros[block * (16 * PER) + (lane & 15) * PER + s] : 8.0f;
      }
    }
    raw8<T> r[MT][4];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int s = 0; s < 4; s++) {
        const int k = b * kBlockK + s * 32 + g * 8;
        const bool in = there[m] && k < a.in_dim;
#pragma unroll
        for (int e = 0; e < (int)sizeof(T) / 2; e++)
          r[m][s].v[e] = in ? *reinterpret_cast<const u32x4_t*>(x[m] + k + e * 4) : u32x4_t{0, 0, 0, 0};
      }
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
          const s16x8_t c = decode<M>(w[o][s], zero[o][s0]);
#pragma unroll
          for (int m = 0; m < MT; m++)
#pragma unroll
            for (int e = 0; e < mul<T>::parts; e++) sum[o][m] = mma(M{}, c, p[m][e], sum[o][m]);
        }
      }
#pragma unroll
      for (int o = 0; o < OT; o++)
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int i = 0; i < 4; i++) acc[o][m][i] = __builtin_fmaf(scale[o][s0][i], sum[o][m][i], acc[o][m][i]);
    }
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

template <typename T, int GROUP, int OT, int MT>
hipError_t launch(const sg_q4_args& a, hipStream_t s) {
  const int64_t tiles = (a.out_dim + 15) / 16, blocks = (tiles + OT - 1) / OT * (((int64_t)a.rows + MT * 16 - 1) / (MT * 16));
  return sgp::run_kernel(k_q4<T, GROUP, OT, MT>, dim3((unsigned)blocks), dim3(64 * kWaves), 0, s, a);
}

template <typename T, int GROUP>
hipError_t by_rows(const sg_q4_args& a, hipStream_t s) {
  const int tiles = (a.out_dim + 15) / 16;
  if (a.rows > 32) return launch<T, GROUP, 2, 4>(a, s);
  if (a.rows > 16) return launch<T, GROUP, 2, 2>(a, s);
  if (a.rows > 2 && tiles >= 1024) return launch<T, GROUP, 4, 1>(a, s);
  return launch<T, GROUP, 1, 1>(a, s);
}

template <typename T>
hipError_t by_group(const sg_q4_args& a, hipStream_t s) {
  if (a.group == 32) return by_rows<T, 32>(a, s);
  if (a.group == 64) return by_rows<T, 64>(a, s);
  return by_rows<T, 128>(a, s);
}

}  // namespace

namespace sgk {

int64_t q4_blocks(int out_dim, int in_dim) { return (int64_t)((out_dim + 15) / 16) * ((in_dim + kBlockK - 1) / kBlockK); }

int64_t q4_threads(int rows, int out_dim) {
  // The most that any form launches: 16 outputs and 16 rows to a workgroup up to 16 rows, 32 and 32 or 64 above.
  const int64_t tiles = (out_dim + 15) / 16;
  return (rows > 16 ? (tiles + 1) / 2 * (((int64_t)rows + 31) / 32) : tiles) * 64 * kWaves;
}

hipError_t q4_pack(const uint8_t* codes, const void* scales, int scale_dtype, const uint8_t* zeros, int out_dim, int in_dim,
                   int group, uint32_t* w, void* packed_scales, uint8_t* packed_zeros, hipStream_t s) {
  const int64_t blocks = q4_blocks(out_dim, in_dim);
  const plain_src src{codes, scales, zeros, scale_dtype, in_dim, in_dim / group, group};
  return sgp::run_kernel(k_q4_pack<plain_src>, dim3((unsigned)std::min<int64_t>(blocks, 1 << 16)), dim3(256), 0, s, src, out_dim,
                         in_dim, blocks, w, packed_scales, scale_dtype != SG_F16, packed_zeros);
}

hipError_t q4_pack_q4_0(const uint8_t* raw, int out_dim, int in_dim, uint32_t* w, void* packed_scales, hipStream_t s) {
  const int64_t blocks = q4_blocks(out_dim, in_dim);
  const q4_0_src src{raw, in_dim / 32, 32};
  return sgp::run_kernel(k_q4_pack<q4_0_src>, dim3((unsigned)std::min<int64_t>(blocks, 1 << 16)), dim3(256), 0, s, src, out_dim,
                         in_dim, blocks, w, packed_scales, 0, nullptr);
}

hipError_t matmul_q4(const sg_q4_args& a, int dtype, hipStream_t s) {
  if (dtype == SG_F32) return by_group<float>(a, s);
  if (dtype == SG_F16) return by_group<_Float16>(a, s);
  return by_group<bf16_t>(a, s);
}

}  // namespace sgk
