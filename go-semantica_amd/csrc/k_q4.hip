// k_q4.hip -- packing of 4-bit weights (sg_q4_weight_create) into the order of sg_q4.h.
#include <algorithm>

#include "sg_q4.h"

namespace {

using sgp::bf16_t;
using sgp::elem;
using sgq::kBlockK;
using sgq::kWaves;

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

}  // namespace

namespace sgk {

int64_t q4_blocks(int out_dim, int in_dim) { return (int64_t)((out_dim + 15) / 16) * ((in_dim + kBlockK - 1) / kBlockK); }

int64_t q4_threads(int rows, int out_dim) {
  // No form has workgroups of less than 16 outputs and 16 rows.
  return (int64_t)((out_dim + 15) / 16) * (((int64_t)rows + 15) / 16) * 64 * kWaves;
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
  if (dtype == SG_F32) return matmul_q4_f32(a, s);
  if (dtype == SG_F16) return matmul_q4_f16(a, s);
  return matmul_q4_bf16(a, s);
}

}  // namespace sgk
