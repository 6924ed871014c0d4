// k_block_norm.hip -- what stands between two blocks of a layer, one pass over
// the rows:
//   y  = x * rsqrt(mean x^2 + eps) * w_post      (the block's post-norm; y = x without w_post)
//   h' = h + scale * gate * y                    (gate per column, shared or per sequence)
//   xn = h' * rsqrt(mean h'^2 + eps) * w_pre     (the next block's pre-norm)
// Sums and values in float32; h' enters the second norm before it is rounded
// to the tensors' type.
//
// Bound by memory: x and h are read, h' and xn written, once each.  A row stays
// in the registers of the 64, 256 or 512 threads that hold it (four 16-byte
// pieces of each input a thread at most), so neither norm reads it again.  A
// group of threads takes consecutive rows: the norm weights and the gate stay
// in registers from row to row (read again for every row they would be 12 bytes
// of L2 traffic beside a float32 column's 16), and the next row's loads are
// issued before the current row's two reductions.  Measured: 32768 x 768 float32 82
// us, 20001 x 5120 bf16 182 us, 4.9 and 4.5 TB/s of the four tensors (a copy of 1 GB
// moves 5.0); 32 rows 5.7 us, three dependent round trips to memory.
#include <algorithm>

#include "semantica_gpu.h"
#include "sg_kernels.h"
#include "sg_packed.h"

namespace {

static_assert(sgk::kBlockNormCols <= 4 * 256 * 8 && sgk::kBlockNormCols <= 4 * 512 * 4, "longest row in registers");

using sgp::chunk;
using sgp::elem;

// One 16-byte piece at column c of a row; FULL: rows of whole, aligned pieces.
template <typename T, bool FULL>
__device__ __forceinline__ chunk<T> load_piece(const T* row, int c, int cols) {
  constexpr int V = elem<T>::vec;
  chunk<T> r{};
  if constexpr (FULL) {
    if (c < cols) r = *reinterpret_cast<const chunk<T>*>(row + c);
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
      if (c + i < cols) r.v[i] = row[c + i];
  }
  return r;
}

template <typename T, bool FULL>
__device__ __forceinline__ void store_piece(T* row, int c, int cols, const float* f) {
  constexpr int V = elem<T>::vec;
  if constexpr (FULL) {
    if (c < cols) {
      chunk<T> r;
#pragma unroll
      for (int i = 0; i < V; i++) r.v[i] = elem<T>::from(f[i]);
      *reinterpret_cast<chunk<T>*>(row + c) = r;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
      if (c + i < cols) row[c + i] = elem<T>::from(f[i]);
  }
}

__device__ __forceinline__ float weight(const float* w, int c, int cols, float none) {
  return w ? (c < cols ? w[c] : 0.0f) : none;
}

// The sum over a row's TPR threads, the same value in all of them.  The caller
// alternates between two halves of LDS: a half is written again only behind the
// other half's barrier, which no wave passes before it has read this one.
template <int TPR>
__device__ __forceinline__ float row_sum(float a, float* red) {
  a = sgp::wave_sum(a);
  if constexpr (TPR == SG_WAVE) return a;
  constexpr int W = TPR / SG_WAVE;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < W; i++) s += red[i];
  return s;
}

template <typename T, int TPR, int NCH, bool FULL>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_block_norm(sg_block_norm_args a, int rows_each) {
  constexpr int V = elem<T>::vec, NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR;
  __shared__ float red[2][TPR / SG_WAVE];
  const int t = threadIdx.x % TPR, lane = threadIdx.x & 63;
  const int64_t first = ((int64_t)blockIdx.x * RPB + threadIdx.x / TPR) * rows_each;
  // Uniform over the row's threads (and so over the workgroup where they share
  // a barrier).
  const int row0 = (int)min(first, (int64_t)a.rows), row1 = (int)min(first + rows_each, (int64_t)a.rows);
  if (row0 >= row1) return;

  int c[NCH];
#pragma unroll
  for (int k = 0; k < NCH; k++) c[k] = (k * TPR + t) * V;
  float post[NCH][V], pre[NCH][V], gate[NCH][V];
#pragma unroll
  for (int k = 0; k < NCH; k++)
#pragma unroll
    for (int i = 0; i < V; i++) {
      post[k][i] = weight(a.w_post, c[k] + i, a.cols, 1.0f);
      pre[k][i] = weight(a.w_pre, c[k] + i, a.cols, 1.0f);
    }

  const T* x = static_cast<const T*>(a.x);
  const T* h = static_cast<const T*>(a.h);
  chunk<T> xr[NCH], hr[NCH];
  auto load = [&](int row) {
#pragma unroll
    for (int k = 0; k < NCH; k++) {
      xr[k] = load_piece<T, FULL>(x + row * a.ldx, c[k], a.cols);
      hr[k] = load_piece<T, FULL>(h + row * a.ldh, c[k], a.cols);
    }
  };
  load(row0);

  // The sequence of the current row: rows [s0, s1).
  int seq = a.off ? -1 : 0, s0 = a.off ? INT32_MIN : 0, s1 = a.off ? INT32_MIN : a.rows;
  bool fresh = true;  // gate not loaded for this sequence yet
  int half = 0;
  for (int row = row0; row < row1; row++) {
    float xv[NCH][V], hv[NCH][V];
#pragma unroll
    for (int k = 0; k < NCH; k++)
#pragma unroll
      for (int i = 0; i < V; i++) {
        xv[k][i] = elem<T>::to(xr[k].v[i]);
        hv[k][i] = elem<T>::to(hr[k].v[i]);
      }
    if (row + 1 < row1) load(row + 1);
    if (a.off) {
      // The next one, as a rule; else (the first row's, or past empty ones) it is looked up.
      if (row >= s1 && seq + 1 < a.n_seq) {
        fresh = true;
        seq++;
        s0 = a.off[seq];
        s1 = a.off[seq + 1];
        if (row >= s1) {
          seq = max(sgp::find_seq(a.off, a.n_seq, row, lane), 0);
          s0 = a.off[seq];
          s1 = a.off[seq + 1];
        }
      }
      if (row < s0 || row >= s1) continue;  // of no sequence: left as it was
    }
    if (fresh) {
      fresh = false;
      const float* g = a.gate ? a.gate + (int64_t)seq * (a.off ? a.cols : 0) : nullptr;
#pragma unroll
      for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int i = 0; i < V; i++) gate[k][i] = weight(g, c[k] + i, a.cols, 1.0f) * a.scale;
    }
    if (a.w_post) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int i = 0; i < V; i++) s = __builtin_fmaf(xv[k][i], xv[k][i], s);
      const float inv = 1.0f / sqrtf(row_sum<TPR>(s, red[half ^= 1]) / (float)a.cols + a.eps);
#pragma unroll
      for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int i = 0; i < V; i++) xv[k][i] = xv[k][i] * inv * post[k][i];
    }
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < NCH; k++) {
#pragma unroll
      for (int i = 0; i < V; i++) {
        hv[k][i] = __builtin_fmaf(gate[k][i], xv[k][i], hv[k][i]);
        s = __builtin_fmaf(hv[k][i], hv[k][i], s);
      }
      store_piece<T, FULL>(static_cast<T*>(a.sum) + row * a.lds, c[k], a.cols, hv[k]);
    }
    if (a.xn) {
      const float inv = 1.0f / sqrtf(row_sum<TPR>(s, red[half ^= 1]) / (float)a.cols + a.eps);
#pragma unroll
      for (int k = 0; k < NCH; k++) {
#pragma unroll
        for (int i = 0; i < V; i++) hv[k][i] = hv[k][i] * inv * pre[k][i];
        store_piece<T, FULL>(static_cast<T*>(a.xn) + row * a.ldxn, c[k], a.cols, hv[k]);
      }
    }
  }
}

template <typename T, int TPR, int NCH, bool FULL>
hipError_t launch(const sg_block_norm_args& a, hipStream_t s) {
  constexpr int NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR;
  // Rows a group takes one after another: enough groups to fill the GPU first
  // (2048 threads a CU), then longer runs.
  const int64_t groups = 256 * (2048 / NT) * RPB;
  const int each = (int)((a.rows + groups - 1) / groups);
  const int64_t blocks = ((int64_t)a.rows + (int64_t)RPB * each - 1) / ((int64_t)RPB * each);
  return sgp::run_kernel(k_block_norm<T, TPR, NCH, FULL>, dim3((unsigned)blocks), dim3(NT), 0, s, a, each);
}

template <typename T, int TPR, bool FULL>
hipError_t by_pieces(const sg_block_norm_args& a, int n, hipStream_t s) {
  if (n <= 1) return launch<T, TPR, 1, FULL>(a, s);
  if (n == 2) return launch<T, TPR, 2, FULL>(a, s);
  if (n == 3) return launch<T, TPR, 3, FULL>(a, s);
  return launch<T, TPR, 4, FULL>(a, s);
}

template <typename T, bool FULL>
hipError_t by_threads(const sg_block_norm_args& a, hipStream_t s) {
  constexpr int V = elem<T>::vec;
  const int pieces = (a.cols + V - 1) / V;
  if (pieces <= 4 * 64) return by_pieces<T, 64, FULL>(a, (pieces + 63) / 64, s);
  if constexpr (V == 4) {  // (kBlockNormCols 16-bit values are four pieces of 256 threads)
    if (pieces > 4 * 256) return by_pieces<T, 512, FULL>(a, (pieces + 511) / 512, s);
  }
  return by_pieces<T, 256, FULL>(a, (pieces + 255) / 256, s);
}

template <typename T>
hipError_t by_type(const sg_block_norm_args& a, hipStream_t s) {
  constexpr int V = elem<T>::vec;
  auto whole = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % V == 0; };
  const bool full = a.cols % V == 0 && whole(a.x, a.ldx) && whole(a.h, a.ldh) && whole(a.sum, a.lds) &&
                    (!a.xn || whole(a.xn, a.ldxn));
  return full ? by_threads<T, true>(a, s) : by_threads<T, false>(a, s);
}

}  // namespace

namespace sgk {

hipError_t block_norm(const sg_block_norm_args& a, int dtype, hipStream_t s) {
  if (dtype == SG_F32) return by_type<float>(a, s);
  if (dtype == SG_F16) return by_type<_Float16>(a, s);
  return by_type<sgp::bf16_t>(a, s);
}

}  // namespace sgk
