// k_adapters.hip -- low-rank adapters of many requests beside one shared
// projection: dst_t = base_t + scale_a * B_a (A_a x_t), a the adapter of the
// sequence that holds row t (none: dst_t = base_t).
//
// Two launches.  "Down" forms u = A_a x (rank values a row, float32) and "up"
// adds scale_a * B_a u to the base.  One launch that did both would read every
// adapter of its rows once for each slice of output columns, and a batch of
// single tokens with an adapter each needs many slices to fill the GPU; the
// detour of u through memory is rank * 8 bytes a row.  Down's sum over in_dim is
// split over up to kMostSplit workgroups where the rows alone are too few, up
// adds the parts in order, so a call gives the same bits every time.
//
// Rows of different adapters share a tile of 16: a workgroup takes its tile's
// distinct adapters one by one, multiplies the whole tile and keeps the rows
// that are that adapter's.  A tile of one sequence, the common case, takes one
// turn; sixteen single tokens take sixteen, each with the 16-row product that a
// single row needs as well (the matrix core's rows are free, the adapters'
// weights are what such a batch has to read).
//
// Operands.  Weights are laid out once in fragment order, a wave's load being one
// contiguous kilobyte:
//   A  [adapter][rank / 16][in_dim step][64 lanes x 16 bytes]: lane (m, g) holds
//      rank 16 rb + m, the step's elements g * V .. + V - 1 (V elements of 16
//      bytes; a step is 4 V of them);
//   B  [adapter][32-column pair][2][rank / 16][lanes x 16 bytes]: block j of a
//      pair holds in its row m = 4 g + i column 32 p + 8 g + 4 j + i, so that the
//      two blocks leave a lane with eight columns side by side: 16-byte loads
//      and stores of base and dst.
// 16-bit types multiply on v_mfma_f32_16x16x32: down a step each; up takes
// 16 ranks as its 32, u's upper bf16 (fp16) half against B and the rest that
// the half leaves against the same B, so u is not rounded to 8 (11) bits between
// the products, at no cost (the unpadded rank of most adapters is 16).  float32
// multiplies on v_mfma_f32_16x16x4_f32, four of them a 16-byte piece.
#include <algorithm>

#include "semantica_gpu.h"
#include "sg_kernels.h"
#include "sg_packed.h"

namespace {

using sgp::bf16_t;
using sgp::chunk;
using sgp::elem;

constexpr int kWaves = 4, kNT = kWaves * SG_WAVE;
constexpr int kTile = 16;       // rows of a matrix core tile
constexpr int kMostSplit = 16;  // parts of down's sum
constexpr int kCus = 256;

template <typename T>
constexpr int step_of() { return 4 * elem<T>::vec; }  // in_dim elements a step

template <typename T>
__device__ __forceinline__ f32x4_t mfma(const chunk<T>& a, const chunk<T>& b, f32x4_t c);
template <>
__device__ __forceinline__ f32x4_t mfma<_Float16>(const chunk<_Float16>& a, const chunk<_Float16>& b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4_t mfma<bf16_t>(const chunk<bf16_t>& a, const chunk<bf16_t>& b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(sgp::bf16x8_t, a), __builtin_bit_cast(sgp::bf16x8_t, b),
                                                 c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4_t mfma<float>(const chunk<float>& a, const chunk<float>& b, f32x4_t c) {
#pragma unroll
  for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c, 0, 0, 0);
  return c;
}

// The adapters of a workgroup's ROWS rows: own[r] in LDS (kNone: its sequence has
// none; kNoRow: a row of no sequence, which is left as it was), and their distinct
// ids in rising order of first row.
constexpr int kNone = -1, kNoRow = -2;
template <int ROWS>
struct tile_ids {
  int own[ROWS], list[ROWS], count;
};

template <int ROWS>
__device__ __forceinline__ void find_ids(const sg_adapters_args& a, int row0, tile_ids<ROWS>& t, int tid) {
  static_assert(ROWS <= SG_WAVE, "a lane per row");
  if (tid < SG_WAVE) {
    const int lane = tid, last = min(row0 + ROWS, a.rows) - 1;
    const int i0 = sgp::find_seq(a.off, a.n_seq, row0, lane), i1 = sgp::find_seq(a.off, a.n_seq, last, lane);
    const int row = min(row0 + lane, last);
    int lo = max(i0, 0), hi = max(i1, lo);  // the row's sequence lies between the first and the last row's
    while (lo < hi) {
      const int mid = lo + (hi - lo + 1) / 2;
      if (a.off[mid] <= row) lo = mid;
      else hi = mid - 1;
    }
    int id = kNoRow;
    if (lane < ROWS && row0 + lane <= last && a.off[lo] <= row && row < a.off[lo + 1]) {
      id = a.ids[lo];
      if (id < 0 || id >= a.n_adapters) id = kNone;
    }
    if (lane < ROWS) t.own[lane] = id;
    int n = 0;
    uint64_t left = __ballot(id >= 0);
    while (left) {
      const int pick = __builtin_amdgcn_readfirstlane(__shfl(id, __builtin_ctzll(left)));
      if (lane == 0) t.list[n] = pick;
      n++;
      left &= ~__ballot(id == pick);
    }
    if (lane == 0) t.count = n;
  }
  __syncthreads();
}

// ---- down: u[part][row][rank] ------------------------------------------------
// A workgroup: RT tiles of 16 rows, one part of in_dim, NRB blocks of 16 ranks.
// Its four waves take a quarter of the part's steps each and add up through LDS.
template <typename T, int RT, int NRB>
__global__ __launch_bounds__(kNT) void k_adapter_down(sg_adapters_args a, int parts, int steps_each) {
  constexpr int V = elem<T>::vec, STEP = step_of<T>(), ROWS = RT * kTile;
  __shared__ tile_ids<ROWS> ids;
  __shared__ float sums[kWaves][ROWS][NRB * 16 + 4];  // + 4: rows on different banks
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int part = blockIdx.x % parts, row0 = (int)(blockIdx.x / parts) * ROWS;
  const int rb0 = blockIdx.y * NRB, rbs = a.rank_pad / 16;
  find_ids<ROWS>(a, row0, ids, tid);
  const int steps = (a.in_dim + STEP - 1) / STEP;
  const int p0 = part * steps_each, p1 = min(steps, p0 + steps_each);
  const int each = (p1 - p0 + kWaves - 1) / kWaves;
  const int k0 = min(p1, p0 + w * each), k1 = min(p1, k0 + each);
  const T* x[RT];
#pragma unroll
  for (int r = 0; r < RT; r++)
    x[r] = static_cast<const T*>(a.x) + (int64_t)min(row0 + r * kTile + n, a.rows - 1) * a.ldx + g * V;

  for (int i = 0; i < ids.count; i++) {
    const int id = __builtin_amdgcn_readfirstlane(ids.list[i]);
    const chunk<T>* wa = static_cast<const chunk<T>*>(a.wa) + ((int64_t)id * rbs + rb0) * steps * 64 + lane;
    f32x4_t acc[RT][NRB] = {};
    // U steps' loads go out before their products (the compiler does not unroll
    // loops with matrix instructions); a step past the wave's last is zeros.
    constexpr int U = RT * NRB <= 2 ? 8 : RT * NRB <= 4 ? 4 : 2;
    for (int k = k0; k < k1; k += U) {
      chunk<T> xf[U][RT], af[U][NRB];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const bool on = k + u < k1;
#pragma unroll
        for (int b = 0; b < NRB; b++)
          af[u][b] = on && rb0 + b < rbs ? wa[((int64_t)b * steps + k + u) * 64] : chunk<T>{};
#pragma unroll
        for (int r = 0; r < RT; r++)
          xf[u][r] = on && (k + u) * STEP + g * V < a.in_dim
                         ? *reinterpret_cast<const chunk<T>*>(x[r] + (int64_t)(k + u) * STEP)
                         : chunk<T>{};
      }
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int b = 0; b < NRB; b++)
#pragma unroll
          for (int r = 0; r < RT; r++) acc[r][b] = mfma<T>(af[u][b], xf[u][r], acc[r][b]);
    }
#pragma unroll
    for (int r = 0; r < RT; r++)
      if (ids.own[r * kTile + n] == id) {
#pragma unroll
        for (int b = 0; b < NRB; b++)
          *reinterpret_cast<f32x4_t*>(&sums[w][r * kTile + n][16 * b + 4 * g]) = acc[r][b];
      }
  }
  __syncthreads();
  const int width = min(NRB, rbs - rb0) * 4;  // float4 a row
  for (int i = tid; i < ROWS * width; i += kNT) {
    const int r = i / width, c = (i % width) * 4;
    if (ids.own[r] < 0) continue;  // (rows past the end have none)
    f32x4_t s = *reinterpret_cast<const f32x4_t*>(&sums[0][r][c]);
#pragma unroll
    for (int v = 1; v < kWaves; v++) s += *reinterpret_cast<const f32x4_t*>(&sums[v][r][c]);
    *reinterpret_cast<f32x4_t*>(a.u + ((int64_t)part * a.rows + row0 + r) * a.rank_pad + rb0 * 16 + c) = s;
  }
}

// ---- up: dst = base + scale B u ------------------------------------------------
// u's operand of one 16-rank block in LDS, ready to load: 16-bit types, lane (n, g)
// 8 values: ranks 8 (g & 1) .. + 7 of row n, upper halves for g < 2, what they
// leave for g >= 2; float32, lane (n, g) ranks 4 g .. + 3.
template <typename T>
__device__ __forceinline__ void put_u(chunk<T>* at, int n, int r4, const f32x4_t& u) {  // ranks r4 .. + 3 of the block
  T* p = at[16 * (r4 >> 3) + n].v + (r4 & 4);
  T* q = at[32 + 16 * (r4 >> 3) + n].v + (r4 & 4);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    p[i] = elem<T>::from(u[i]);
    q[i] = elem<T>::from(u[i] - elem<T>::to(p[i]));
  }
}
template <>
__device__ __forceinline__ void put_u<float>(chunk<float>* at, int n, int r4, const f32x4_t& u) {
  *reinterpret_cast<f32x4_t*>(&at[16 * (r4 >> 2) + n]) = u;
}

// A workgroup: RT tiles of 16 rows and `cols` columns (a multiple of 32), the
// 32-column pairs dealt over its waves.
template <typename T, int RT>
__global__ __launch_bounds__(kNT) void k_adapter_up(sg_adapters_args a, int parts, int cols, int slices) {
  constexpr int V = elem<T>::vec, ROWS = RT * kTile, BL = V == 4 ? 64 : 32;  // lanes that a B fragment holds
  extern __shared__ char smem[];
  __shared__ tile_ids<ROWS> ids;
  __shared__ float back[ROWS];
  chunk<T>* us = reinterpret_cast<chunk<T>*>(smem);  // [RT][rank_pad / 16][64]
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int slice = blockIdx.x % slices, row0 = (int)(blockIdx.x / slices) * ROWS;
  const int rbs = a.rank_pad / 16;
  find_ids<ROWS>(a, row0, ids, tid);
  {
    // TPR threads a row, up to kHeld pieces of four ranks each.  A row's u times
    // its adapter's scale is multiplied by the power of two that brings its
    // largest value to 2^10 .. 2^11 (exact; undone below): fp16 then holds every
    // u that float32 holds, and its second half stays clear of the subnormals.
    constexpr int TPR = kNT / ROWS, kHeld = sgk::kAdapterMaxRank / 4 / (kNT / kTile);
    static_assert(kHeld * TPR * 4 * RT >= sgk::kAdapterMaxRank, "row_tiles keeps RT * rank within 256");
    const int r = tid / TPR;
    const int id = ids.own[r];
    const float* u = a.u + (int64_t)(row0 + r) * a.rank_pad;
    f32x4_t s[kHeld];
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < kHeld; k++) {
      const int c = (tid % TPR + k * TPR) * 4;
      s[k] = f32x4_t{0, 0, 0, 0};
      if (id >= 0 && c < a.rank_pad) {
        for (int p = 0; p < parts; p++) s[k] += *reinterpret_cast<const f32x4_t*>(u + (int64_t)p * a.rows * a.rank_pad + c);
        s[k] *= a.scales[id];
      }
#pragma unroll
      for (int i = 0; i < 4; i++) top = fmaxf(top, fabsf(s[k][i]));
    }
#pragma unroll
    for (int o = TPR / 2; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const int e = min(max((int)(__float_as_uint(top) >> 23), 11), 254);
    const float up = __uint_as_float((uint32_t)min(264 - e, 254) << 23);
    if (tid % TPR == 0) back[r] = 1.0f / up;
#pragma unroll
    for (int k = 0; k < kHeld; k++) {
      const int c = (tid % TPR + k * TPR) * 4;
      if (c < a.rank_pad) put_u<T>(us + ((r / kTile) * rbs + c / 16) * 64, r % kTile, c & 15, s[k] * up);
    }
  }
  __syncthreads();
  int own[RT];
  float by[RT];
#pragma unroll
  for (int r = 0; r < RT; r++) {
    own[r] = ids.own[r * kTile + n];
    by[r] = back[r * kTile + n];
  }
  const int pairs = (a.out_dim + 31) / 32;
  const int c1 = min(a.out_dim, (slice + 1) * cols);
  const T* base = static_cast<const T*>(a.base);
  T* dst = static_cast<T*>(a.dst);
  for (int col0 = slice * cols + 32 * w; col0 < c1; col0 += 32 * kWaves) {
    const int col = col0 + 8 * g;
    chunk<T> bv[RT][8 / V];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int h = 0; h < 8 / V; h++)
        if (own[r] != kNoRow && col < a.out_dim)
          bv[r][h] = *reinterpret_cast<const chunk<T>*>(base + (int64_t)(row0 + r * kTile + n) * a.ldb + col + h * V);
    f32x4_t sum[RT][2] = {};
    for (int i = 0; i < ids.count; i++) {
      const int id = __builtin_amdgcn_readfirstlane(ids.list[i]);
      const chunk<T>* wb =
          static_cast<const chunk<T>*>(a.wb) + ((int64_t)id * pairs + col0 / 32) * 2 * rbs * BL + (lane & (BL - 1));
      f32x4_t acc[RT][2] = {};
      constexpr int U = RT <= 2 ? 4 : 2;
      for (int b = 0; b < rbs; b += U) {
        chunk<T> wf[U][2];
#pragma unroll
        for (int u = 0; u < U; u++)
          if (b + u < rbs) {
            wf[u][0] = wb[(b + u) * BL];
            wf[u][1] = wb[(rbs + b + u) * BL];
          }
#pragma unroll
        for (int u = 0; u < U; u++)
          if (b + u < rbs) {
#pragma unroll
            for (int r = 0; r < RT; r++) {
              const chunk<T> uf = us[(r * rbs + b + u) * 64 + lane];
              acc[r][0] = mfma<T>(wf[u][0], uf, acc[r][0]);
              acc[r][1] = mfma<T>(wf[u][1], uf, acc[r][1]);
            }
          }
      }
      // The other adapters' rows are dropped, not multiplied by zero: a weight
      // that is no number stays with its own requests.
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int j = 0; j < 2; j++) sum[r][j] = own[r] == id ? acc[r][j] : sum[r][j];
    }
#pragma unroll
    for (int r = 0; r < RT; r++) {
      if (own[r] == kNoRow || col >= a.out_dim) continue;
#pragma unroll
      for (int h = 0; h < 8 / V; h++) {
        chunk<T> o;
#pragma unroll
        for (int i = 0; i < V; i++) {
          const int e = h * V + i;
          o.v[i] = own[r] >= 0 ? elem<T>::from(__builtin_fmaf(sum[r][e >> 2][e & 3], by[r], elem<T>::to(bv[r][h].v[i])))
                               : bv[r][h].v[i];
        }
        *reinterpret_cast<chunk<T>*>(dst + (int64_t)(row0 + r * kTile + n) * a.ldd + col + h * V) = o;
      }
    }
  }
}

// ---- packing ---------------------------------------------------------------------
template <typename T>
__global__ void k_pack_a(const T* __restrict__ a, int rank, int in_dim, int rbs, int steps, int64_t total,
                         chunk<T>* __restrict__ out) {
  constexpr int V = elem<T>::vec;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const int lane = (int)(i & 63);
  const int64_t f = i >> 6;
  const int k = (int)(f % steps), rb = (int)(f / steps % rbs);
  const int64_t id = f / steps / rbs;
  const int r = 16 * rb + (lane & 15), c = k * 4 * V + (lane >> 4) * V;
  chunk<T> o{};
#pragma unroll
  for (int e = 0; e < V; e++)
    if (r < rank && c + e < in_dim) o.v[e] = a[(id * rank + r) * in_dim + c + e];
  out[i] = o;
}

template <typename T>
__global__ void k_pack_b(const T* __restrict__ b, int rank, int out_dim, int rbs, int pairs, int64_t total,
                         chunk<T>* __restrict__ out) {
  constexpr int V = elem<T>::vec, BL = V == 4 ? 64 : 32;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const int lane = (int)(i % BL);
  const int64_t f = i / BL;
  const int rb = (int)(f % rbs), j = (int)(f / rbs % 2), p = (int)(f / rbs / 2 % pairs);
  const int64_t id = f / rbs / 2 / pairs;
  const int m = lane & 15, col = 32 * p + 8 * (m >> 2) + 4 * j + (m & 3), r = 16 * rb + (lane >> 4) * V;
  chunk<T> o{};
#pragma unroll
  for (int e = 0; e < V; e++)
    if (col < out_dim && r + e < rank) o.v[e] = b[(id * out_dim + col) * rank + r + e];
  out[i] = o;
}

template <typename T>
int64_t a_chunks(int n, int rank, int in_dim) {
  return (int64_t)n * (sgk::adapters_rank_pad(rank) / 16) * ((in_dim + step_of<T>() - 1) / step_of<T>()) * 64;
}
template <typename T>
int64_t b_chunks(int n, int rank, int out_dim) {
  return (int64_t)n * ((out_dim + 31) / 32) * 2 * (sgk::adapters_rank_pad(rank) / 16) * (elem<T>::vec == 4 ? 64 : 32);
}

template <typename T>
hipError_t pack(const void* a, const void* b, int n, int rank, int in_dim, int out_dim, void* wa, void* wb, hipStream_t s) {
  const int rbs = sgk::adapters_rank_pad(rank) / 16;
  const int64_t na = a_chunks<T>(n, rank, in_dim), nb = b_chunks<T>(n, rank, out_dim);
  hipLaunchKernelGGL((k_pack_a<T>), dim3((unsigned)((na + 255) / 256)), dim3(256), 0, s, static_cast<const T*>(a), rank, in_dim,
                     rbs, (in_dim + step_of<T>() - 1) / step_of<T>(), na, static_cast<chunk<T>*>(wa));
  hipLaunchKernelGGL((k_pack_b<T>), dim3((unsigned)((nb + 255) / 256)), dim3(256), 0, s, static_cast<const T*>(b), rank, out_dim,
                     rbs, (out_dim + 31) / 32, nb, static_cast<chunk<T>*>(wb));
  return hipGetLastError();
}

// ---- launches ----------------------------------------------------------------------
// Tiles a workgroup takes: more rows share its weight loads, as long as that
// leaves a workgroup for every CU.
int row_tiles(int rows, int rank_pad) {
  for (int rt = 4; rt > 1; rt /= 2)
    if (rt * rank_pad <= 256 && (rows + rt * kTile - 1) / (rt * kTile) >= kCus) return rt;
  return 1;
}

// Parts of down's sum: enough workgroups for the CUs, four steps of each wave at least.
template <typename T>
int parts_of(int rows, int in_dim, int rank_pad) {
  const int rt = row_tiles(rows, rank_pad);
  const int wgs = (rows + rt * kTile - 1) / (rt * kTile), steps = (in_dim + step_of<T>() - 1) / step_of<T>();
  const int most = std::min(kMostSplit, std::max(1, steps / (4 * kWaves)));
  return std::max(1, std::min(most, kCus / std::max(1, wgs)));
}

template <typename T, int RT>
hipError_t apply_rt(const sg_adapters_args& a, hipStream_t s) {
  const int parts = parts_of<T>(a.rows, a.in_dim, a.rank_pad);
  const int tiles = (a.rows + RT * kTile - 1) / (RT * kTile), rbs = a.rank_pad / 16;
  const int steps = (a.in_dim + step_of<T>() - 1) / step_of<T>(), each = (steps + parts - 1) / parts;
  if (rbs == 1)
    hipLaunchKernelGGL((k_adapter_down<T, RT, 1>), dim3((unsigned)tiles * parts, 1), dim3(kNT), 0, s, a, parts, each);
  else if (rbs == 2)
    hipLaunchKernelGGL((k_adapter_down<T, RT, 2>), dim3((unsigned)tiles * parts, 1), dim3(kNT), 0, s, a, parts, each);
  else
    hipLaunchKernelGGL((k_adapter_down<T, RT, 4>), dim3((unsigned)tiles * parts, (rbs + 3) / 4), dim3(kNT), 0, s, a, parts, each);
  // Columns a workgroup takes: a pair for every wave at least, more while the
  // grid keeps four workgroups a CU.  The slice is the fast index of the grid
  // (and workgroup i runs on XCD i % 8): with eight slices or a multiple, an
  // XCD's L2 holds its own slice of the adapters' B and no other.
  int cols = 32 * kWaves;
  while (cols < 1024 && (int64_t)tiles * ((a.out_dim + 2 * cols - 1) / (2 * cols)) >= 4 * kCus) cols *= 2;
  const int slices = (a.out_dim + cols - 1) / cols;
  hipLaunchKernelGGL((k_adapter_up<T, RT>), dim3((unsigned)tiles * slices), dim3(kNT), (size_t)RT * rbs * 64 * 16, s, a, parts,
                     cols, slices);
  return hipGetLastError();
}

template <typename T>
hipError_t apply(const sg_adapters_args& a, hipStream_t s) {
  const int rt = row_tiles(a.rows, a.rank_pad);
  return rt == 4 ? apply_rt<T, 4>(a, s) : rt == 2 ? apply_rt<T, 2>(a, s) : apply_rt<T, 1>(a, s);
}

}  // namespace

namespace sgk {

size_t adapters_a_bytes(int dtype, int n, int rank, int in_dim) {
  return 16 * (size_t)(dtype == SG_F32 ? a_chunks<float>(n, rank, in_dim) : a_chunks<_Float16>(n, rank, in_dim));
}
size_t adapters_b_bytes(int dtype, int n, int rank, int out_dim) {
  return 16 * (size_t)(dtype == SG_F32 ? b_chunks<float>(n, rank, out_dim) : b_chunks<_Float16>(n, rank, out_dim));
}
hipError_t adapters_pack(int dtype, const void* a, const void* b, int n, int rank, int in_dim, int out_dim, void* wa,
                         void* wb, hipStream_t s) {
  if (dtype == SG_F32) return pack<float>(a, b, n, rank, in_dim, out_dim, wa, wb, s);
  if (dtype == SG_F16) return pack<_Float16>(a, b, n, rank, in_dim, out_dim, wa, wb, s);
  return pack<bf16_t>(a, b, n, rank, in_dim, out_dim, wa, wb, s);
}
size_t adapters_work_bytes(int dtype, int rows, int in_dim, int rank_pad) {
  const int parts = dtype == SG_F32 ? parts_of<float>(rows, in_dim, rank_pad) : parts_of<_Float16>(rows, in_dim, rank_pad);
  return sizeof(float) * (size_t)parts * rows * rank_pad;
}
hipError_t adapters_apply(const sg_adapters_args& a, int dtype, hipStream_t s) {
  if (dtype == SG_F32) return apply<float>(a, s);
  if (dtype == SG_F16) return apply<_Float16>(a, s);
  return apply<bf16_t>(a, s);
}

}  // namespace sgk
