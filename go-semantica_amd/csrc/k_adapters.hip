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
// distinct adapters one by one (down a few together where there are many),
// multiplies the whole tile and keeps the rows that are that adapter's.  A tile of
// one sequence, the common case, takes one turn; sixteen single tokens take
// sixteen, each with the 16-row product that a single row needs as well (the
// matrix core's rows are free, the adapters' weights are what such a batch has to
// read).
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
//
// Bound by memory where rows are many, by the chain of dependent loads (offsets, ids,
// weights, then the second launch) where they are few.  Measured, us of down + up and
// the TB/s of x, base, dst and the weights (a copy of 1 GB moves 5.0):
//   30,725 float32 rows, 768 to 1280, rank 16, 8 adapters      35 + 64   4.1
//   16384 bf16 rows, 2048 to 8192, rank 64, 12 adapters       28 + 132  3.9
//   64 single bf16 tokens, 4096 to 4096, rank 16, 48          6.5 + 9   0.7
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
// ids in rising order of first row, each with the 16-row tiles that hold it (bits).
constexpr int kNone = -1, kNoRow = -2;
template <int ROWS>
struct tile_ids {
  int own[ROWS], list[ROWS], tiles[ROWS], count;
};

// From each row's id in lane 0 .. ROWS - 1 of the first wave.
template <int ROWS>
__device__ __forceinline__ void list_ids(int id, tile_ids<ROWS>& t, int lane) {
  if (lane < ROWS) t.own[lane] = id;
  int n = 0;
  uint64_t left = __ballot(lane < ROWS && id >= 0);
  while (left) {
    const int pick = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const uint64_t its = __ballot(lane < ROWS && id == pick);
    int bits = 0;
#pragma unroll
    for (int r = 0; r < ROWS / kTile; r++) bits |= ((its >> (r * kTile)) & 0xffff) ? 1 << r : 0;
    if (lane == 0) {
      t.list[n] = pick;
      t.tiles[n] = bits;
    }
    n++;
    left &= ~its;
  }
  if (lane == 0) t.count = n;
}

// The same from the offsets, by every thread of the workgroup.
template <int ROWS>
__device__ __forceinline__ void find_ids(const sg_adapters_args& a, int row0, tile_ids<ROWS>& t, int tid) {
  static_assert(ROWS <= SG_WAVE, "a lane per row");
  if (tid < SG_WAVE) {
    const int lane = tid, last = min(row0 + ROWS, a.rows) - 1, row = min(row0 + lane, last);
    int seq, s0, s1;
    sgp::row_seq(a.off, a.n_seq, row0, last, row, lane, seq, s0, s1);
    int id = kNoRow;
    if (lane < ROWS && row0 + lane <= last && s0 <= row && row < s1) {
      id = a.ids[seq];
      if (id < 0 || id >= a.n_adapters) id = kNone;
    }
    list_ids<ROWS>(id, t, lane);
  }
  __syncthreads();
}

// u's operand of one 16-rank block, ready to load: 16-bit types, lane (n, g)
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

// fp16: a row's u, four values in each of TPR lanes side by side, is multiplied by the
// power of two that brings its largest value to 2^10 .. 2^11 (exact, and undone by
// `back`): fp16 then holds every u that float32 holds, and its second half stays
// clear of the subnormals.  The other types have float32's range: u as it is, since with
// their weights (above 2^109) the product of a u brought up could leave it.
template <typename T, int TPR>
__device__ __forceinline__ float to_range(const f32x4_t& s, float& back, float top = 0.0f) {
  back = 1.0f;
  if constexpr (!__is_same(T, _Float16)) return 1.0f;
#pragma unroll
  for (int i = 0; i < 4; i++) top = fmaxf(top, fabsf(s[i]));
#pragma unroll
  for (int o = TPR / 2; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  const int e = min(max((int)(__float_as_uint(top) >> 23), 11), 254);
  const float up = __uint_as_float((uint32_t)min(264 - e, 254) << 23);
  back = 1.0f / up;
  return up;
}

// ---- down: u[part][row][rank], times the adapter's scale, and the rows' ids ----------
// A workgroup: RT tiles of 16 rows, one part of in_dim, NRB blocks of 16 ranks, and
// every gridDim.z-th of the rows' adapters, G of them at a time.  Its four waves take a
// quarter of the part's steps each and add up through LDS.
template <typename T, int RT, int NRB, int G>
__global__ __launch_bounds__(kNT) void k_adapter_down(sg_adapters_args a, int parts, int steps_each) {
  constexpr int V = elem<T>::vec, STEP = step_of<T>(), ROWS = RT * kTile;
  __shared__ tile_ids<ROWS> ids;
  __shared__ float sums[kWaves][ROWS][NRB * 16 + 4];  // + 4: rows on different banks
  __shared__ float scale[ROWS];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int part = blockIdx.x % parts, row0 = (int)(blockIdx.x / parts) * ROWS;
  const int rb0 = blockIdx.y * NRB, rbs = a.rank_pad / 16;
  const int steps = (a.in_dim + STEP - 1) / STEP;
  const int p0 = part * steps_each, p1 = min(steps, p0 + steps_each);
  const int each = (p1 - p0 + kWaves - 1) / kWaves;
  const int k0 = min(p1, p0 + w * each), k1 = min(p1, k0 + each);
  const T* x[RT];
#pragma unroll
  for (int r = 0; r < RT; r++)
    x[r] = static_cast<const T*>(a.x) + (int64_t)min(row0 + r * kTile + n, a.rows - 1) * a.ldx + g * V;
  // U steps' loads go out before their products (the compiler does not unroll loops
  // with matrix instructions); a step past the wave's last is zeros.  The first of
  // x go out before the rows' adapters are known.  Eight steps for one tile of one
  // block, whose waves are few; four else (two for several adapters), which keeps three
  // or four waves on a SIMD, two where two tiles meet four rank blocks or several adapters'
  // two (30,725 float32 rows of 768, rank 16, four waves: 34 us, 44 with eight steps, 35 with
  // two; the next steps' x ahead of the products instead: 37 to 45).
  constexpr int U = RT * NRB * G == 1 ? 8 : G == 1 || RT * NRB * G <= 4 ? 4 : 2;
  chunk<T> xf[U][RT];
  auto load_x = [&](int k, int tiles) {
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int r = 0; r < RT; r++)
        xf[u][r] = k + u < k1 && (tiles >> r & 1) && (k + u) * STEP + g * V < a.in_dim
                       ? *reinterpret_cast<const chunk<T>*>(x[r] + (int64_t)(k + u) * STEP)
                       : chunk<T>{};
  };
  load_x(k0, (1 << RT) - 1);
  find_ids<ROWS>(a, row0, ids, tid);
  if (tid < ROWS) scale[tid] = ids.own[tid] >= 0 ? a.scales[ids.own[tid]] : 0.0f;  // read behind the loop's barrier

  for (int i = blockIdx.z; i < ids.count; i += G * gridDim.z) {
    int id[G], in[G], tiles = 0;  // in: the tiles that hold it
    const chunk<T>* wa[G];
#pragma unroll
    for (int j = 0; j < G; j++) {
      const int at = min(i + j * (int)gridDim.z, ids.count - 1);
      id[j] = __builtin_amdgcn_readfirstlane(ids.list[at]);
      in[j] = i + j * (int)gridDim.z < ids.count ? __builtin_amdgcn_readfirstlane(ids.tiles[at]) : 0;
      wa[j] = static_cast<const chunk<T>*>(a.wa) + ((int64_t)id[j] * rbs + rb0) * steps * 64 + lane;
      tiles |= in[j];
    }
    f32x4_t acc[G][RT][NRB] = {};
    for (int k = k0; k < k1; k += U) {
      chunk<T> af[G][U][NRB];
#pragma unroll
      for (int j = 0; j < G; j++)
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int b = 0; b < NRB; b++)
            af[j][u][b] = (G == 1 || in[j]) && k + u < k1 && rb0 + b < rbs ? wa[j][((int64_t)b * steps + k + u) * 64] : chunk<T>{};
      if (k > k0 || i != (int)blockIdx.z) load_x(k, tiles);
#pragma unroll
      for (int j = 0; j < G; j++)
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int b = 0; b < NRB; b++)
#pragma unroll
            for (int r = 0; r < RT; r++)
              if (RT * G == 1 || (in[j] >> r & 1)) acc[j][r][b] = mfma<T>(af[j][u][b], xf[u][r], acc[j][r][b]);
    }
#pragma unroll
    for (int j = 0; j < G; j++)
#pragma unroll
      for (int r = 0; r < RT; r++)
        if ((G == 1 || in[j]) && ids.own[r * kTile + n] == id[j]) {
#pragma unroll
          for (int b = 0; b < NRB; b++)
            *reinterpret_cast<f32x4_t*>(&sums[w][r * kTile + n][16 * b + 4 * g]) = acc[j][r][b];
        }
  }
  __syncthreads();
  constexpr int WIDTH = NRB * 4;  // float4 a row
  for (int i = tid; i < ROWS * WIDTH; i += kNT) {
    const int r = i / WIDTH, c = (i % WIDTH) * 4;
    if (a.ready) {
      // One part and all the ranks: u as up's operand.
      f32x4_t s = {0, 0, 0, 0};
      if (ids.own[r] >= 0) {
#pragma unroll
        for (int v = 0; v < kWaves; v++) s += *reinterpret_cast<const f32x4_t*>(&sums[v][r][c]);
        s *= scale[r];
      }
      float by;
      const float up = to_range<T, WIDTH>(s, by);
      bool mine = ids.own[r] < 0 && blockIdx.z == 0;  // (zeros) or of an adapter that this workgroup took
      for (int j = blockIdx.z; j < ids.count; j += gridDim.z) mine |= ids.own[r] == ids.list[j];
      if (row0 + r >= a.rows || !mine) continue;
      if (c < a.rank_pad)
        put_u<T>(static_cast<chunk<T>*>(a.ready) + ((int64_t)(row0 + r) / kTile * rbs + c / 16) * 64, (row0 + r) % kTile, c & 15,
                 s * up);
      if (c == 0) a.back[row0 + r] = by;
      continue;
    }
    if (c >= (rbs - rb0) * 16) continue;
    // Rows of the adapters that this workgroup took (rows past the end have none).
    bool mine = false;
    for (int j = blockIdx.z; j < ids.count; j += gridDim.z) mine |= ids.own[r] == ids.list[j];
    if (!mine) continue;
    f32x4_t s = *reinterpret_cast<const f32x4_t*>(&sums[0][r][c]);
#pragma unroll
    for (int v = 1; v < kWaves; v++) s += *reinterpret_cast<const f32x4_t*>(&sums[v][r][c]);
    *reinterpret_cast<f32x4_t*>(a.u + ((int64_t)part * a.rows + row0 + r) * a.rank_pad + rb0 * 16 + c) = s * scale[r];
  }
  if (part == 0 && blockIdx.y == 0 && blockIdx.z == 0 && tid < ROWS && row0 + tid < a.rows) a.row_ids[row0 + tid] = ids.own[tid];
}

// ---- up: dst = base + scale B u ------------------------------------------------
// A workgroup: RT tiles of 16 rows and CW = 128 PAIRS columns, a wave PAIRS of their
// 32-column pairs.  The products go through LDS so that base and dst are read and
// written in rows of CW columns.  (A loop over tiles that loads the next one's base
// and u ahead took the registers of a third of the waves, 207 us for 190 at the bf16
// sizes below; a workgroup of 1024 columns in turn, 197.)
template <typename T, int RT, int PAIRS>
__global__ __launch_bounds__(kNT) void k_adapter_up(sg_adapters_args a, int parts, int slices) {
  constexpr int V = elem<T>::vec, ROWS = RT * kTile, BL = V == 4 ? 64 : 32;  // lanes that a B fragment holds
  constexpr int CW = 128 * PAIRS, LD = CW + 4, PIECES = ROWS * CW / V / kNT;  // 16-byte pieces a thread
  extern __shared__ char smem[];
  __shared__ tile_ids<ROWS> ids;
  __shared__ float back[ROWS];
  chunk<T>* us = reinterpret_cast<chunk<T>*>(smem);  // [RT][rank_pad / 16][64]
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int slice = blockIdx.x % slices, rbs = a.rank_pad / 16, pairs = (a.out_dim + 31) / 32;
  float* const delta = reinterpret_cast<float*>(us + RT * rbs * 64);  // [ROWS][LD]
  // Piece i of this thread: row r0 + i RSTEP of a tile, columns col .. .
  constexpr int RSTEP = kNT / (CW / V);
  const int r0 = tid / (CW / V), cc = tid % (CW / V) * V, col = slice * CW + cc;
  const bool in = col < a.out_dim;
  // TPR threads a row of u, up to kHeld pieces of four ranks each.
  constexpr int TPR = kNT / ROWS, kHeld = sgk::kAdapterMaxRank / 4 / (kNT / kTile);
  static_assert(kHeld * TPR * 4 * RT >= sgk::kAdapterMaxRank, "row_tiles keeps RT * rank within 256");
  // The wave's pairs.  (One past the last is the last again; it is not stored.)
  const chunk<T>* wb[PAIRS];
#pragma unroll
  for (int p = 0; p < PAIRS; p++)
    wb[p] = static_cast<const chunk<T>*>(a.wb) + (int64_t)min(slice * (CW / 32) + w * PAIRS + p, pairs - 1) * 2 * rbs * BL +
            (lane & (BL - 1));

  chunk<T> bv[PIECES];
  f32x4_t s[kHeld];
  int rid = kNoRow;
  auto load = [&](int row0) {
    if (in)
#pragma unroll
      for (int i = 0; i < PIECES; i++)
        if (row0 + r0 + i * RSTEP < a.rows)
          bv[i] = *reinterpret_cast<const chunk<T>*>(static_cast<const T*>(a.base) + (int64_t)(row0 + r0 + i * RSTEP) * a.ldb + col);
    const float* u = a.u + (int64_t)min(row0 + tid / TPR, a.rows - 1) * a.rank_pad;
#pragma unroll
    for (int k = 0; k < kHeld; k++) {
      const int c = (tid % TPR + k * TPR) * 4;
      s[k] = f32x4_t{0, 0, 0, 0};
      if (c < a.rank_pad)
        for (int p = 0; p < parts; p += 8) {  // eight loads in flight; their sum in order
          f32x4_t t[8] = {};
#pragma unroll
          for (int i = 0; i < 8; i++)
            if (p + i < parts) t[i] = *reinterpret_cast<const f32x4_t*>(u + (int64_t)(p + i) * a.rows * a.rank_pad + c);
#pragma unroll
          for (int i = 0; i < 8; i++) s[k] += t[i];
        }
    }
    rid = tid < ROWS && row0 + tid < a.rows ? a.row_ids[row0 + tid] : kNoRow;
  };
  const int row0 = (int)(blockIdx.x / slices) * ROWS;
  load(row0);
  if (tid < SG_WAVE) list_ids<ROWS>(rid, ids, lane);
  __syncthreads();
  {
    // A row without an adapter has no u: what down left there goes no further.
    const int r = tid / TPR;
    const bool has = ids.own[r] >= 0;
    float top = 0.0f, by;
#pragma unroll
    for (int k = 0; k < kHeld; k++) {
      s[k] = has ? s[k] : f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; i++) top = fmaxf(top, fabsf(s[k][i]));
    }
    const float up = to_range<T, TPR>(s[0], by, top);
    if (tid % TPR == 0) back[r] = by;
#pragma unroll
    for (int k = 0; k < kHeld; k++) {
      const int c = (tid % TPR + k * TPR) * 4;
      if (c < a.rank_pad) put_u<T>(us + ((r / kTile) * rbs + c / 16) * 64, r % kTile, c & 15, s[k] * up);
    }
  }
  __syncthreads();
  int own[RT], owner[PIECES];
#pragma unroll
  for (int r = 0; r < RT; r++) own[r] = ids.own[r * kTile + n];
#pragma unroll
  for (int i = 0; i < PIECES; i++) owner[i] = ids.own[r0 + i * RSTEP];
  const int turns = ids.count * rbs;
  f32x4_t sum[PAIRS][RT][2] = {}, acc[PAIRS][RT][2] = {};
  // The adapters' rank blocks one after another, U of them loaded at a time.
  constexpr int U = 4 / PAIRS;
  int li = 0, lrb = 0, ci = 0, crb = 0;
  for (int e = 0; e < turns; e += U) {
    chunk<T> wf[U][PAIRS][2];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (e + u < turns) {
        const int64_t first = (int64_t)__builtin_amdgcn_readfirstlane(ids.list[li]) * pairs * 2 * rbs * BL + lrb * BL;
#pragma unroll
        for (int p = 0; p < PAIRS; p++) {
          wf[u][p][0] = wb[p][first];
          wf[u][p][1] = wb[p][first + rbs * BL];
        }
        if (++lrb == rbs) {
          lrb = 0;
          li++;
        }
      }
#pragma unroll
    for (int u = 0; u < U; u++)
      if (e + u < turns) {
        const int tiles = __builtin_amdgcn_readfirstlane(ids.tiles[ci]);
#pragma unroll
        for (int r = 0; r < RT; r++) {
          if (RT > 1 && !(tiles >> r & 1)) continue;
          const chunk<T> uf = us[(r * rbs + crb) * 64 + lane];
#pragma unroll
          for (int p = 0; p < PAIRS; p++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[p][r][j] = mfma<T>(wf[u][p][j], uf, acc[p][r][j]);
        }
        if (++crb == rbs) {
          // The other adapters' rows are dropped, not multiplied by zero: a weight
          // that is no number stays with its own requests.
          const int id = __builtin_amdgcn_readfirstlane(ids.list[ci]);
          crb = 0;
          ci++;
          if (ids.count > 1) {
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
              for (int p = 0; p < PAIRS; p++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                  sum[p][r][j] = own[r] == id ? acc[p][r][j] : sum[p][r][j];
                  acc[p][r][j] = f32x4_t{0, 0, 0, 0};
                }
          } else {  // (a row without an adapter ignores its sum)
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
              for (int p = 0; p < PAIRS; p++)
#pragma unroll
                for (int j = 0; j < 2; j++) sum[p][r][j] = acc[p][r][j];
          }
        }
      }
  }
#pragma unroll
  for (int p = 0; p < PAIRS; p++)
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int j = 0; j < 2; j++)
        *reinterpret_cast<f32x4_t*>(delta + (r * kTile + n) * LD + (w * PAIRS + p) * 32 + 8 * g + 4 * j) = sum[p][r][j];
  __syncthreads();
  if (in) {
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
      if (owner[i] == kNoRow) continue;
      chunk<T> o = bv[i];
      const int r = r0 + i * RSTEP;
      if (owner[i] >= 0) {
        const float f = back[r];
#pragma unroll
        for (int q = 0; q < V; q += 4) {
          const f32x4_t d = *reinterpret_cast<const f32x4_t*>(delta + r * LD + cc + q);
#pragma unroll
          for (int k = 0; k < 4; k++) o.v[q + k] = elem<T>::from(__builtin_fmaf(d[k], f, elem<T>::to(o.v[q + k])));
        }
      }
      *reinterpret_cast<chunk<T>*>(static_cast<T*>(a.dst) + (int64_t)(row0 + r) * a.ldd + col) = o;
    }
  }
}

// The same from operands that down left ready (one part of in_dim, at most 64 ranks:
// batches of many rows): u's fragments come straight from memory into registers, so
// that nothing of a tile is prepared once for each of its slices, which was half of
// up's vector instructions (both kernels at the sizes below: 115 / 190 us so, 111 /
// 162 now; the bytes take 82 / 123 at a copy's rate).
template <typename T, int RT, int PAIRS, int NRB>
__global__ __launch_bounds__(kNT) void k_adapter_up_ready(sg_adapters_args a, int slices) {
  constexpr int V = elem<T>::vec, ROWS = RT * kTile, BL = V == 4 ? 64 : 32;
  constexpr int CW = 128 * PAIRS, LD = CW + 4, PIECES = ROWS * CW / V / kNT;
  __shared__ float delta[ROWS][LD];
  __shared__ tile_ids<ROWS> ids;
  __shared__ float back[ROWS];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int slice = blockIdx.x % slices, row0 = (int)(blockIdx.x / slices) * ROWS;
  const int rbs = a.rank_pad / 16, pairs = (a.out_dim + 31) / 32;
  constexpr int RSTEP = kNT / (CW / V);
  const int r0 = tid / (CW / V), cc = tid % (CW / V) * V, col = slice * CW + cc;
  const bool in = col < a.out_dim;
  int rid = kNoRow;
  if (tid < ROWS && row0 + tid < a.rows) {
    rid = a.row_ids[row0 + tid];
    back[tid] = a.back[row0 + tid];
  }
  chunk<T> bv[PIECES];
  const T* const bp = static_cast<const T*>(a.base) + (int64_t)(row0 + r0) * a.ldb + col;
#pragma unroll
  for (int i = 0; i < PIECES; i++)
    if (in && row0 + r0 + i * RSTEP < a.rows) bv[i] = *reinterpret_cast<const chunk<T>*>(bp + i * RSTEP * a.ldb);
  chunk<T> uf[RT][NRB];
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int b = 0; b < NRB; b++) {
      const int64_t tile = min(row0 / kTile + r, (a.rows - 1) / kTile);
      uf[r][b] = b < rbs ? static_cast<const chunk<T>*>(a.ready)[(tile * rbs + b) * 64 + lane] : chunk<T>{};
    }
  if (tid < SG_WAVE) list_ids<ROWS>(rid, ids, lane);
  __syncthreads();
  int own[RT], owner[PIECES];
#pragma unroll
  for (int r = 0; r < RT; r++) own[r] = ids.own[r * kTile + n];
#pragma unroll
  for (int i = 0; i < PIECES; i++) owner[i] = ids.own[r0 + i * RSTEP];
  const chunk<T>* wb[PAIRS];
#pragma unroll
  for (int p = 0; p < PAIRS; p++)
    wb[p] = static_cast<const chunk<T>*>(a.wb) + (int64_t)min(slice * (CW / 32) + w * PAIRS + p, pairs - 1) * 2 * rbs * BL +
            (lane & (BL - 1));
  f32x4_t sum[PAIRS][RT][2];
  const int count = ids.count;
  for (int i = 0; i < count; i++) {
    const int id = __builtin_amdgcn_readfirstlane(ids.list[i]);
    const int64_t first = (int64_t)id * pairs * 2 * rbs * BL;
    f32x4_t acc[PAIRS][RT][2] = {};
#pragma unroll
    for (int p = 0; p < PAIRS; p++) {
      chunk<T> wf[NRB][2];
#pragma unroll
      for (int b = 0; b < NRB; b++)
#pragma unroll
        for (int j = 0; j < 2; j++) wf[b][j] = b < rbs ? wb[p][first + (j * rbs + b) * BL] : chunk<T>{};
#pragma unroll
      for (int b = 0; b < NRB; b++)
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
          for (int j = 0; j < 2; j++) acc[p][r][j] = mfma<T>(wf[b][j], uf[r][b], acc[p][r][j]);
    }
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int p = 0; p < PAIRS; p++)
#pragma unroll
        for (int j = 0; j < 2; j++) sum[p][r][j] = i == 0 || own[r] == id ? acc[p][r][j] : sum[p][r][j];
  }
  if (count > 0)
#pragma unroll
    for (int p = 0; p < PAIRS; p++)
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int j = 0; j < 2; j++)
          *reinterpret_cast<f32x4_t*>(&delta[r * kTile + n][(w * PAIRS + p) * 32 + 8 * g + 4 * j]) = sum[p][r][j];
  __syncthreads();
  if (!in) return;
  T* const dp = static_cast<T*>(a.dst) + (int64_t)(row0 + r0) * a.ldd + col;
#pragma unroll
  for (int i = 0; i < PIECES; i++) {
    if (owner[i] == kNoRow) continue;
    chunk<T> o = bv[i];
    if (owner[i] >= 0) {
      const int r = r0 + i * RSTEP;
      const float f = back[r];
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        const f32x4_t d = *reinterpret_cast<const f32x4_t*>(&delta[r][cc + q]);
#pragma unroll
        for (int k = 0; k < 4; k++) o.v[q + k] = elem<T>::from(__builtin_fmaf(d[k], f, elem<T>::to(o.v[q + k])));
      }
    }
    *reinterpret_cast<chunk<T>*>(dp + i * RSTEP * a.ldd) = o;
  }
}

// ---- packing ---------------------------------------------------------------------
// (In a loop: a bank may have more chunks than a launch has threads, 2^32.)
constexpr int kPackBlocks = 1 << 16;

template <typename T>
__global__ void k_pack_a(const T* __restrict__ a, int rank, int in_dim, int rbs, int steps, int64_t total,
                         chunk<T>* __restrict__ out) {
  constexpr int V = elem<T>::vec;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
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
}

template <typename T>
__global__ void k_pack_b(const T* __restrict__ b, int rank, int out_dim, int rbs, int pairs, int64_t total,
                         chunk<T>* __restrict__ out) {
  constexpr int V = elem<T>::vec, BL = V == 4 ? 64 : 32;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
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
  auto blocks = [](int64_t chunks) { return dim3((unsigned)std::min<int64_t>((chunks + 255) / 256, kPackBlocks)); };
  const hipError_t e = sgp::run_kernel(k_pack_a<T>, blocks(na), dim3(256), 0, s, static_cast<const T*>(a), rank, in_dim, rbs,
                                       (in_dim + step_of<T>() - 1) / step_of<T>(), na, static_cast<chunk<T>*>(wa));
  if (e != hipSuccess) return e;
  return sgp::run_kernel(k_pack_b<T>, blocks(nb), dim3(256), 0, s, static_cast<const T*>(b), rank, out_dim, rbs,
                         (out_dim + 31) / 32, nb, static_cast<chunk<T>*>(wb));
}

// ---- launches ----------------------------------------------------------------------
// Tiles of 16 rows a workgroup takes: two, which share its weight loads, from ranks of
// 128 down (up's u lies in LDS) and where that leaves two workgroups a CU at least.  Both sides,
// us for 30,725 float32 rows of 768 (rank 16, 1280 columns) / 16384 bf16 rows of 2048
// (rank 64, 8192 columns): up with one tile 107 / 198, two 111 / 162.  Four lose, down's for
// want of registers: 32,768 float32 rows of 768, rank 16, 36 us for two's 32; 65,536
// bf16 rows of 2048, rank 64, 106 for 100; 33,000 rows of eleven thousand sequences, bf16,
// 2944 dims, rank 64, 534 for 339 (rank 32 of the first is the other way, 40 for 46);
// up (an earlier form) 126 / 192 for 115 / 190.
int row_tiles(int rows, int rank_pad) {
  return 2 * rank_pad <= 256 && (rows + 2 * kTile - 1) / (2 * kTile) >= 2 * kCus ? 2 : 1;
}

// Parts of down's sum: enough workgroups for the CUs, four steps of each wave at least.
template <typename T>
int parts_of(int rows, int in_dim, int rank_pad) {
  const int rt = row_tiles(rows, rank_pad);
  const int wgs = (rows + rt * kTile - 1) / (rt * kTile), steps = (in_dim + step_of<T>() - 1) / step_of<T>();
  const int most = std::min(kMostSplit, std::max(1, steps / (4 * kWaves)));
  return std::max(1, std::min(most, kCus / std::max(1, wgs)));
}

template <typename T, int RT, bool MANY>
hipError_t down(const sg_adapters_args& a, int parts, dim3 grid, hipStream_t s) {
  constexpr int G = MANY ? 4 : 1, G4 = MANY ? 2 : 1;  // (of four rank blocks two adapters: 53 us, four 57)
  const int rbs = a.rank_pad / 16, steps = (a.in_dim + step_of<T>() - 1) / step_of<T>(), each = (steps + parts - 1) / parts;
  if (rbs == 1) return sgp::run_kernel(k_adapter_down<T, RT, 1, G>, grid, dim3(kNT), 0, s, a, parts, each);
  if (rbs == 2) return sgp::run_kernel(k_adapter_down<T, RT, 2, G>, grid, dim3(kNT), 0, s, a, parts, each);
  return sgp::run_kernel(k_adapter_down<T, RT, 4, G4>, grid, dim3(kNT), 0, s, a, parts, each);
}

template <typename T, int RT>
hipError_t down(const sg_adapters_args& a, int parts, hipStream_t s) {
  const int tiles = (a.rows + RT * kTile - 1) / (RT * kTile), rbs = a.rank_pad / 16;
  // Adapters that a workgroup's rows are likely to have, over as many workgroups
  // while those are few (64 single tokens with 48 adapters: 6.8 us, 16.4 one after
  // another).
  const int64_t likely = std::min<int64_t>(std::min(a.n_adapters, a.n_seq), ((int64_t)RT * kTile * a.n_seq + a.rows - 1) / a.rows);
  const int z = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(likely, RT * kTile), 4 * kCus / ((int64_t)tiles * parts)));
  const dim3 grid((unsigned)(tiles * parts), rbs <= 2 ? 1 : (rbs + 3) / 4, z);
  // Where a workgroup still has several, it takes them together: their weights' loads are
  // in flight at once, and x is read once for them (4907 sequences of three bf16 tokens
  // with 18 adapters, 2944 dims, rank 7: 47 us, 89 one after another; from two on: 2716 of
  // two fp16 tokens, rank 24, a call 22 us for 18).
  return likely >= 3 * z ? down<T, RT, true>(a, parts, grid, s) : down<T, RT, false>(a, parts, grid, s);
}

template <typename T, int RT, int PAIRS>
hipError_t up(const sg_adapters_args& a, int parts, hipStream_t s) {
  constexpr int CW = 128 * PAIRS;
  const int tiles = (a.rows + RT * kTile - 1) / (RT * kTile), slices = (a.out_dim + CW - 1) / CW;
  const dim3 grid((unsigned)tiles * slices);
  if (a.ready) {
    if (a.rank_pad == 16) return sgp::run_kernel(k_adapter_up_ready<T, RT, PAIRS, 1>, grid, dim3(kNT), 0, s, a, slices);
    if (a.rank_pad == 32) return sgp::run_kernel(k_adapter_up_ready<T, RT, PAIRS, 2>, grid, dim3(kNT), 0, s, a, slices);
    return sgp::run_kernel(k_adapter_up_ready<T, RT, PAIRS, 4>, grid, dim3(kNT), 0, s, a, slices);
  }
  const size_t lds = (size_t)RT * a.rank_pad / 16 * 64 * 16 + sizeof(float) * RT * kTile * (CW + 4);
  return sgp::run_kernel(k_adapter_up<T, RT, PAIRS>, grid, dim3(kNT), lds, s, a, parts, slices);
}

template <typename T, int RT>
hipError_t up(const sg_adapters_args& a, int parts, hipStream_t s) {
  // Columns a workgroup takes: 256 while that leaves eight workgroups a CU, else 128
  // (always 128: 110 / 183 us at the sizes above).  The slice is the fast index of
  // the grid (and workgroup i runs on XCD i % 8): with eight slices or a multiple, an
  // XCD's L2 holds its own slices of the adapters' B and no other.
  const int64_t tiles = (a.rows + RT * kTile - 1) / (RT * kTile);
  return tiles * ((a.out_dim + 255) / 256) >= 8 * kCus ? up<T, RT, 2>(a, parts, s) : up<T, RT, 1>(a, parts, s);
}

template <typename T>
hipError_t apply(sg_adapters_args a, hipStream_t s) {
  const int parts = parts_of<T>(a.rows, a.in_dim, a.rank_pad);
  // The workspace: u (or its operands, of whole tiles), then an id and a factor a row.
  const size_t tiled = (size_t)(a.rows + kTile - 1) / kTile * kTile;
  a.row_ids = reinterpret_cast<int32_t*>(a.u + (parts > 1 ? parts * (size_t)a.rows : tiled) * a.rank_pad);
  a.back = reinterpret_cast<float*>(a.row_ids + a.rows);
  a.ready = parts == 1 && a.rank_pad <= 64 ? a.u : nullptr;
  if (row_tiles(a.rows, a.rank_pad) == 2) {
    const hipError_t e = down<T, 2>(a, parts, s);
    return e == hipSuccess ? up<T, 2>(a, parts, s) : e;
  }
  const hipError_t e = down<T, 1>(a, parts, s);
  return e == hipSuccess ? up<T, 1>(a, parts, s) : e;
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
// Enough for every batch of up to `rows` rows, so that a workspace for the largest one
// serves them all: fewer rows may be split into more parts, whose sums take more than
// one part's of the larger batch.
size_t adapters_work_bytes(int dtype, int rows, int in_dim, int rank_pad) {
  auto parts_at = [&](int r) { return dtype == SG_F32 ? parts_of<float>(r, in_dim, rank_pad) : parts_of<_Float16>(r, in_dim, rank_pad); };
  auto bytes = [&](size_t held, size_t r) { return sizeof(float) * (held * rank_pad + 2 * r); };
  size_t most = 0;
  if (parts_at(rows) == 1) most = bytes((size_t)(rows + kTile - 1) / kTile * kTile, rows);
  // The most rows that p parts are taken for (they are tiles of 16 there).
  for (int p = 2; p <= kMostSplit; p++) {
    const int r = std::min(rows, kCus / p * kTile);
    if (parts_at(r) >= p) most = std::max(most, bytes((size_t)p * r, r));
  }
  return most;
}
// Up's, with slices of 256 columns (those of 128 are for small batches, as down's parts are).
int64_t adapters_threads(int rows, int out_dim, int rank_pad) {
  const int rt = row_tiles(rows, rank_pad);
  return ((int64_t)rows + rt * kTile - 1) / (rt * kTile) * ((out_dim + 255) / 256) * kNT;
}
hipError_t adapters_apply(const sg_adapters_args& a, int dtype, hipStream_t s) {
  if (dtype == SG_F32) return apply<float>(a, s);
  if (dtype == SG_F16) return apply<_Float16>(a, s);
  return apply<bf16_t>(a, s);
}

}  // namespace sgk
