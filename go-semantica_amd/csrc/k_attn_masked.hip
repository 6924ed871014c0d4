// k_attn_masked.hip -- attention of packed sequences with themselves whose scores
// are capped, biased or masked (sg_attention_masked):
//   s_ij = scale * q_i . k_j;  s = cap * tanh(s / cap);  s -= slope_h * |i - j|
//   o_i  = sum_j e^(s_ij - m_i) v_j / sum_j e^(s_ij - m_i)   over the visible j
// in one pass over the keys with a running maximum m_i (in powers of two: scores
// are kept times log2 e).
//
// A query's visible keys are one range [lo, hi) -- its sequence, cut by causal,
// prefix and window -- less the keys of other documents.  So a workgroup takes
// consecutive rows of the packed batch, whatever sequences they belong to, and
// walks the key tiles that any of its rows can see; a tile that all rows of a
// wave see whole skips every comparison.  Nothing about the batch is needed on
// the host.
//
// Layout.  Scores are computed transposed, S^T = K Q^T on 32x32 tiles: a lane
// holds one query's scores of 16 keys, so maxima, sums and rescaling are the
// lane's own (plus one exchange with lane ^ 32), and those 16 registers are, as
// they stand, the B operand of O^T += V^T P^T.  K is read from LDS as the A
// operand, V through the transposing LDS load (ds_read_b64_tr_b16: four keys of
// the lane's dim each).  Rows of 16-byte pieces are stored in LDS with the piece
// index xor-ed by the row (swz_k, swz_v), so neither read meets bank conflicts.
//
// 16-bit types go to LDS by buffer_load ... lds, a tile ahead.  float32 operands
// are split into two fp16 halves each, hi + lo, and products run as hi.hi + hi.lo
// + lo.hi (22 bits of each operand; the dropped lo.lo is 2^-22 of the product).
// Every row of Q, K and V is first brought to the same power of two, so fp16's
// range does not matter: K's power multiplies the score, V's is added to the
// score that the weight is formed from (p' = 2^(s + e_j - m'), |v'| alike for all
// keys), and the softmax's sum takes it out again (sum p' 2^-e_j).  A value keeps
// 22 bits down to 2^-15 of its row's largest and 2^-37 of the largest below that.
//
// A hidden key has weight zero, and zero times an infinity or a NaN in its value
// is a NaN.  Instead of looking at every value, a wave looks at its outputs: rows
// that did not come out finite are computed again one key at a time from the
// visible keys only (careful_row).  That also covers float32 values past the
// fp16 halves' reach (q and k above 2^113, values 2^53 times the first keys').
//
// Two forms (attention_masked has the rule): four waves of 32 rows each, or, for
// batches with too few rows to fill the GPU, waves that share 32 (64) rows and
// split each tile's keys between them, joined through LDS at the end.
#include <algorithm>

#include "semantica_gpu.h"
#include "sg_kernels.h"
#include "sg_packed.h"

namespace {

using sgp::bf16_t;
using sgp::bf16x8_t;
using sgp::chunk;
using sgp::elem;

constexpr int kWaves = 4, kNT = kWaves * SG_WAVE;
constexpr int kSub = 32;  // keys and queries of a matrix core tile
constexpr float kLog2e = 1.44269504088896340736f;
// A row's maximum is raised (and its sums rescaled) only when a score passes it by
// this many powers of two, so most tiles rescale nothing; weights stay below 2^8.
constexpr float kSlack = 8.0f;
constexpr int kScanTiles = 32;  // tiles of one look at the document ids

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));

// How T is multiplied: its own type, or fp16 halves.
template <typename T>
struct mul {
  typedef T type;
  static constexpr int parts = 1;
  static constexpr float shift = 0.0f;
};
template <>
struct mul<_Float16> {
  typedef _Float16 type;
  static constexpr int parts = 1;
  static constexpr float shift = 6.0f;  // weights times 2^6: fp16 holds them to 2^-20 with all its bits
};
template <>
struct mul<float> {
  typedef _Float16 type;
  static constexpr int parts = 2;
  static constexpr float shift = 5.0f;
};

template <typename M>
__device__ __forceinline__ f32x16_t mfma32(s16x8_t a, s16x8_t b, f32x16_t c) {
  if constexpr (__is_same(M, bf16_t))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

template <int D>
__device__ __forceinline__ int swz_k(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }
template <int D>
__device__ __forceinline__ int swz_v(int row) { return D == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }

constexpr int kTop = 13;  // rows are brought to 2^13 .. 2^14 before they are halved
constexpr int kLim = 110;
// V's exponents are kept within this of the workgroup's first keys': 2^-e then sums
// without overflow, and a weight that underflows beside a row of larger values
// is below 2^-26 of the softmax's sum as well.
constexpr int kSpan = 50;

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// floor(log2 m) of a row's largest magnitude, within what pow2 can undo.
__device__ __forceinline__ int row_exp(float m) { return min(max((int)(__float_as_uint(m) >> 23) - 127, -kLim), kLim); }

// The largest finite magnitude of N values (a NaN is passed over by fmaxf).
template <int N>
__device__ __forceinline__ float finite_top(const float* x) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i++) top = fmaxf(top, fabsf(x[i]));
  if (__ballot(top == INFINITY)) {
    top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) top = fmaxf(top, fabsf(x[i]) < INFINITY ? fabsf(x[i]) : 0.0f);
  }
  return top;
}

// Eight values times by, as fp16 halves.
__device__ __forceinline__ void halves(const float* x, float by, s16x8_t& hi, s16x8_t& lo) {
  half8_t h, l;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const hl16 s = split_f16(x[i] * by);
    h[i] = s.hi;
    l[i] = s.lo;
  }
  hi = __builtin_bit_cast(s16x8_t, h);
  lo = __builtin_bit_cast(s16x8_t, l);
}

// tanh.  ACCURATE: Lambert's continued fraction to seven levels below 1.5 (relative
// error 5e-8 at its end), and 1 - 2 / (e^2x + 1) above, where the second term's
// rounding no longer shows; the plain form is off by 1e-7 absolute, which a cap of
// 50 turns into 5e-6 of a weight: nothing beside 16-bit weights.
template <bool ACCURATE>
__device__ __forceinline__ float tanh_of(float x) {
  const float e = __builtin_amdgcn_exp2f(x * (2.0f * kLog2e));
  const float far = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
  if constexpr (!ACCURATE) return far;
  const float z = x * x;
  const float num = x * __builtin_fmaf(__builtin_fmaf(z + 378.0f, z, 17325.0f), z, 135135.0f);
  const float den = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(28.0f, z, 3150.0f), z, 62370.0f), z, 135135.0f);
  const float r = __builtin_amdgcn_rcpf(den), q = num * r;
  const float near = __builtin_fmaf(__builtin_fmaf(-q, den, num), r, q);
  return fabsf(x) < 1.5f ? near : far;
}

template <typename T, int D_, int RW_, int KW_>
struct form {
  static constexpr int D = D_, RW = RW_, KW = KW_;
  static constexpr bool F32 = __is_same(T, float);
  static constexpr int PARTS = mul<T>::parts;
  static constexpr int NSUB = KW > 1 || D == 256 || (F32 && D == 128) ? 1 : 2;  // 32-key blocks a wave takes of a tile
  static constexpr int BK = kSub * KW * NSUB, BM = kSub * RW;
  static constexpr int HALF = BK * D * 2;             // bytes of one tile's K (or V), one part
  static constexpr int TILE = 2 * PARTS * HALF;       // K and V
  static constexpr int STAGES = !F32 && 2 * TILE <= (128 << 10) ? 2 : 1;
  static constexpr int KEYS = F32 ? 3 * BK * 4 : 0;   // per-key powers of a float32 tile
  static constexpr int JOIN = KW > 1 ? kWaves * kSub * D * 4 : 0;
  static constexpr int LDS = (STAGES * TILE + KEYS) > JOIN ? (STAGES * TILE + KEYS) : JOIN;
  static_assert(RW * KW == kWaves, "four waves");
};

// One query's view of the keys.
struct view {
  int lo, hi, doc;
  bool live;  // a row of a sequence
};

// What the scores go through, and what careful_row needs.
template <typename T>
__device__ __forceinline__ float score_of(const sg_attn_masked_args& a, float dot, float slope, int gap) {
  float s = dot * a.scale;
  if (a.softcap > 0.0f) s = a.softcap * tanh_of<true>(s / a.softcap);
  return (s - slope * fabsf((float)gap)) * kLog2e;
}

// out[row][h*hd + d0 .. d1) from the visible keys alone, one at a time, by a wave.
template <typename T, int D>
__device__ __forceinline__ void careful_row(const sg_attn_masked_args& a, int row, int h, int lo, int hi, int doc, int d0, int d1,
                                         int lane) {
  constexpr int N = (D + 63) / 64;
  const int kvh = h / (a.heads / a.kv_heads);
  const float slope = a.slopes ? a.slopes[h] : 0.0f;
  const T* q = static_cast<const T*>(a.q) + (int64_t)row * a.ldq + h * a.hd;
  const T* kp = static_cast<const T*>(a.k) + kvh * a.hd;
  const T* vp = static_cast<const T*>(a.v) + kvh * a.hd;
  float qv[N], o[N] = {};
#pragma unroll
  for (int i = 0; i < N; i++) qv[i] = lane + 64 * i < a.hd ? elem<T>::to(q[lane + 64 * i]) : 0.0f;
  auto score = [&](int j) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++)
      if (lane + 64 * i < a.hd) s = __builtin_fmaf(qv[i], elem<T>::to(kp[(int64_t)j * a.ldk + lane + 64 * i]), s);
    return score_of<T>(a, sgp::wave_sum(s), slope, row - j);
  };
  float m = -INFINITY, l = 0.0f;
  for (int j = lo; j < hi; j++)
    if (!a.docs || a.docs[j] == doc) m = fmaxf(m, score(j));
  for (int j = lo; j < hi; j++) {
    if (a.docs && a.docs[j] != doc) continue;
    const float p = __builtin_amdgcn_exp2f(score(j) - m);
    l += p;
#pragma unroll
    for (int i = 0; i < N; i++)
      if (lane + 64 * i < a.hd) o[i] = __builtin_fmaf(p, elem<T>::to(vp[(int64_t)j * a.ldv + lane + 64 * i]), o[i]);
  }
  T* out = static_cast<T*>(a.out) + (int64_t)row * a.ldo + h * a.hd;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int d = lane + 64 * i;
    if (d >= d0 && d < d1) out[d] = elem<T>::from(o[i] / l);
  }
}

struct yes {
  static constexpr bool value = true;
};
struct no {
  static constexpr bool value = false;
};

// Every wave's copies have landed and its LDS reads are done, in all waves.
__device__ __forceinline__ void publish() {
  sg_wait_vmcnt<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <typename T, int D, int RW, int KW>
__global__ __launch_bounds__(kNT, D == 256 ? 1 : 2) void k_attn_masked(sg_attn_masked_args a,
                                                                                                  int row_tiles) {
  typedef form<T, D, RW, KW> F;
  typedef typename mul<T>::type M;
  typedef __attribute__((address_space(3))) void* lds_ptr;
  typedef __attribute__((address_space(3))) s16x4_t* lds_s4;
  constexpr int C = D / 8;      // 16-byte pieces of an LDS row
  constexpr int KS = D / 16;    // k-steps of a score
  constexpr int DB = D / kSub;  // 32-dim blocks of an output
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  __shared__ int range[kWaves][4];
  __shared__ uint32_t scan;
  __shared__ int first_e;
  __shared__ float ml[kWaves][2][kSub];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = w % RW, kw = w / RW;
  const int n = lane & 31, g = lane >> 5;
  const int h = blockIdx.x % a.heads, tile_i = (int)(blockIdx.x / a.heads);
  const int row0 = (a.causal ? row_tiles - 1 - tile_i : tile_i) * F::BM;  // causal: the long rows first
  const int kvh = h / (a.heads / a.kv_heads);
  const int row = row0 + kSub * rw + n, rc = min(row, a.rows - 1);

  // ---- the row's keys ----
  view me;
  {
    const int last = min(row0 + F::BM, a.rows) - 1;
    const int i0 = sgp::find_seq(a.off, a.n_seq, row0, lane), i1 = sgp::find_seq(a.off, a.n_seq, last, lane);
    int lo = max(i0, 0), hi = max(i1, lo);
    while (lo < hi) {
      const int mid = lo + (hi - lo + 1) / 2;
      if (a.off[mid] <= rc) lo = mid;
      else hi = mid - 1;
    }
    const int s0 = sgp::clamp_row(a.off[lo], a.rows), s1 = sgp::clamp_row(a.off[lo + 1], a.rows);
    me.live = row < a.rows && s0 <= row && row < s1;
    me.lo = s0;
    me.hi = s1;
    if (a.causal) {
      const int free = a.prefix ? s0 + min(max(a.prefix[lo], 0), max(s1 - s0, 0)) : 0;
      me.hi = min(s1, max(rc + 1, free));
    }
    if (a.window > 0) {
      const int wd = min(a.window, a.rows);
      me.lo = max(me.lo, rc - wd + 1);
      me.hi = min(me.hi, rc + wd);
    }
    me.doc = a.docs ? a.docs[rc] : 0;
    if (!me.live || me.doc < 0) {
      me.lo = INT32_MAX;
      me.hi = 0;
    }
  }
  {
    int v[4] = {me.lo, -me.hi, me.hi ? me.doc : INT32_MAX, me.hi ? -me.doc : INT32_MAX};
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1)
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = min(v[i], __shfl_xor(v[i], o));
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < 4; i++) range[w][i] = v[i];
    if (tid == 0) first_e = INT32_MIN;
  }
  __syncthreads();
  int all[4];
#pragma unroll
  for (int i = 0; i < 4; i++)
    all[i] = __builtin_amdgcn_readfirstlane(min(min(range[0][i], range[1][i]), min(range[2][i], range[3][i])));
  const int kend = -all[1];
  const int kbeg = all[0] < kend ? all[0] & ~(kSub - 1) : 0;
  const int nt = all[0] < kend ? (kend - kbeg + F::BK - 1) / F::BK : 0;

  // ---- Q as the B operand: lane (n, g), step ks: dims 16 ks + 8 g .. + 7 of the row ----
  s16x8_t q[F::PARTS][KS];
  float qf = a.scale;  // a score's factor
  {
    const T* qp = static_cast<const T*>(a.q) + (int64_t)rc * a.ldq + h * a.hd + 8 * g;
    if constexpr (F::F32) {
      float x[KS][8];
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        const bool on = 16 * ks + 8 * g < a.hd;
#pragma unroll
        for (int i = 0; i < 2; i++)
          *reinterpret_cast<f32x4_t*>(&x[ks][4 * i]) =
              on ? *reinterpret_cast<const f32x4_t*>(qp + 16 * ks + 4 * i) : f32x4_t{0, 0, 0, 0};
      }
      float top = finite_top<8 * KS>(&x[0][0]);
      top = fmaxf(top, __shfl_xor(top, 32));
      const int e = row_exp(top);
#pragma unroll
      for (int ks = 0; ks < KS; ks++) halves(x[ks], pow2(kTop - e), q[0][ks], q[F::PARTS - 1][ks]);
      qf *= pow2(e - kTop);
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
        q[0][ks] = 16 * ks + 8 * g < a.hd ? *reinterpret_cast<const s16x8_t*>(qp + 16 * ks) : s16x8_t{};
    }
  }
  const bool capped = a.softcap > 0.0f;
  const float before = capped ? qf / a.softcap : qf * kLog2e;
  const float after = a.softcap * kLog2e;
  const float slope = a.slopes ? a.slopes[h] * kLog2e : 0.0f;

  // ---- tiles ----
  // The first tile from t on that may hold a key of a document of this
  // workgroup's rows (nt: none).
  uint32_t mask = 0;
  int scan0 = 0, scan1 = 0;
  auto next = [&](int t) {
    if (!a.docs) return t;
    while (t < nt) {
      if (t >= scan1) {
        scan0 = t;
        scan1 = t + kScanTiles;
        __syncthreads();
        if (tid == 0) scan = 0;
        __syncthreads();
        const int end = min(kend, kbeg + scan1 * F::BK);
        for (int j = kbeg + scan0 * F::BK + tid; j < end; j += kNT) {
          const int d = a.docs[j];
          if (d >= all[2] && -d >= all[3]) atomicOr(&scan, 1u << ((j - kbeg) / F::BK - scan0));
        }
        __syncthreads();
        mask = __builtin_amdgcn_readfirstlane(scan);
      }
      const uint32_t left = mask >> (t - scan0);
      if (left) return t + __builtin_ctz(left);
      t = scan1;
    }
    return nt;
  };

  // Tile t's K and V into LDS.  Keys past the tensors' end repeat the last row,
  // pieces past head_dim the last piece: they meet zeros of Q, or make outputs
  // that are not stored.
  float* const key_mul = reinterpret_cast<float*>(lds + F::STAGES * F::TILE);  // [3][BK]: K's power, V's exponent, V's power
  int e_ref = INT32_MIN;  // float32: the largest exponent of the first 32 keys' V
  auto stage = [&](int st, int t) {
    const int k0 = kbeg + t * F::BK;
    if constexpr (!F::F32) {
      constexpr int COPIES = F::HALF / 1024 / kWaves;
      const uint32_t base = (uint32_t)(uintptr_t)(lds_ptr)(lds + st * F::TILE);
      const i32x4_t rk = sg_raw_rsrc(static_cast<const T*>(a.k) + (int64_t)k0 * a.ldk + kvh * a.hd);
      const i32x4_t rv = sg_raw_rsrc(static_cast<const T*>(a.v) + (int64_t)k0 * a.ldv + kvh * a.hd);
#pragma unroll
      for (int i = 0; i < COPIES; i++) {
        const int at = (w * COPIES + i) * 64 + lane, r = at / C, s = at % C;
        const int from = min(r, a.rows - 1 - k0);
        const int ck = min(s ^ swz_k<D>(r), a.hd / 8 - 1), cv = min(s ^ swz_v<D>(r), a.hd / 8 - 1);
        const uint32_t dst = base + (uint32_t)(w * COPIES + i) * 1024u;
        sg_lds_copy16(dst, (uint32_t)(from * (int)a.ldk + ck * 8) * 2u, rk, 0);
        sg_lds_copy16(dst + F::HALF, (uint32_t)(from * (int)a.ldv + cv * 8) * 2u, rv, 0);
      }
    } else {
      constexpr int CL = C / 8;  // pieces of eight values a thread takes of a row, eight threads a row
      const int j = tid & 7;
#pragma unroll
      for (int p = 0; p < F::BK / (kNT / 8); p++) {
        const int r = p * (kNT / 8) + tid / 8;
        const int64_t from = min(k0 + r, a.rows - 1);
#pragma unroll
        for (int v = 0; v < 2; v++) {
          const T* src = v ? static_cast<const T*>(a.v) + from * a.ldv : static_cast<const T*>(a.k) + from * a.ldk;
          float x[CL][8];
#pragma unroll
          for (int i = 0; i < CL; i++) {
            const int c = j + 8 * i;
            const bool on = c < a.hd / 8;
#pragma unroll
            for (int u = 0; u < 2; u++)
              *reinterpret_cast<f32x4_t*>(&x[i][4 * u]) =
                  on ? *reinterpret_cast<const f32x4_t*>(src + kvh * a.hd + 8 * c + 4 * u) : f32x4_t{0, 0, 0, 0};
          }
          float top = finite_top<8 * CL>(&x[0][0]);
#pragma unroll
          for (int o = 4; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
          int e = row_exp(top);
          if (v) {
            if (e_ref == INT32_MIN) {
              if (j == 0 && top > 0.0f) atomicMax(&first_e, e);
              __syncthreads();
              e_ref = __builtin_amdgcn_readfirstlane(first_e);
              if (e_ref == INT32_MIN) e_ref = 0;
            }
            e = min(max(e, max(e_ref - kSpan, -kLim)), min(e_ref + kSpan, kLim));
          }
#pragma unroll
          for (int i = 0; i < CL; i++) {
            const int c = j + 8 * i;
            s16x8_t hi, lo;
            halves(x[i], pow2(kTop - e), hi, lo);
            unsigned char* dst =
                lds + v * F::PARTS * F::HALF + (r * C + (c ^ (v ? swz_v<D>(r) : swz_k<D>(r)))) * 16;
            *reinterpret_cast<s16x8_t*>(dst) = hi;
            *reinterpret_cast<s16x8_t*>(dst + F::HALF) = lo;
          }
          if (j == 0) {
            if (v) {
              key_mul[F::BK + r] = (float)(e - e_ref);
              key_mul[2 * F::BK + r] = pow2(e_ref - e);
            } else {
              key_mul[r] = pow2(e - kTop);
            }
          }
        }
      }
    }
  };

  f32x16_t o[DB] = {};
  float m = -INFINITY, l = 0.0f;  // l: this lane's keys only

  // The scores of 32 keys from k on, at row kr of the LDS tile, and their part of o.
  auto block = [&](const unsigned char* tile, int k, int kr, auto masked) {
    constexpr bool MASKED = decltype(masked)::value;
    f32x16_t s = {};
    const unsigned char* kt = tile + (kr + n) * (D * 2);
    const int sk = swz_k<D>(kr + n);
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      const unsigned char* p = kt + (((2 * ks + g) ^ sk) << 4);
      const s16x8_t kh = *reinterpret_cast<const s16x8_t*>(p);
      if constexpr (F::F32) {
        const s16x8_t kl = *reinterpret_cast<const s16x8_t*>(p + F::HALF);
        s = mfma32<M>(kl, q[0][ks], s);
        s = mfma32<M>(kh, q[F::PARTS - 1][ks], s);
      }
      s = mfma32<M>(kh, q[0][ks], s);
    }
    // Register r: key 8 (r / 4) + 4 g + r % 4.
    float pv[16];
    if constexpr (F::F32) {
#pragma unroll
      for (int b = 0; b < 4; b++) {
        const f32x4_t km = *reinterpret_cast<const f32x4_t*>(key_mul + kr + 8 * b + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; i++) s[4 * b + i] *= km[i];
      }
    }
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] *= before;
    if (capped) {
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = tanh_of<F::F32>(s[r]) * after;
    }
    if (a.slopes) {
      const float far = (float)(row - k - 4 * g);
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = __builtin_fmaf(-slope, fabsf(far - (float)(8 * (r >> 2) + (r & 3))), s[r]);
    }
    if constexpr (F::F32) {
#pragma unroll
      for (int b = 0; b < 4; b++) {
        const f32x4_t ve = *reinterpret_cast<const f32x4_t*>(key_mul + F::BK + kr + 8 * b + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; i++) s[4 * b + i] += ve[i];
      }
    }
    if constexpr (MASKED) {
      const int lo = me.lo - k - 4 * g, hi = me.hi - k - 4 * g;
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int c = 8 * (r >> 2) + (r & 3);
        s[r] = c >= lo && c < hi ? s[r] : -INFINITY;
      }
      if (a.docs) {
        const int d = a.docs[min(k + n, a.rows - 1)];
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = __shfl(d, 8 * (r >> 2) + 4 * g + (r & 3)) == me.doc ? s[r] : -INFINITY;
      }
    }
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; r++) top = fmaxf(top, s[r]);
    top = fmaxf(top, __shfl_xor(top, 32));
    if (__ballot(top > m + kSlack)) {  // (-inf + 8 is -inf: a row's first visible key raises it)
      const float to = fmaxf(m, top);
      const float by = to > m ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
      m = to;
      l *= by;
#pragma unroll
      for (int d = 0; d < DB; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] *= by;
    }
    const float from = (m == -INFINITY ? 0.0f : m) - mul<T>::shift;
#pragma unroll
    for (int r = 0; r < 16; r++) pv[r] = __builtin_amdgcn_exp2f(s[r] - from);
    if constexpr (F::F32) {
#pragma unroll
      for (int b = 0; b < 4; b++) {
        const f32x4_t vw = *reinterpret_cast<const f32x4_t*>(key_mul + 2 * F::BK + kr + 8 * b + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; i++) l = __builtin_fmaf(pv[4 * b + i], vw[i], l);
      }
    } else {
#pragma unroll
      for (int r = 0; r < 16; r++) l += pv[r];
    }
    // P^T, 16 keys a step: the lane's registers 8 st .. + 7.
    s16x8_t p[F::PARTS][2];
#pragma unroll
    for (int st = 0; st < 2; st++) {
      if constexpr (F::F32) {
        halves(pv + 8 * st, 1.0f, p[0][st], p[F::PARTS - 1][st]);
      } else {
        chunk<M> c;
#pragma unroll
        for (int i = 0; i < 8; i++) c.v[i] = elem<M>::from(pv[8 * st + i]);
        p[0][st] = __builtin_bit_cast(s16x8_t, c);
      }
    }
    // V^T: lane dim 32 d + n, keys 16 st + 4 g + 0..3 and + 8; the transposing load
    // takes from lane i of 16 the row i / 4's dims 4 (i % 4) .. + 3.
    const int vr = kr + 4 * g + ((lane & 15) >> 2);
    const int vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), vb = (lane & 1) * 8;
    const unsigned char* vt = tile + F::PARTS * F::HALF;
#pragma unroll
    for (int d = 0; d < DB; d++) {
#pragma unroll
      for (int st = 0; st < 2; st++) {
        s16x8_t vf[F::PARTS];
#pragma unroll
        for (int part = 0; part < F::PARTS; part++) {
          s16x4_t half[2];
#pragma unroll
          for (int u = 0; u < 2; u++) {
            const int r = vr + 16 * st + 8 * u;
            const unsigned char* at = vt + part * F::HALF + r * (D * 2) + (((4 * d + vc) ^ swz_v<D>(r)) << 4) + vb;
            half[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(at));
          }
          vf[part] = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
        if constexpr (F::F32) {
          o[d] = mfma32<M>(vf[F::PARTS - 1], p[0][st], o[d]);
          o[d] = mfma32<M>(vf[0], p[F::PARTS - 1][st], o[d]);
        }
        o[d] = mfma32<M>(vf[0], p[0][st], o[d]);
      }
    }
  };
  auto compute = [&](int st, int t) {
    const unsigned char* tile = lds + st * F::TILE;
#pragma unroll
    for (int i = 0; i < F::NSUB; i++) {
      const int kr = (kw + KW * i) * kSub, k = kbeg + t * F::BK + kr;
      if (!__ballot(me.lo < k + kSub && me.hi > k)) continue;
      if (!a.docs && !__ballot(me.live && (me.lo > k || me.hi < k + kSub)))
        block(tile, k, kr, no{});
      else
        block(tile, k, kr, yes{});
    }
  };

  if constexpr (F::STAGES == 2) {
    int t = next(0), st = 0;
    if (t < nt) stage(0, t);
    while (t < nt) {
      const int tn = next(t + 1);
      publish();
      if (tn < nt) stage(st ^ 1, tn);
      compute(st, t);
      st ^= 1;
      t = tn;
    }
  } else {
    for (int t = next(0); t < nt; t = next(t + 1)) {
      __syncthreads();
      stage(0, t);
      if constexpr (F::F32) __syncthreads();
      else publish();
      compute(0, t);
    }
  }
  l += __shfl_xor(l, 32);

  // ---- the waves that shared these rows ----
  int db0 = 0, db1 = DB;
  if constexpr (KW > 1) {
    if (g == 0) {
      ml[w][0][n] = m;
      ml[w][1][n] = l;
    }
    publish();  // nobody reads the tiles any more
    float top = m;
#pragma unroll
    for (int i = 0; i < KW; i++) top = fmaxf(top, ml[i * RW + rw][0][n]);
    const float from = top == -INFINITY ? 0.0f : top;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < KW; i++) l += ml[i * RW + rw][1][n] * __builtin_amdgcn_exp2f(ml[i * RW + rw][0][n] - from);
    const float by = __builtin_amdgcn_exp2f(m - from);
    float* mine = reinterpret_cast<float*>(lds) + w * (kSub * D) + lane;
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
      for (int r = 0; r < 16; r++) mine[(d * 16 + r) * 64] = o[d][r] * by;
    __syncthreads();
    constexpr int EACH = (DB + KW - 1) / KW;
    db0 = min(DB, kw * EACH);
    db1 = min(DB, db0 + EACH);
#pragma unroll
    for (int d = 0; d < EACH; d++) {
      if (db0 + d >= db1) continue;
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const float* from0 = reinterpret_cast<const float*>(lds) + ((db0 + d) * 16 + r) * 64 + lane;
        float s = from0[rw * (kSub * D)];
#pragma unroll
        for (int i = 1; i < KW; i++) s += from0[(i * RW + rw) * (kSub * D)];
        o[d][r] = s;
      }
    }
  }

  // ---- out ----
  const bool sees = me.live && l != 0.0f;  // (a NaN is not 0)
  const float inv = sees ? 1.0f / l : 0.0f;
  const float back = F::F32 && e_ref != INT32_MIN ? pow2(e_ref - kTop) : 1.0f;
  bool bad = false;
  T* out = static_cast<T*>(a.out) + (int64_t)rc * a.ldo + h * a.hd;
  constexpr int KEEP = KW > 1 ? (DB + KW - 1) / KW : DB;
#pragma unroll
  for (int d = 0; d < KEEP; d++) {
    if (db0 + d >= db1) continue;
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const int at = (db0 + d) * kSub + 8 * b + 4 * g;
      if (at >= a.hd) continue;
      struct alignas(4 * sizeof(T)) { T v[4]; } piece;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float x = sees ? o[d][4 * b + i] * inv * back : 0.0f;
        bad |= !(fabsf(x) < INFINITY);
        piece.v[i] = elem<T>::from(x);
      }
      if (me.live) *reinterpret_cast<decltype(piece)*>(out + at) = piece;
    }
  }
  uint64_t again = __ballot(bad && me.live);
  again = (again | (again >> 32)) & 0xffffffffu;
  while (again) {
    const int i = __builtin_ctzll(again);
    again &= again - 1;
    careful_row<T, D>(a, row0 + kSub * rw + i, h, __builtin_amdgcn_readlane(me.lo, i), __builtin_amdgcn_readlane(me.hi, i),
                      __builtin_amdgcn_readlane(me.doc, i), db0 * kSub, min(a.hd, db1 * kSub), lane);
  }
}

template <typename T, int D, int RW, int KW>
hipError_t launch(const sg_attn_masked_args& a, hipStream_t s) {
  typedef form<T, D, RW, KW> F;
  const int64_t tiles = ((int64_t)a.rows + F::BM - 1) / F::BM;
  if (tiles * a.heads > INT32_MAX) return hipErrorInvalidValue;
  hipLaunchKernelGGL((k_attn_masked<T, D, RW, KW>), dim3((unsigned)(tiles * a.heads)), dim3(kNT), F::LDS, s, a, (int)tiles);
  return hipGetLastError();
}

template <typename T, int D>
hipError_t by_form(const sg_attn_masked_args& a, hipStream_t s) {
  const int64_t wide = ((int64_t)a.rows + 127) / 128 * a.heads;
  if (wide >= 512) return launch<T, D, 4, 1>(a, s);
  if constexpr (__is_same(T, float) && D == 256) return launch<T, D, 2, 2>(a, s);
  else return launch<T, D, 1, 4>(a, s);
}

template <typename T>
hipError_t by_dim(const sg_attn_masked_args& a, hipStream_t s) {
  return a.hd <= 64 ? by_form<T, 64>(a, s) : a.hd <= 128 ? by_form<T, 128>(a, s) : by_form<T, 256>(a, s);
}

}  // namespace

namespace sgk {

hipError_t attention_masked(const sg_attn_masked_args& a, int dtype, hipStream_t s) {
  if (dtype == SG_F32) return by_dim<float>(a, s);
  if (dtype == SG_F16) return by_dim<_Float16>(a, s);
  return by_dim<bf16_t>(a, s);
}

}  // namespace sgk
