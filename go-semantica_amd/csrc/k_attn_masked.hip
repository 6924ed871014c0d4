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
// 16-bit types go to LDS by buffer_load ... lds, a tile ahead.  Their weights are rounded to
// the type for the second product and summed as they are multiplied: against 64 bits
// bf16 outputs are off by 2.1e-3 (1.6e-3 with float32 weights, which is the outputs' own
// rounding), fp16 by 2.6e-4 (2.1e-4); weights of two halves would be half as much matrix work
// again.
//
// float32 operands are split into two fp16 halves each, hi + lo, and products run as hi.hi +
// hi.lo + lo.hi (22 bits of each operand; the dropped lo.lo is 2^-22 of the product).
// Every row of Q, K and V is first brought to the same power of two, so fp16's
// range does not matter: Q's and K's powers multiply the score, V's is added to the
// score that the weight is formed from (p' = 2^(s + e_j - m'), |v'| alike for all
// keys), and the softmax's sum takes it out again (sum p' 2^-e_j).  A value keeps
// 22 bits down to 2^-15 of its row's largest and 2^-37 of the largest below that; p', which
// has the maximum at 2^5 or above, 22 bits down to 2^-9 and 2^-25 below.
//
// A hidden key has weight zero, and zero times an infinity or a NaN in its value
// is a NaN.  Instead of looking at every value, a wave looks at its outputs: rows
// that did not come out finite are computed again one key at a time from the
// visible keys only (careful_row; some 400 times slower at 1000 tokens, so tiles leave
// out what lies around the batch, where padding may hold anything).  That also covers
// float32 values past the fp16 halves' reach (q and k above 2^113, values 2^53 times
// the first keys').
//
// What bounds it.  A wave's products and exponentials come one after the other, and two
// or three waves a SIMD fill each other's gaps only in part: at 4 x 4096 bf16 tokens the
// matrix core is busy 36 % of the time and the vector unit 60 %.  A score costs an
// exponential (16 cycles of a wave; a multiplication 2.6) and about ten other vector
// instructions under a cap beside 4 head_dim flops, so few of them per score is what the
// code goes for: the range check once a tile and wave, bf16 under a cap without a maximum,
// tanh as a polynomial, the sum of weights as a dot product of the packed ones.  Measured
// (us, and the rate of the visible pairs' 4 head_dim flops):
//   4 x 4096, bf16, causal, cap, 32 heads over 8 of 128            708   776 TFLOP/s
//   8 of 1024 .. 2048, fp16, causal, prefix, 16 over 8 of 128      155   625
//   16391 rows, documents of 900, bf16, distance bias, 12 of 64    159   317
//   64 x 512, float32, window of 256, 3 over 1 of 256              218   178
// (690 to 730 for the first over several cards.  Its scores stay below 0.35 of the cap of 50,
// so tanh is the polynomial throughout: with a cap of 20, where half of the blocks take the
// exact form, 766 for 743 on one card, with a cap of 8 789, without one 616.)
// float32 (three products each; 372 TFLOP/s is the matrix cores' limit) waits about
// half its time: a workgroup's eight waves load, halve, multiply in step, and no second
// one fits beside two stages of its tiles (two workgroups of 64 rows and one stage each:
// 265 us).  Its LDS reads of V meet two-way conflicts with 16 queries; a xor of three
// bits that avoids them costs more in addresses (241 us against 236).  Tried as well:
// eight 32-row waves a workgroup (4 x 4096 683 us for 697, but documents 213 for 162),
// causal tiles sorted by length (193 for 171 at the prefix case: L2 locality lost), the
// bias as the products' start value (175 for 163), s_setprio round the products (equal).
//
// Two forms (by_form has the rule): waves with 32 (16) rows of their own, 128 (64) to
// a workgroup, or, for batches with too few rows to fill the GPU, waves that share 32
// rows and split each tile's keys between them, joined through LDS at the end.
#include <algorithm>

#include "semantica_gpu.h"
#include "sg_kernels.h"
#include "sg_packed.h"

namespace {

using sgp::bf16_t;
using sgp::bf16x8_t;
using sgp::chunk;
using sgp::elem;

constexpr int kSub = 32;  // keys of a block: one or two matrix core tiles
constexpr float kLog2e = 1.44269504088896340736f;
// A row's maximum is raised (and its sums rescaled) only when a score passes it by
// this many powers of two, so most tiles rescale nothing; weights stay below 2^8.
constexpr float kSlack = 8.0f;
constexpr int kScanWords = 64;  // 32 tiles each: one look at the document ids

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

// The matrix core tile of QT queries: accumulator type, and one step of M's type.
template <int QT>
struct core;
template <>
struct core<32> {
  typedef f32x16_t acc;
  static constexpr int REGS = 16;
  template <typename M>
  static __device__ __forceinline__ acc step(s16x8_t a, s16x8_t b, acc c) {
    if constexpr (__is_same(M, bf16_t))
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
  }
};
template <>
struct core<16> {
  typedef f32x4_t acc;
  static constexpr int REGS = 4;
  template <typename M>
  static __device__ __forceinline__ acc step(s16x8_t a, s16x8_t b, acc c) {
    if constexpr (__is_same(M, bf16_t))
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
  }
};

// What a row's piece index is xor-ed by.  An LDS cycle serves 256 bytes: 16 lanes of a
// K load (16 rows, one piece), or 32 lanes of a transposing V load (four rows, four
// pieces each).  Rows of 64 dims are 128 bytes, two to a cycle's banks.  (An xor of
// three bits, for cycles of 128 bytes, doubled the LDS time.)
template <int D>
__device__ __forceinline__ constexpr int swz_k(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }
template <int D>
__device__ __forceinline__ constexpr int swz_v(int row) { return D == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }

constexpr int kTop = 13;  // rows are brought to 2^13 .. 2^14 before they are halved
constexpr int kLim = 110;
// V's exponents are kept within this of the workgroup's first keys': 2^-e then sums
// without overflow, and a weight that underflows beside a row of larger values
// is below 2^-26 of the softmax's sum as well.  A row of V below that span is held to
// 2^-88 of the first keys' power, so an output above 2^-51 of it is as exact as any;
// smaller ones (the large first keys were hidden from it) careful_row takes.
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
    asm volatile("");  // (a branch, not sixteen selects for everyone)
    top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) top = fmaxf(top, fabsf(x[i]) < INFINITY ? fabsf(x[i]) : 0.0f);
  }
  return top;
}

// Eight values times `by` (a power of two), as fp16 halves: hi = fp16(x by) and lo =
// fp16(x by - hi), each rounded once, two instructions a value.
__device__ __forceinline__ void halves(const float* x, float by, s16x8_t& hi, s16x8_t& lo) {
  typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
  u32x4_t h, l;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t hh, ll;
    asm("v_fma_mixlo_f16 %0, %2, %4, 0\n\t"
        "v_fma_mixhi_f16 %0, %3, %4, 0\n\t"
        "v_fma_mixlo_f16 %1, %2, %4, -%0 op_sel_hi:[0,0,1]\n\t"
        "v_fma_mixhi_f16 %1, %3, %4, -%0 op_sel:[0,0,1] op_sel_hi:[0,0,1]"
        : "=&v"(hh), "=&v"(ll)
        : "v"(x[2 * i]), "v"(x[2 * i + 1]), "v"(by));
    h[i] = hh;
    l[i] = ll;
  }
  hi = __builtin_bit_cast(s16x8_t, h);
  lo = __builtin_bit_cast(s16x8_t, l);
}

// The sum of the eight 16-bit values of p, added to l.
template <typename M>
__device__ __forceinline__ float add_up(s16x8_t p, float l) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (__is_same(M, bf16_t)) {
      typedef __bf16 b2 __attribute__((ext_vector_type(2)));
      const b2 ones = {(__bf16)1.0f, (__bf16)1.0f};
      const short two[2] = {p[2 * i], p[2 * i + 1]};
      l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, two), ones, l, false);
    } else {
      typedef _Float16 h2 __attribute__((ext_vector_type(2)));
      const h2 ones = {(_Float16)1, (_Float16)1};
      const short two[2] = {p[2 * i], p[2 * i + 1]};
      l = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, two), ones, l, false);
    }
  }
  return l;
}

// tanh of the scores of a block.  Below a limit an odd polynomial, Chebyshev's in x^2:
// degree 2 below 0.35 (16-bit types: 3e-6 relative, under a cap of 50 scores to 17
// within 5e-5), degree 5 below 0.5 (float32: 9e-8); no exponential or reciprocal,
// each of which costs six multiplications' time.  A block with a larger score takes
// the exact forms.
constexpr float kNear16 = 0.35f, kNear32 = 0.5f;
constexpr float kTanh16[3] = {0.999997118f, -0.332908736f, 0.123943759f};
__device__ __forceinline__ float tanh_near32(float x) {
  const float z = x * x;
  float p = __builtin_fmaf(z, -0.00661201408f, 0.021273822f);
  p = __builtin_fmaf(z, p, -0.0538932246f);
  p = __builtin_fmaf(z, p, 0.133329003f);
  p = __builtin_fmaf(z, p, -0.333333241f);
  p = __builtin_fmaf(z, p, 1.0f);
  return x * p;
}
// bf16 has float32's exponents, so under a cap its weights need no running maximum, unless
// a negative slope lets scores grow with the distance: 2^+-kMostCap2 (a bias only lowers
// weights, and a query's own not at all) and sums of them times values below 2^40 are in range
// (a value that overflows the sum makes an output that is not finite, and careful_row takes
// it; so it does outputs below 2^-110 before the division by a sum of weights that is small,
// where products of tiny values underflow).
constexpr float kMostCap2 = 80.0f;
// Lambert's continued fraction to seven levels below 1.5 (relative error 5e-8 at its
// end), and 1 - 2 / (e^2x + 1) above, where the second term's rounding no longer shows.
__device__ __forceinline__ float tanh_f32(float x) {
  const float e = __builtin_amdgcn_exp2f(x * (2.0f * kLog2e));
  const float far = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
  const float z = x * x;
  const float num = x * __builtin_fmaf(__builtin_fmaf(z + 378.0f, z, 17325.0f), z, 135135.0f);
  const float den = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(28.0f, z, 3150.0f), z, 62370.0f), z, 135135.0f);
  const float r = __builtin_amdgcn_rcpf(den), q = num * r;
  const float near = __builtin_fmaf(__builtin_fmaf(-q, den, num), r, q);
  return fabsf(x) < 1.5f ? near : far;
}

// The largest over the lanes of a query (lanes n, n + QT, ...).
template <int QT>
__device__ __forceinline__ float query_max(float v) {
  if constexpr (QT == 16) {
    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
  }
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}

// A form: QT queries a wave, RW groups of them and KW shares of each tile's keys.
template <typename T, int D_, int QT_, int RW_, int KW_>
struct form {
  static constexpr int D = D_, QT = QT_, RW = RW_, KW = KW_;
  static constexpr int NW = RW * KW, NT = NW * SG_WAVE;
  static constexpr bool F32 = __is_same(T, float);
  static constexpr int PARTS = mul<T>::parts;
  static constexpr int NSUB = KW > 1 || D == 256 || (F32 && D == 128 && QT == 32) ? 1 : 2;  // 32-key blocks a wave takes of a tile
  static constexpr int KB = kSub * NSUB;  // which are adjacent, and taken together
  static constexpr int BK = kSub * KW * NSUB, BM = QT * RW;
  static constexpr int HALF = BK * D * 2;             // bytes of one tile's K (or V), one part
  static constexpr int TILE = 2 * PARTS * HALF;       // K and V
  // float32 rows of 64 dims hold no tile ahead: its registers are a third workgroup's.
  static constexpr int STAGES = (!F32 || (KW == 1 && D != 64)) && 2 * TILE <= (128 << 10) ? 2 : 1;
  static constexpr int KEYS = F32 ? STAGES * 3 * BK * 4 : 0;  // per-key powers of a float32 tile
  static constexpr int JOIN = KW > 1 ? NW * QT * D * 4 : 0;
  static constexpr int LDS = (STAGES * TILE + KEYS) > JOIN ? (STAGES * TILE + KEYS) : JOIN;
  static constexpr int WAVES = (QT == 32 && D == 256) || (NW == 4 && KW > 1) ? 1 : D == 64 && (!F32 || KW == 1) ? 3 : 2;  // a SIMD has registers for
  // Lane (n, g): query n; of a 32-key block, register r is key KSTR (r / 4) + 4 g + r % 4.
  static constexpr int G = SG_WAVE / QT, KSTR = 4 * G;
  static constexpr int SR = KB / G;            // a lane's scores of its keys of a tile
  static constexpr int KDIM = 8 * G;           // dims of a score step; keys of an output step
  static constexpr int KS = D / KDIM, DB = D / QT, PS = KB / KDIM;
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
  if (a.softcap > 0.0f) s = a.softcap * tanh_f32(s / a.softcap);
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
  // The weights' sum comes first, so that what is added up is a mean: values near the type's
  // end leave no range.
  float m = -INFINITY, l = 0.0f;
  for (int j = lo; j < hi; j++) {
    if (a.docs && a.docs[j] != doc) continue;
    const float s = score(j), to = fmaxf(m, s), from = to == -INFINITY ? 0.0f : to;
    l = l * __builtin_amdgcn_exp2f(m - from) + __builtin_amdgcn_exp2f(s - from);
    m = to;
  }
  const float inv = 1.0f / l;
  for (int j = l != 0.0f ? lo : hi; j < hi; j++) {  // (scores of -inf alone: zeros, as where all is hidden)
    if (a.docs && a.docs[j] != doc) continue;
    const float p = __builtin_amdgcn_exp2f(score(j) - m) * inv;
#pragma unroll
    for (int i = 0; i < N; i++)
      if (lane + 64 * i < a.hd) o[i] = __builtin_fmaf(p, elem<T>::to(vp[(int64_t)j * a.ldv + lane + 64 * i]), o[i]);
  }
  T* out = static_cast<T*>(a.out) + (int64_t)row * a.ldo + h * a.hd;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int d = lane + 64 * i;
    if (d >= d0 && d < d1) out[d] = elem<T>::from(o[i]);
  }
}

// Every wave's copies have landed and its LDS reads are done, in all waves.
__device__ __forceinline__ void publish() {
  sg_wait_vmcnt<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <typename T, int D, int QT, int RW, int KW>
__global__ __launch_bounds__(RW * KW * SG_WAVE, (form<T, D, QT, RW, KW>::WAVES)) void k_attn_masked(
    sg_attn_masked_args a, int row_tiles) {
  typedef form<T, D, QT, RW, KW> F;
  typedef core<QT> X;
  typedef typename X::acc acc_t;
  typedef typename mul<T>::type M;
  typedef __attribute__((address_space(3))) void* lds_ptr;
  typedef __attribute__((address_space(3))) s16x4_t* lds_s4;
  constexpr int C = D / 8;      // 16-byte pieces of an LDS row
  constexpr int kNT = F::NT, kWaves = F::NW, G = F::G, KS = F::KS, DB = F::DB, SR = F::SR, R = X::REGS;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  __shared__ int range[kWaves][4];
  __shared__ uint32_t scan[kScanWords];
  __shared__ int first_e, raised;  // float32: the largest exponent of the first 32 keys' V; rows of V lie far below it
  __shared__ float ml[kWaves][2][QT];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = w % RW, kw = w / RW;
  const int n = lane % QT, g = lane / QT;
  // Workgroups go round the 8 XCDs: heads are dealt so that one XCD's are neighbours, which
  // share keys and values in its L2 (bf16, 4 x 4096, 32 heads over 8: 698 us against 705).
  const int each = a.heads / 8;
  const int h = a.heads % 8 == 0 ? (int)(blockIdx.x % 8) * each + (int)(blockIdx.x / 8) % each : (int)(blockIdx.x % a.heads);
  const int row0 = (a.causal ? row_tiles - 1 - (int)(blockIdx.x / a.heads) : (int)(blockIdx.x / a.heads)) * F::BM;  // causal: the long rows first
  const int kvh = h / (a.heads / a.kv_heads);
  const int row = row0 + QT * rw + n, rc = min(row, a.rows - 1);

  // ---- Q's loads go out first: lane (n, g), step ks: dims KDIM ks + 8 g .. + 7 of the row ----
  const T* const qp = static_cast<const T*>(a.q) + (int64_t)rc * a.ldq + h * a.hd;
  constexpr int QV = F::F32 ? 2 : 1;  // 16-byte loads of eight values
  f32x4_t qx[KS][QV];
#pragma unroll
  for (int ks = 0; ks < KS; ks++)
#pragma unroll
    for (int i = 0; i < QV; i++)
      qx[ks][i] = *reinterpret_cast<const f32x4_t*>(qp + min(F::KDIM * ks + 8 * g, a.hd - 8) + 4 * i);
  if (a.hd != D)
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int i = 0; i < QV; i++)
        if (F::KDIM * ks + 8 * g >= a.hd) qx[ks][i] = f32x4_t{0, 0, 0, 0};

  // ---- the row's keys ----
  view me;
  {
    int lo, s0, s1;
    sgp::row_seq(a.off, a.n_seq, row0, min(row0 + F::BM, a.rows) - 1, rc, lane, lo, s0, s1);
    s0 = sgp::clamp_row(s0, a.rows);
    s1 = sgp::clamp_row(s1, a.rows);
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
      me.hi = min(me.hi, rc + min(wd, a.rows - rc));
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
    for (int o = QT / 2; o >= 1; o >>= 1)
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = min(v[i], __shfl_xor(v[i], o));
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < 4; i++) range[w][i] = v[i];
    if (tid == 0) first_e = INT32_MIN, raised = 0;
  }
  __syncthreads();
  int all[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    all[i] = range[0][i];
#pragma unroll
    for (int v = 1; v < kWaves; v++) all[i] = min(all[i], range[v][i]);
    all[i] = __builtin_amdgcn_readfirstlane(all[i]);
  }
  const int kend = -all[1];
  const int kbeg = all[0] < kend ? all[0] & ~(kSub - 1) : 0;
  const int nt = all[0] < kend ? (kend - kbeg + F::BK - 1) / F::BK : 0;
  // The rows that tiles are read from: the sequences', whatever lies before and behind them
  // (as far as the offsets can be believed: never less than the keys that are seen).
  const int from_row = min(max(a.off[0], 0), all[0]), last_row = max(min(a.off[a.n_seq], a.rows), kend) - 1;

  // ---- Q as the B operand, its sign turned where the scale is negative ----
  s16x8_t q[F::PARTS][KS];
  float qf = fabsf(a.scale);  // a score's factor
  {
    if constexpr (F::F32) {
      float top = finite_top<8 * KS>(reinterpret_cast<const float*>(&qx[0][0]));
#pragma unroll
      for (int o = QT; o < SG_WAVE; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
      const int e = row_exp(top);
      const float by = a.scale < 0.0f ? -pow2(kTop - e) : pow2(kTop - e);
#pragma unroll
      for (int ks = 0; ks < KS; ks++) halves(reinterpret_cast<const float*>(&qx[ks][0]), by, q[0][ks], q[F::PARTS - 1][ks]);
      qf *= pow2(e - kTop);
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        q[0][ks] = __builtin_bit_cast(s16x8_t, qx[ks][0]);
        if (a.scale < 0.0f) q[0][ks] ^= (short)0x8000;
      }
    }
  }
  // A score in powers of two is what the matrix core gives times cs, or, under a
  // cap, cap2 times the tanh of that.
  const bool capped = a.softcap > 0.0f;
  const float cs = capped ? qf / a.softcap : qf * kLog2e;
  const float cap2 = a.softcap * kLog2e;
  // 16-bit types: cap2 tanh(s ce) = s (t0 + s^2 (t1 + s^2 t2)) where |s| <= near; ce is
  // cs, or 1 where its powers might leave float32's range and s is multiplied first.
  const bool apart = F::F32 || !(cs > 1e-5f && cs < 1e5f);
  // What a key's distance takes off a score.  16-bit types take it off ahead of cs, which
  // saves the multiplication; not float32, whose cs holds the row's own power of two (of a
  // row of zeros 2^-110, and the quotient would leave float32's range), nor a far-off cs.
  const bool early = !F::F32 && apart && (capped || a.slopes);  // scores are multiplied by cs ahead of all else
  const float after = F::F32 || capped || early ? 1.0f : cs;    // and by this behind it
  const float steep = a.slopes ? a.slopes[h] * kLog2e / after : 0.0f;
  const float ce = apart ? 1.0f : cs;
  const float t0 = cap2 * ce * kTanh16[0], t1 = cap2 * ce * ce * ce * kTanh16[1];
  const float t2 = cap2 * ce * ce * (ce * ce) * ce * kTanh16[2];
  const float near = F::F32 ? kNear32 : kNear16 / ce;
  const bool fixed = __is_same(T, bf16_t) && capped && cap2 <= kMostCap2 && (!a.slopes || a.slopes[h] >= 0.0f);

  // ---- tiles ----
  // The first tile from t on that may hold a key of a document of this
  // workgroup's rows (nt: none).  A look covers kScanWords * 32 tiles, four ids a
  // thread and load.
  int scan0 = 0, scan1 = 0;
  auto next = [&](int t) {
    if (!a.docs) return t;
    while (t < nt) {
      if (t >= scan1) {
        scan0 = t;
        scan1 = t + kScanWords * 32;
        __syncthreads();
        if (tid < kScanWords) scan[tid] = 0;
        __syncthreads();
        const int first = kbeg + scan0 * F::BK, count = min(kend - first, (scan1 - scan0) * F::BK);
        const int32_t* ids = a.docs + first;
        const bool whole = (reinterpret_cast<uintptr_t>(ids) & 15) == 0;
        constexpr int U = 4;  // loads in flight
        for (int j0 = 0; j0 < count; j0 += 4 * kNT * U) {
          i32x4_t d[U];
#pragma unroll
          for (int u = 0; u < U; u++) {
            const int j = j0 + 4 * (u * kNT + tid);
            d[u] = i32x4_t{-1, -1, -1, -1};
            if (whole && j + 4 <= count) {
              d[u] = *reinterpret_cast<const i32x4_t*>(ids + j);
            } else {
#pragma unroll
              for (int i = 0; i < 4; i++)
                if (j + i < count) d[u][i] = ids[j + i];
            }
          }
#pragma unroll
          for (int u = 0; u < U; u++) {
            const int tile = (j0 + 4 * (u * kNT + tid)) / F::BK;
            bool any = false;
#pragma unroll
            for (int i = 0; i < 4; i++) any |= d[u][i] >= all[2] && -d[u][i] >= all[3];
            // A tile's BK / 4 lanes lie together; the first of them speaks for all.
            constexpr int L = F::BK / 4;
            const uint64_t b = __ballot(any) >> (lane & ~(L - 1));
            if ((lane & (L - 1)) == 0 && (b & ((1ull << L) - 1))) atomicOr(&scan[tile >> 5], 1u << (tile & 31));
          }
        }
        __syncthreads();
      }
      const uint32_t left = __builtin_amdgcn_readfirstlane(scan[(t - scan0) >> 5]) >> ((t - scan0) & 31);
      if (left) return t + __builtin_ctz(left);
      t += 32 - ((t - scan0) & 31);
    }
    return nt;
  };

  // Tile t's K and V into LDS.  Keys before the first sequence or behind the last repeat
  // the row next to them (padding there may hold NaN, which would send every row of the
  // tile to careful_row), pieces past head_dim the last piece: they meet zeros of Q, or
  // make outputs that are not stored.
  float* const key_muls = reinterpret_cast<float*>(lds + F::STAGES * F::TILE);  // [stage][3][BK]: K's power, V's exponent, V's power
  int e_ref = INT32_MIN;  // first_e
  // 16-bit types: a copy is 64 pieces, RPC rows of the tile.  Row r of a tile is row
  // (w COPIES + i) RPC + lane / C; its piece index is xor-ed by swz(r), which is the
  // xor of the two terms' (their bits are apart), so all but an xor of a copy's
  // address is one lane offset and scalars.
  constexpr int COPIES = F::HALF / 1024 / kWaves, RPC = SG_WAVE / C;
  const uint32_t row_k = (uint32_t)(lane / C) * (uint32_t)a.ldk * 2u, row_v = (uint32_t)(lane / C) * (uint32_t)a.ldv * 2u;
  const uint32_t piece_k = (uint32_t)((lane % C) ^ swz_k<D>(lane / C)) * 16u;
  const uint32_t piece_v = (uint32_t)((lane % C) ^ swz_v<D>(lane / C)) * 16u;
  auto copy = [&](int st, int t) {
    const int k0 = kbeg + t * F::BK;
    const uint32_t base = (uint32_t)(uintptr_t)(lds_ptr)(lds + st * F::TILE) + (uint32_t)(w * COPIES) * 1024u;
    const i32x4_t rk = sg_raw_rsrc(static_cast<const T*>(a.k) + (int64_t)k0 * a.ldk + kvh * a.hd);
    const i32x4_t rv = sg_raw_rsrc(static_cast<const T*>(a.v) + (int64_t)k0 * a.ldv + kvh * a.hd);
    if (a.hd == D && k0 >= from_row && k0 + F::BK - 1 <= last_row) {
#pragma unroll
      for (int i = 0; i < COPIES; i++) {
        const int r = (w * COPIES + i) * RPC;
        sg_lds_copy16(base + 1024u * i, row_k + (piece_k ^ (uint32_t)(swz_k<D>(r) * 16)), rk, (uint32_t)r * (uint32_t)a.ldk * 2u);
        sg_lds_copy16(base + F::HALF + 1024u * i, row_v + (piece_v ^ (uint32_t)(swz_v<D>(r) * 16)), rv,
                      (uint32_t)r * (uint32_t)a.ldv * 2u);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < COPIES; i++) {
        const int r = (w * COPIES + i) * RPC + lane / C;
        const uint32_t from = (uint32_t)(min(max(k0 + r, from_row), last_row) - k0);
        const int ck = min((lane % C) ^ swz_k<D>(r), a.hd / 8 - 1), cv = min((lane % C) ^ swz_v<D>(r), a.hd / 8 - 1);
        sg_lds_copy16(base + 1024u * i, (from * (uint32_t)a.ldk + ck * 8) * 2u, rk, 0);
        sg_lds_copy16(base + F::HALF + 1024u * i, (from * (uint32_t)a.ldv + cv * 8) * 2u, rv, 0);
      }
    }
  };

  // float32: a tile's rows through registers, TPR threads a row, CL pieces of eight
  // values a thread and round.
  constexpr int TPR = kNT / F::BK > 8 ? kNT / F::BK : 8;
  constexpr int CL = F::F32 ? C / TPR : 1, ROUNDS = F::F32 ? F::BK * TPR / kNT : 1;
  f32x4_t held[F::F32 ? 2 : 1][ROUNDS][CL][2];
  const int jt = tid % TPR;
  auto load = [&](int t) {
    const int k0 = kbeg + t * F::BK;
#pragma unroll
    for (int p = 0; p < ROUNDS; p++) {
      const int64_t from = min(max(k0 + p * (kNT / TPR) + tid / TPR, from_row), last_row);
#pragma unroll
      for (int v = 0; v < 2; v++) {
        const T* src = v ? static_cast<const T*>(a.v) + from * a.ldv : static_cast<const T*>(a.k) + from * a.ldk;
#pragma unroll
        for (int i = 0; i < CL; i++)
#pragma unroll
          for (int u = 0; u < 2; u++)
            held[v][p][i][u] =
                *reinterpret_cast<const f32x4_t*>(src + kvh * a.hd + 8 * min(jt + TPR * i, a.hd / 8 - 1) + 4 * u);
      }
    }
  };
  auto put = [&](int st) {
    float* const key_mul = key_muls + st * 3 * F::BK;
#pragma unroll
    for (int p = 0; p < ROUNDS; p++) {
      const int r = p * (kNT / TPR) + tid / TPR;
#pragma unroll
      for (int v = 0; v < 2; v++) {
        float top = finite_top<8 * CL>(reinterpret_cast<const float*>(&held[v][p][0][0]));
#pragma unroll
        for (int o = TPR / 2; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        int e = row_exp(top);
        if (v) {
          if (e_ref == INT32_MIN) {
            if (jt == 0 && top > 0.0f) atomicMax(&first_e, e);
            __syncthreads();
            e_ref = __builtin_amdgcn_readfirstlane(first_e);
            if (e_ref == INT32_MIN) e_ref = 0;
          }
          if (top > 0.0f && e < e_ref - kSpan) raised = 1;
          e = min(max(e, max(e_ref - kSpan, -kLim)), min(e_ref + kSpan, kLim));
        }
#pragma unroll
        for (int i = 0; i < CL; i++) {
          const int c = jt + TPR * i;
          s16x8_t hi, lo;
          halves(reinterpret_cast<const float*>(&held[v][p][i][0]), pow2(kTop - e), hi, lo);
          unsigned char* dst = lds + st * F::TILE + v * F::PARTS * F::HALF + (r * C + (c ^ (v ? swz_v<D>(r) : swz_k<D>(r)))) * 16;
          *reinterpret_cast<s16x8_t*>(dst) = hi;
          *reinterpret_cast<s16x8_t*>(dst + F::HALF) = lo;
        }
        if (jt == 0) {
          if (v) {
            key_mul[F::BK + r] = (float)(e - e_ref);
            key_mul[2 * F::BK + r] = pow2(e_ref - e);
          } else {
            key_mul[r] = pow2(e - kTop);
          }
        }
      }
    }
  };

  acc_t o[DB] = {};
  float m = fixed ? 0.0f : -INFINITY, l = 0.0f;  // l: this lane's keys only

  // Addresses within a tile: K, lane n's row; V, the transposing load's row and
  // piece.  The xor reaches a piece's low four bits: a variant for each of their
  // values (of 32-query tiles' V: 4 d + 0..3; of 16-query tiles': 2 d + 0..1, whose
  // lowest d bit it leaves alone), immediates for the rest.
  constexpr int KVAR = KS < 16 / G ? KS : 16 / G, VLOW = QT == 32 ? 1 : 2, VVAR = DB / VLOW < 4 ? DB / VLOW : 4;
  uint32_t k_at[KVAR], v_at[VVAR];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)(lds);
#pragma unroll
  for (int i = 0; i < KVAR; i++) k_at[i] = lds0 + (uint32_t)(n * (D * 2) + (((G * i + g) ^ swz_k<D>(n)) << 4));
  {
    // The transposing load takes from lane i of 16 row i / 4's dims 4 (i % 4) .. + 3.
    const int r = 4 * g + ((lane & 15) >> 2), c = (QT == 32 ? 2 * ((lane >> 4) & 1) : 0) + ((lane & 3) >> 1);
#pragma unroll
    for (int i = 0; i < VVAR; i++)
      v_at[i] = lds0 + (uint32_t)(F::PARTS * F::HALF + r * (D * 2) + (((4 * i + c) ^ swz_v<D>(r)) << 4) + (lane & 1) * 8);
  }
  typedef __attribute__((address_space(3))) const s16x8_t* lds_s8;

  // The scores of this wave's KB keys of a tile, from k on, at row kr of LDS stage
  // st, and their part of o.  masked: this lane sees keys [lo, hi), and if `mixed`
  // those of them whose document (of key k + lane % KB: ids) is its own.
  auto block = [&](int st, int k, int kr, bool masked, int lo, int hi, bool mixed, int ids) {
    const uint32_t at = (uint32_t)(st * F::TILE + kr * (D * 2));
    const float* const key_mul = key_muls + st * 3 * F::BK + kr;
    // A step's products go to different accumulators one after another: a matrix
    // instruction that adds to the last one's result waits for it.
    constexpr int NS = F::KB / QT, CH = F::F32 ? 3 : 1;
    acc_t c[NS][CH] = {};
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      // Step ks: piece G ks + g, the low four bits in k_at.
      const lds_s8 p = (lds_s8)(uintptr_t)(k_at[ks % KVAR] + at) + ks / KVAR * 16;
      s16x8_t kf[NS][F::PARTS];
#pragma unroll
      for (int sub = 0; sub < NS; sub++)
#pragma unroll
        for (int part = 0; part < F::PARTS; part++) kf[sub][part] = p[(sub * QT * D * 2 + part * F::HALF) / 16];
#pragma unroll
      for (int sub = 0; sub < NS; sub++) c[sub][0] = X::template step<M>(kf[sub][0], q[0][ks], c[sub][0]);
      if constexpr (F::F32) {
#pragma unroll
        for (int sub = 0; sub < NS; sub++) c[sub][1] = X::template step<M>(kf[sub][0], q[F::PARTS - 1][ks], c[sub][1]);
#pragma unroll
        for (int sub = 0; sub < NS; sub++) c[sub][CH - 1] = X::template step<M>(kf[sub][F::PARTS - 1], q[0][ks], c[sub][CH - 1]);
      }
    }
    float s[SR];
#pragma unroll
    for (int sub = 0; sub < NS; sub++)
#pragma unroll
      for (int r = 0; r < R; r++) s[sub * R + r] = F::F32 ? c[sub][0][r] + (c[sub][CH / 2][r] + c[sub][CH - 1][r]) : c[sub][0][r];
    // Register r: key KSTR (r / 4) + 4 g + r % 4.  The score is s after.
    // float32: the key's power of two times cs first, since either alone may take a score
    // out of range that both bring back.
    if constexpr (F::F32) {
      if (capped) {
#pragma unroll
        for (int b = 0; b < SR / 4; b++) {
          const f32x4_t km = *reinterpret_cast<const f32x4_t*>(key_mul + F::KSTR * b + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; i++) s[4 * b + i] *= km[i] * cs;
        }
      }
    }
    if (early) {
#pragma unroll
      for (int r = 0; r < SR; r++) s[r] *= cs;
    }
    if (capped) {
      float most = 0.0f;
#pragma unroll
      for (int r = 0; r < SR; r++) most = fmaxf(most, fabsf(s[r]));
      if (__ballot(most > near)) {
        // (Through an empty asm: the compiler would compute this side for both.)
#pragma unroll
        for (int r = 0; r < SR; r++) asm volatile("" : "+v"(s[r]));
#pragma unroll
        for (int r = 0; r < SR; r++)
          s[r] = F::F32 ? tanh_f32(s[r]) * cap2
                        : __builtin_fmaf(-2.0f * cap2,
                                         __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[r] * ce * (2.0f * kLog2e)) + 1.0f), cap2);
      } else {
#pragma unroll
        for (int r = 0; r < SR; r++) {
          const float z = s[r] * s[r];
          s[r] = F::F32 ? tanh_near32(s[r]) * cap2 : s[r] * __builtin_fmaf(z, __builtin_fmaf(z, t2, t1), t0);
        }
      }
    }
    if constexpr (F::F32) {
#pragma unroll
      for (int b = 0; b < SR / 4; b++) {
        const f32x4_t km = *reinterpret_cast<const f32x4_t*>(key_mul + F::KSTR * b + 4 * g);
        const f32x4_t ve = *reinterpret_cast<const f32x4_t*>(key_mul + F::BK + F::KSTR * b + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; i++) s[4 * b + i] = capped ? s[4 * b + i] + ve[i] : __builtin_fmaf(s[4 * b + i], km[i] * cs, ve[i]);
      }
    }
    if (a.slopes) {
      const float far = (float)(row - k - 4 * g);
#pragma unroll
      for (int r = 0; r < SR; r++)
        s[r] = __builtin_fmaf(-steep, fabsf(far - (float)(F::KSTR * (r >> 2) + (r & 3))), s[r]);
    }
    if (masked) {
      const int c0 = lo - k - 4 * g, c1 = hi - k - 4 * g;
#pragma unroll
      for (int r = 0; r < SR; r++) {
        const int c = F::KSTR * (r >> 2) + (r & 3);
        s[r] = c >= c0 && c < c1 ? s[r] : -INFINITY;
      }
      if (mixed) {
#pragma unroll
        for (int r = 0; r < SR; r++) s[r] = __shfl(ids, F::KSTR * (r >> 2) + 4 * g + (r & 3)) == me.doc ? s[r] : -INFINITY;
      }
    }
    if (!fixed) {
      float top = s[0];
#pragma unroll
      for (int r = 1; r < SR; r++) top = fmaxf(top, s[r]);
      top = query_max<QT>(top) * (F::F32 ? 1.0f : after);
      if (__ballot(top > m + kSlack)) {  // (-inf + 8 is -inf: a row's first visible key raises it)
        const float to = fmaxf(m, top);
        const float by = to > m ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
        m = to;
        l *= by;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
          for (int r = 0; r < R; r++) o[d][r] *= by;
      }
    }
    const float from = mul<T>::shift - (m == -INFINITY ? 0.0f : m);
    // P^T, KDIM keys a step: the lane's registers 8 st .. + 7.
    s16x8_t p[F::PARTS][F::PS];
#pragma unroll
    for (int ps = 0; ps < F::PS; ps++) {
      float pv[8];
#pragma unroll
      for (int i = 0; i < 8; i++)
        pv[i] = __builtin_amdgcn_exp2f(F::F32 ? s[8 * ps + i] + from : fixed ? s[8 * ps + i] : __builtin_fmaf(s[8 * ps + i], after, from));
      if constexpr (F::F32) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const f32x4_t vw = *reinterpret_cast<const f32x4_t*>(key_mul + 2 * F::BK + F::KSTR * (2 * ps + b) + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; i++) l = __builtin_fmaf(pv[4 * b + i], vw[i], l);
        }
        halves(pv, 1.0f, p[0][ps], p[F::PARTS - 1][ps]);
      } else {
        chunk<M> c;
#pragma unroll
        for (int i = 0; i < 8; i++) c.v[i] = elem<M>::from(pv[i]);
        p[0][ps] = __builtin_bit_cast(s16x8_t, c);
        l = add_up<M>(p[0][ps], l);  // the weights as they are multiplied
      }
    }
    // V^T: lane dim QT d + n, its eight keys those of the lane's p; DG blocks of dims
    // in turn (as above).
    constexpr int DG = F::F32 ? (QT == 16 ? 4 : 2) : (DB < 4 ? DB : 4);
#pragma unroll
    for (int d0 = 0; d0 < DB; d0 += DG) {
#pragma unroll
      for (int ps = 0; ps < F::PS; ps++) {
        s16x8_t vf[DG][F::PARTS];
#pragma unroll
        for (int i = 0; i < DG; i++) {
          const int d = d0 + i;
#pragma unroll
          for (int part = 0; part < F::PARTS; part++) {
            s16x4_t half[2];
#pragma unroll
            for (int u = 0; u < 2; u++)
              half[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (lds_s4)(uintptr_t)(v_at[d / VLOW % VVAR] + at) +
                  (part * F::HALF + F::KSTR * (2 * ps + u) * D * 2 + d % VLOW * 32 + d / VLOW / VVAR * 256) / 8);
            vf[i][part] = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
          }
        }
#pragma unroll
        for (int i = 0; i < DG; i++) o[d0 + i] = X::template step<M>(vf[i][0], p[0][ps], o[d0 + i]);
        if constexpr (F::F32) {
#pragma unroll
          for (int i = 0; i < DG; i++) o[d0 + i] = X::template step<M>(vf[i][0], p[F::PARTS - 1][ps], o[d0 + i]);
#pragma unroll
          for (int i = 0; i < DG; i++) o[d0 + i] = X::template step<M>(vf[i][F::PARTS - 1], p[0][ps], o[d0 + i]);
        }
      }
    }
  };

  // The document of key l % KB of this wave's in lane l, loaded with the tile.
  const int kr = kw * F::KB;
  auto load_ids = [&](int t) { return a.docs ? a.docs[min(kbeg + t * F::BK + kr + lane % F::KB, a.rows - 1)] : 0; };
  auto compute = [&](int st, int t, int ids) {
    const int k = kbeg + t * F::BK + kr;
    int lo = me.lo, hi = me.hi;
    bool mixed = false;
    if (a.docs) {
      const int one = __builtin_amdgcn_readfirstlane(ids);
      mixed = __ballot(ids != one) != 0;
      if (!mixed && me.doc != one) hi = 0;  // one document's keys, and not this row's
    }
    if (!__ballot(lo < k + F::KB && hi > k)) return;
    const bool masked = mixed || __ballot(me.live && (lo > k || hi < k + F::KB)) != 0;
    block(st, k, kr, masked, lo, hi, mixed, ids);
  };

  int t = next(0);
  if constexpr (F::STAGES == 2) {
    // A tile ahead: 16-bit types' copies are in flight while the tile before is
    // computed, float32 rows are loaded before it and halved behind it.
    int st = 0, ids = 0;
    if (t < nt) {
      if constexpr (F::F32) {
        load(t);
        put(0);
      } else {
        copy(0, t);
      }
      ids = load_ids(t);
    }
    while (t < nt) {
      const int tn = next(t + 1);
      int ahead = 0;
      publish();
      if (tn < nt) {
        if constexpr (F::F32) load(tn);
        else copy(st ^ 1, tn);
        ahead = load_ids(tn);
      }
      compute(st, t, ids);
      st ^= 1;
      if (F::F32 && tn < nt) put(st);
      t = tn;
      ids = ahead;
    }
  } else {
    for (; t < nt; t = next(t + 1)) {
      if constexpr (F::F32) load(t);
      __syncthreads();  // the previous tile is done with
      if constexpr (F::F32) put(0);
      else copy(0, t);
      const int ids = load_ids(t);
      publish();
      compute(0, t, ids);
    }
  }
#pragma unroll
  for (int x = QT; x < SG_WAVE; x *= 2) l += __shfl_xor(l, x);

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
    float* mine = reinterpret_cast<float*>(lds) + w * (QT * D) + lane;
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
      for (int r = 0; r < R; r++) mine[(d * R + r) * 64] = o[d][r] * by;
    __syncthreads();
    constexpr int EACH = (DB + KW - 1) / KW;
    db0 = min(DB, kw * EACH);
    db1 = min(DB, db0 + EACH);
#pragma unroll
    for (int d = 0; d < EACH; d++) {
      if (db0 + d >= db1) continue;
#pragma unroll
      for (int r = 0; r < R; r++) {
        const float* from0 = reinterpret_cast<const float*>(lds) + ((db0 + d) * R + r) * 64 + lane;
        float sum = from0[rw * (QT * D)];
#pragma unroll
        for (int i = 1; i < KW; i++) sum += from0[(i * RW + rw) * (QT * D)];
        o[d][r] = sum;
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
    for (int b = 0; b < R / 4; b++) {
      const int at = (db0 + d) * QT + 8 * b + 4 * g;
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
  // Outputs that may have lost bits that their type holds.
  if (F::F32 ? raised != 0 : fixed && __ballot(l < 0x1p-20f)) {
    const float least = F::F32 ? pow2(max(e_ref - kSpan, -126)) : l < 0x1p-20f ? 0x1p-110f * inv : 0.0f;
#pragma unroll
    for (int d = 0; d < KEEP; d++)
#pragma unroll
      for (int r = 0; r < R; r++) bad |= sees && db0 + d < db1 && fabsf(o[d][r] * inv * back) < least;
  }
  uint64_t again = __ballot(bad && me.live);
#pragma unroll
  for (int x = 32; x >= QT; x /= 2) again |= again >> x;
  again &= (1ull << QT) - 1;
  while (again) {
    const int i = __builtin_ctzll(again);
    again &= again - 1;
    careful_row<T, D>(a, row0 + QT * rw + i, h, __builtin_amdgcn_readlane(me.lo, i), __builtin_amdgcn_readlane(me.hi, i),
                      __builtin_amdgcn_readlane(me.doc, i), db0 * QT, min(a.hd, db1 * QT), lane);
  }
}

template <typename T, int D, int QT, int RW, int KW>
hipError_t launch(const sg_attn_masked_args& a, hipStream_t s) {
  typedef form<T, D, QT, RW, KW> F;
  const int64_t tiles = ((int64_t)a.rows + F::BM - 1) / F::BM;
  return sgp::run_kernel(k_attn_masked<T, D, QT, RW, KW>, dim3((unsigned)(tiles * a.heads)), dim3(F::NT), F::LDS, s, a,
                         (int)tiles);
}

// Which form: waves that share 32 rows as long as a workgroup for each 32 rows and head
// fits the GPU at once (one to a CU; two of the 16-bit types' four waves of 64 dims),
// else waves of their own rows.  Whole sequences of 512, 12 heads, microseconds of the
// shared and the own form:
//                    512 rows          1024              2048
//   bf16, 64 dims     8   13           10   13           16   13
//   bf16, 128        11   19           21   17           32   19
//   bf16, 256        18   33           36   33           57   35
//   float32, 64      18   25           33   26           50   35
//   float32, 128     24   36           47   37           71   40
//   float32, 256     49   70           98   70          147   75
// (512 rows are 192 such workgroups.)  float32 rows are 16 to a wave, so that they stay
// in registers (own form, 16384 rows: 150 us against 189 with 32 rows at 128 dims, 230
// against 263 at 256), eight waves to a workgroup that halves a tile once for them all,
// or four at 64 dims, where three workgroups of one tile stage fit a CU (116 us; two
// stages 139; eight waves 130; four of 32 rows 125).  The shared form has eight waves
// to split a tile's halving between, where LDS holds tiles that wide: 32 rows of 128
// dims 11.2 us, 12.9 with four; 256 dims take four.
template <typename T, int D>
hipError_t by_form(const sg_attn_masked_args& a, hipStream_t s) {
  constexpr bool F32 = __is_same(T, float);
  const bool share = ((int64_t)a.rows + 31) / 32 * a.heads <= (D == 64 && !F32 ? 512 : 256);
  if constexpr (F32) {
    return share ? launch<T, D, 16, 2, D == 256 ? 2 : 4>(a, s) : launch<T, D, 16, D == 64 ? 4 : 8, 1>(a, s);
  } else {
    return share ? launch<T, D, 32, 1, 4>(a, s) : launch<T, D, 32, 4, 1>(a, s);
  }
}

template <typename T>
hipError_t by_dim(const sg_attn_masked_args& a, hipStream_t s) {
  return a.hd <= 64 ? by_form<T, 64>(a, s) : a.hd <= 128 ? by_form<T, 128>(a, s) : by_form<T, 256>(a, s);
}

}  // namespace

namespace sgk {

// (64 rows to 256 threads are no more than 128 to 512; rows are shared in small batches only.)
int64_t attention_masked_threads(int dtype, int rows, int heads) {
  return ((int64_t)rows + 127) / 128 * heads * (dtype == SG_F32 ? 512 : 256);
}
hipError_t attention_masked(const sg_attn_masked_args& a, int dtype, hipStream_t s) {
  if (dtype == SG_F32) return by_dim<float>(a, s);
  if (dtype == SG_F16) return by_dim<_Float16>(a, s);
  return by_dim<bf16_t>(a, s);
}

}  // namespace sgk
