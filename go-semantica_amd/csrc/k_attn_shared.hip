// k_attn_shared.hip -- attention over kept keys and values (sg_attention_shared): the plan of a
// call, the join of its pieces, and what is launched.  sg_attn_shared.h has the kernels between.
//
// The plan is one workgroup's work: for every row which places it sees, for every job its tiles,
// and the running total of those, from which workers find their shares.  Offsets, ranges and
// lengths come from device memory, so everything that is addressed later is cut here to the
// tensors and the cache.  It is a chain of loads, searches and barriers: 5 us for one query, 13 for 64
// behind one prefix, 10 for 10476 and 16384 rows (sixteen waves).
//
// The join reads a float32 output for each piece of each (row, head): 27 rows of 32 heads whose
// prefix is split over the GPU 12 us, 16384 rows of which the jobs of 512 workers were cut 21.
#include <algorithm>

#include "semantica_gpu.h"
#include "sg_kernels.h"
#include "sg_kv_cache.h"

namespace {

using sgc::kTile;
using sgp::clamp_row;
using sgp::elem;

constexpr int kPlanSeqs = 2048, kPlanPrefixes = 512;  // numbers of so many are kept in LDS

// The largest i in [0, n) with at(i) <= x for ascending at, 0 if there is none.
template <typename F>
__device__ __forceinline__ int last_at_most(int n, int x, F at) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (at(mid) <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Running totals over a workgroup: put(0, base), put(i + 1, before + count(i)), none above
// `most`.  Returns the last.
template <int THREADS, typename P, typename F>
__device__ int64_t running(int n, int64_t base, int64_t most, P put, F count) {
  __shared__ int64_t wave_sum[THREADS / 64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  if (t == 0) put(0, base);
  for (int i0 = 0; i0 < n; i0 += THREADS) {
    const int i = i0 + t;
    int64_t v = i < n ? count(i) : 0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t u = __shfl_up(v, o);
      if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 63) wave_sum[wave] = v;
    __syncthreads();
    int64_t total = base;
    for (int w = 0; w < THREADS / 64; w++) {
      if (w == wave) v += total;
      total += wave_sum[w];
    }
    if (i < n) put(i + 1, min(v, most));
    base = min(total, most);
  }
  __syncthreads();
  return base;
}

// A range of slots, empty unless it lies in the cache.
__device__ __forceinline__ int kept_length(int start, int length, int64_t slots) {
  return start >= 0 && length > 0 && (int64_t)start + length <= slots ? length : 0;
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void k_attn_plan(sg_attn_shared_args a, sg_attn_batch b, sg_attn_list la,
                                                            sg_attn_list lb, int one_list, int join_rows, int2* seen_out,
                                                            int4* where_out) {
  __shared__ int32_t off_lds[kPlanSeqs + 1], seq_jobs_lds[kPlanSeqs + 1];
  __shared__ int32_t group_lds[kPlanPrefixes + 1], prefix_jobs_lds[kPlanPrefixes + 1];
  __shared__ int2 keys_lds[kPlanSeqs], prefix_lds[kPlanPrefixes];  // start, length (0 outside the cache)
  const int t = threadIdx.x;
  const bool small = b.n_seq <= kPlanSeqs, few = b.n_prefix <= kPlanPrefixes;
  auto range = [&](int start, int length) { return make_int2(start, kept_length(start, length, b.slots)); };
  if (small)
    for (int i = t; i <= b.n_seq; i += THREADS) {
      off_lds[i] = clamp_row(b.off[i], a.rows);
      if (i < b.n_seq) keys_lds[i] = range(b.starts[i], b.lengths[i]);
    }
  if (few && b.n_prefix > 0)
    for (int i = t; i <= b.n_prefix; i += THREADS) {
      group_lds[i] = min(max(b.shared[i], 0), b.n_seq);
      if (i < b.n_prefix) prefix_lds[i] = range(b.prefix_starts[i], b.prefix_lengths[i]);
    }
  __syncthreads();
  // (Loads from LDS and from memory stay two instructions, not one by a pointer that may be either.)
  auto lds = [](int v) {
    asm volatile("" : "+v"(v));
    return v;
  };
  auto off = [&](int i) { return small ? lds(off_lds[i]) : clamp_row(b.off[i], a.rows); };
  auto group_at = [&](int p) { return few ? lds(group_lds[p]) : min(max(b.shared[p], 0), b.n_seq); };
  auto seq_jobs = [&](int i) { return small ? lds(seq_jobs_lds[i]) : b.seq_jobs[i]; };
  auto prefix_jobs = [&](int p) { return few ? lds(prefix_jobs_lds[p]) : b.prefix_jobs[p]; };
  auto own_keys = [&](int i) { return small ? make_int2(lds(keys_lds[i].x), lds(keys_lds[i].y)) : range(b.starts[i], b.lengths[i]); };
  auto prefix_keys = [&](int p) {
    if (p < 0) return make_int2(0, 0);
    return few ? make_int2(lds(prefix_lds[p].x), lds(prefix_lds[p].y)) : range(b.prefix_starts[p], b.prefix_lengths[p]);
  };

  auto prefix_of = [&](int i) {  // of a sequence; -1: none
    if (b.n_prefix == 0) return -1;
    const int p = last_at_most(b.n_prefix, i, group_at);
    return i >= group_at(p) && i < group_at(p + 1) ? p : -1;
  };
  // (m is a power of two; rows * group stay below 2^26.)
  auto tiles_of = [&](int rows, int m) { return (rows * a.group + m - 1) >> (31 - __clz(m)); };
  auto rows_of = [&](int i) { return max(off(i + 1) - off(i), 0); };
  auto rows_behind = [&](int p) { return max(off(group_at(p + 1)) - off(group_at(p)), 0); };

  // Where jobs go.  Again: prefixes with every sequence's own keys, read again for each; or apart,
  // which pays for results of two parts that go through memory (kTraffic a pair) and for a plan and
  // a join of both (kApart): prefixes in the wide list and own keys in the narrow, one after the
  // other (kLaunch), or both in one of the two, if what that list does worse is little.
  // us (32 heads over 8 of 128 dims, 64 tokens with 40 own keys; again, two lists, narrow, wide):
  //   bf16, codes   behind 512  34 47 32 37    2048  50 51 38 39    8192  120 58 57 53
  //   float32       behind 512  55 59 44 77    2048 199 70 83 91    8192  695 117 221 141
  bool all_keys = b.all_keys != 0, together = false, wide = false;
  if (!all_keys) {
    constexpr int64_t kTraffic = 6, kApart = 96000, kLaunch = 160000;  // in sixteenths of a nanosecond
    __shared__ int64_t sums[5][THREADS / 64];
    auto tiles = [&](int keys) { return (int64_t)(a.window > 0 ? min(keys, a.window) : keys) / kTile + 1; };
    int64_t sum[5] = {0, 0, 0, 0, 0};  // prefixes' units by la and lb, own keys' by la and lb, again by lb
    for (int p = t; p < b.n_prefix; p += THREADS) {
      const int rows = rows_behind(p);
      const int64_t n = tiles(prefix_keys(p).y);
      sum[0] += tiles_of(rows, la.m) * (n + la.job_cost);
      sum[1] += tiles_of(rows, lb.m) * (n + lb.job_cost);
    }
    for (int i = t; i < b.n_seq; i += THREADS) {
      const int rows = rows_of(i), p = prefix_of(i);
      const int64_t n = tiles(own_keys(i).y);
      sum[2] += tiles_of(rows, la.m) * (n + la.job_cost);
      sum[3] += tiles_of(rows, lb.m) * (n + lb.job_cost);
      sum[4] += tiles_of(rows, lb.m) * (n + lb.job_cost + (p < 0 ? 0 : tiles(prefix_keys(p).y)));
    }
#pragma unroll
    for (int k = 0; k < 5; k++) {
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) sum[k] += __shfl_xor(sum[k], o);
      if ((t & 63) == 0) sums[k][t >> 6] = sum[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 5; k++) {
      sum[k] = 0;
      for (int w = 0; w < THREADS / 64; w++) sum[k] += sums[k][w];
    }
    // Units of a list one after another over the GPU, a worker's least at the least.
    auto time = [&](const sg_attn_list& l, int64_t units) {
      return max(units * a.kv_heads, (int64_t)l.min_units * l.workers) * l.unit_cost;
    };
    const int64_t apart = (int64_t)a.rows * a.heads * kTraffic + kApart;
    const int64_t again = time(lb, sum[4]), narrow = time(lb, sum[1] + sum[3]) + apart;
    const int64_t other = one_list ? INT64_MAX : time(la, sum[0] + sum[2]) + apart;
    const int64_t two = one_list ? INT64_MAX : time(la, sum[0]) + time(lb, sum[3]) + apart + kLaunch;
    all_keys = again <= min(min(narrow, other), two);
    together = min(narrow, other) <= two;
    wide = other < narrow;
  }
  const bool prefixes = !all_keys;
  auto plan_of = [&](const sg_attn_list& l, int64_t units, int jobs) {  // (workers are a power of two)
    const int64_t per = (units * a.kv_heads + l.workers - 1) >> (31 - __clz(l.workers));
    return sg_attn_plan{units, max(per, (int64_t)l.min_units), jobs, all_keys, 0, 0};
  };
  const bool one = one_list || (prefixes && together);
  // (One list: what stands in it is found by the jobs' kinds, the other is empty.)
  const sg_attn_list pl = prefixes && together && !wide ? lb : la, ol = prefixes && together && wide ? la : lb;

  // Jobs of each prefix and sequence: those of prefixes first where both stand in one list; with
  // all_keys there are only sequences'.
  int end[2] = {0, 0}, own0 = 0;
#pragma unroll 1
  for (int own = prefixes ? 0 : 1; own < 2; own++) {
    if (own) own0 = one ? end[0] : 0;
    const int m = own ? ol.m : pl.m;
    const int last = (int)running<THREADS>(
        own ? b.n_seq : b.n_prefix, own0, own ? ol.cap : pl.cap,
        [&](int i, int64_t v) {
          (own ? b.seq_jobs : b.prefix_jobs)[i] = (int)v;
          if (own ? small : few) (own ? seq_jobs_lds : prefix_jobs_lds)[i] = (int)v;
        },
        [&](int i) { return tiles_of(own ? rows_of(i) : rows_behind(i), m); });
    if (own) end[1] = last;
    else end[0] = last;
  }
  // What each row sees of a prefix that sequences share, and where the join finds it.
  if (join_rows || !all_keys)
    for (int row = t; row < a.rows; row += THREADS) {
      const int i = last_at_most(b.n_seq, row, off);
      const int r0 = off(i), r1 = off(i + 1);
      int4 seen = make_int4(0, 0, 0, 0), where = make_int4(-2, 0, -2, 0);
      if (row >= r0 && row < r1) {
        where = make_int4(-1, 0, seq_jobs(i), r0);
        const int p = prefixes ? prefix_of(i) : -1;
        if (p >= 0) {
          where.x = prefix_jobs(p);
          where.y = off(group_at(p));
          const int plen = prefix_keys(p).y, len = own_keys(i).y;
          seen = sgc::places_seen((int64_t)plen + len - (r1 - r0) + (row - r0), plen, len, a.causal, a.window);
        }
      }
      if (prefixes) seen_out[row] = make_int2(seen.x, seen.y);
      where_out[row] = where;
    }
  __syncthreads();

  // The jobs, and the running total of their costs.
  int64_t base = 0;
#pragma unroll 1
  for (int pass = prefixes ? 0 : 1; pass < 2; pass++) {
    const bool prefix = pass == 0;
    const sg_attn_list list = prefix ? pl : ol;
    const int j0 = prefix ? 0 : own0, n = (prefix ? end[0] : end[1]) - j0;
    const int kind = prefix ? kPrefixKeys : all_keys ? kAllKeys : kOwnKeys;
    base = running<THREADS>(
        n, prefix || one ? base : 0, INT64_MAX, [&](int j, int64_t v) { list.cum[j0 + j] = v; },
        [&](int j) {
          const int i = prefix ? last_at_most(b.n_prefix, j + j0, prefix_jobs) : last_at_most(b.n_seq, j + j0, seq_jobs);
          const int r0 = off(prefix ? group_at(i) : i), r1 = off(prefix ? group_at(i + 1) : i + 1), rows = max(r1 - r0, 0);
          const int2 pk = prefix_keys(prefix ? i : prefix_of(i)), ok = prefix ? make_int2(0, 0) : own_keys(i);
          const int plen = pk.y, len = ok.y;
          const int tile = j + j0 - (prefix ? prefix_jobs(i) : seq_jobs(i));
          const int from = (int)((uint32_t)(tile * list.m) / (uint32_t)a.group);
          const int to = min(rows, (int)((uint32_t)((tile + 1) * list.m - 1) / (uint32_t)a.group) + 1);
          int2 see[2] = {make_int2(0, 0), make_int2(0, 0)};  // of the prefix, of their own
          if (prefix && a.window == 0) {
            see[0] = make_int2(0, plen);  // (some row sees it all, as a rule, and a wave that does not looks at each key)
          } else if (prefix) {
            see[0].x = INT32_MAX;
            for (int r = from; r < to; r++) {
              const int2 s = seen_out[r0 + r];
              see[0].x = min(see[0].x, s.x < s.y ? s.x : INT32_MAX);
              see[0].y = max(see[0].y, s.x < s.y ? s.y : 0);
            }
          } else if (from < to) {
            // Both ends of a range grow with the row, empty or not: the first row's begin, the last one's end.
            const int64_t pos0 = (int64_t)plen + len - rows;
            const int4 s0 = sgc::places_seen(pos0 + from, plen, len, a.causal, a.window);
            const int4 s1 = sgc::places_seen(pos0 + to - 1, plen, len, a.causal, a.window);
            see[0] = make_int2(s0.x, s1.y);
            see[1] = make_int2(s0.z, s1.w);
          }
          // (Cut once more: where offsets do not ascend, a row's range is another group's.)
          int slot_tile[2], tiles[2];
#pragma unroll
          for (int own = 0; own < 2; own++) {
            const int start = own ? ok.x : pk.x, stop = min(see[own].y, own ? len : plen);
            const bool any = see[own].x < stop && !(own ? prefix : kind == kOwnKeys);
            slot_tile[own] = any ? (int)((uint32_t)(start + see[own].x) / kTile) : 0;
            tiles[own] = any ? (int)((uint32_t)(start + stop - 1) / kTile) - slot_tile[own] + 1 : 0;
          }
          // (Own keys alone stand in the first place.)
          const bool alone = kind == kOwnKeys;
          list.jobs[j + j0] = sg_attn_job{r0, rows, tile, kind, {alone ? ok.x : pk.x, ok.x},
                                          {alone ? slot_tile[1] : slot_tile[0], slot_tile[1]},
                                          {alone ? tiles[1] : tiles[0], alone ? 0 : tiles[1]}, plen, len};
          const int64_t count = (int64_t)tiles[0] + tiles[1];
          return count + (count > 0 || kind == kAllKeys ? list.job_cost : 0);
        });
    if (t == 0) *list.plan = plan_of(list, base, j0 + n);
  }
  if (t == 0) {
    if (!one_list && (all_keys || together)) {  // the empty one
      const sg_attn_list none = ol.plan == la.plan ? lb : la;
      *none.plan = plan_of(none, 0, 0);
    }
    la.plan->prefixes = pl.plan != la.plan;  // whose lists are the other's
    lb.plan->own = ol.plan != lb.plan;
  }
}

// The workers that have tiles of a job: [first, last], as of a whole list.
struct holders {
  int64_t first, last;
  bool any;
};
__device__ __forceinline__ holders holders_of(const sg_attn_list& list, int kv, int64_t job) {
  const int64_t c0 = list.cum[job], c1 = list.cum[job + 1], head = kv * list.plan->units, per = list.plan->per;
  holders h{0, 0, c1 - c0 > list.job_cost};
  if (h.any) {
    h.first = sgc::quotient(head + c0 + list.job_cost, per);
    h.last = sgc::quotient(head + c1 - 1, per);
  }
  return h;
}

// A pair's running maximum, sum and output, D / 64 dims a lane, and what it is joined with.
template <int D>
struct joined {
  static constexpr int V = D / 64;
  typedef float vec __attribute__((ext_vector_type(V)));
  float m = -INFINITY, l = 0.0f;
  vec o = 0.0f;
  __device__ __forceinline__ void add(float om, float ol, vec oo) {
    const float top = fmaxf(m, om);  // (maxima are no NaN)
    const float base = top == -INFINITY ? 0.0f : top;
    const float by = __builtin_amdgcn_exp2f(m - base), now = __builtin_amdgcn_exp2f(om - base);
    l = l * by + ol * now;
    if (by != 0.0f && now != 0.0f) {
      o = o * by + oo * now;
    } else {
#pragma unroll
      for (int v = 0; v < V; v++) o[v] = sgc::faded(o[v], by) + sgc::faded(oo[v], now);
    }
    m = top;
  }
  // The pieces at `at` of workers w0, w0 + step, ... up to w1: four loads at a time.
  template <typename F>
  __device__ __forceinline__ void add(const sg_attn_shared_args& a, int64_t w0, int64_t w1, int step, int lane, F at) {
    for (int64_t w = w0; w <= w1; w += 4 * step) {
      float2 ml[4];
      vec x[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int64_t p = at(min(w + i * step, w1));
        ml[i] = a.part_ml[p];
        x[i] = *reinterpret_cast<const vec*>(a.part_o + p * D + lane * V);
      }
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (w + i * step <= w1) add(ml[i].x, ml[i].y, x[i]);
    }
  }
  // A query that sees nothing, or nothing but scores of -infinity, has zeros.
  template <typename T>
  __device__ __forceinline__ void put(const sg_attn_shared_args& a, int row, int head, int lane) const {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = static_cast<T*>(a.out) + row * a.ldo + (int64_t)head * a.hd;
#pragma unroll
    for (int v = 0; v < V; v++)
      if (lane * V + v < a.hd) out[lane * V + v] = elem<T>::from(l == 0.0f ? 0.0f : o[v] * inv);
  }
};

__device__ __forceinline__ int64_t piece_of(const sg_attn_list& list, int64_t worker, bool first, int in_job) {
  return list.piece0 + (worker * 2 + (first ? 1 : 0)) * list.piece_pairs + in_job;
}

// One (row, head) for NW waves: what there is of its prefix's job and of its own keys', or of
// the job that has both.
template <typename T, int D, int NW>
__device__ __forceinline__ void join_one(const sg_attn_shared_args& a, const sg_attn_list& la, const sg_attn_list& lb, int64_t i,
                                         int wave, int lane) {
  const bool all_keys = lb.plan->all_keys != 0;
  const bool prefixes_in_lb = la.plan->prefixes != 0, own_in_la = lb.plan->own != 0;
  const int row = (int)((uint32_t)i / (uint32_t)a.heads), head = (int)(i - (int64_t)row * a.heads);
  const int4 where = a.where[row];
  if (where.z == -2) return;  // a row of no sequence
  const int kv = head / a.group, hg = head - kv * a.group;
  joined<D> x;
#pragma unroll
  for (int own = 0; own < 2; own++) {
    const sg_attn_list list = (own ? !own_in_la : prefixes_in_lb) ? lb : la;
    const int job0 = own ? where.z : where.x;
    if (job0 < 0) continue;
    const int64_t pair = (int64_t)(row - (own ? where.w : where.y)) * a.group + hg, job = job0 + (pair >> (31 - __clz(list.m)));
    if (pair < 0 || job >= list.plan->jobs) continue;  // (offsets that do not ascend)
    const holders h = holders_of(list, kv, job);
    if (all_keys && (!h.any || h.first == h.last)) return;  // written
    if (!h.any) continue;
    const int in_job = (int)pair & (list.m - 1);
    x.add(a, h.first + (NW == 1 ? 0 : wave), h.last, NW, lane, [&](int64_t w) {
      return h.first == h.last ? (int64_t)(own ? a.rows : 0) * a.heads + i : piece_of(list, w, w == h.first, in_job);
    });
  }
  if constexpr (NW > 1) {
    __shared__ float ms[NW], ls[NW];
    __shared__ typename joined<D>::vec os[NW][64];
    os[wave][lane] = x.o;
    if (lane == 0) {
      ms[wave] = x.m;
      ls[wave] = x.l;
    }
    __syncthreads();
    if (wave != 0) return;
    for (int w = 1; w < NW; w++) x.add(ms[w], ls[w], os[w][lane]);
  }
  x.template put<T>(a, row, head, lane);
}
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void k_attn_join(sg_attn_shared_args a, sg_attn_list la, sg_attn_list lb) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if constexpr (NW > 1) {
    join_one<T, D, NW>(a, la, lb, blockIdx.x, wave, lane);
  } else {
    if (lb.plan->all_keys) return;  // k_attn_join_split's
    for (int64_t i = (int64_t)blockIdx.x * 4 + wave; i < (int64_t)a.rows * a.heads; i += (int64_t)gridDim.x * 4)
      join_one<T, D, 1>(a, la, lb, i, wave, lane);
  }
}

// The jobs with all keys that lie across workers, for many rows: a block column for each
// worker that ends inside a job and began it.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_attn_join_split(sg_attn_shared_args a, sg_attn_list list) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t units = list.plan->units, per = list.plan->per, worker = blockIdx.x, end = (worker + 1) * per;
  if (!list.plan->all_keys) return;
  if (end >= units * a.kv_heads) return;
  const int kv = (int)sgc::quotient(end, units);
  const int64_t at = end - kv * units;
  const int job = sgc::last_at_most(list.cum, list.plan->jobs, at, lane);
  const holders h = holders_of(list, kv, job);
  if (!h.any || h.first != worker || h.last == worker) return;
  const sg_attn_job jb = list.jobs[job];
  // Four pairs a wave, a piece of each at a time.
  const int in_job = blockIdx.y * 16 + wave * 4;
  const int64_t pair0 = (int64_t)jb.tile * list.m + in_job, pairs = (int64_t)jb.rows * a.group;
  if (pair0 >= pairs) return;
  joined<D> x[4];
  for (int64_t w = h.first; w <= h.last; w++) {
    float2 ml[4];
    typename joined<D>::vec o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int64_t at = piece_of(list, w, w == h.first, in_job + (int)min((int64_t)i, pairs - 1 - pair0));
      ml[i] = a.part_ml[at];
      o[i] = *reinterpret_cast<const typename joined<D>::vec*>(a.part_o + at * D + lane * joined<D>::V);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) x[i].add(ml[i].x, ml[i].y, o[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int64_t pair = pair0 + i;
    if (pair >= pairs) return;
    const int r = (int)(pair / a.group);
    x[i].template put<T>(a, jb.row0 + r, kv * a.group + (int)(pair - (int64_t)r * a.group), lane);
  }
}

// Time of a unit with all workers busy, in sixteenths of a nanosecond.  Measured at 128 dims (at 256 twice
// that): bf16 2 ns narrow, 3 wide, over codes 1 and 3; float32 6 and 14, over codes 1.6 and 4.
int unit_cost(int dtype, bool q8, int D, bool wide) {
  if (dtype != SG_F32) return wide ? 3 * D / 8 : q8 ? D / 8 : D / 4;
  return q8 ? (wide ? D / 2 : D / 5) : wide ? 7 * D / 4 : 3 * D / 4;
}

// The form of each kind of job.  Up to so many pairs of a group on average, waves work for
// themselves.
// (Prefix of 16384 behind one key head, us, narrow and wide: float32 of 256 dims 16 pairs 53 and 54, 32 57
// and 55, 64 69 and 58; bf16 over codes 128 pairs 37 and 41, where the plan takes either, but with 8 key
// heads and 131072 places 136 pairs 301 and 128.)
constexpr int kNarrowPairs = 32;
// So many full jobs a sequence, and it takes a prefix again rather than in two parts (64 sequences of
// 512 bf16 tokens of 4 heads behind 2048: 247 us, in two parts 405).
constexpr int kFullJobs = 4;
// (row, head) up to here: 16 waves each, four; beyond: one, in turn.  64: 29 us with 16, 32 with four, 38
// with one; 512: 53, 49, 51; 2048: 81, 59, 56; 8192: 180, 103, 91.
constexpr int64_t kJoinFew = 256, kJoinSome = 2048;
constexpr int64_t kJoinBlocks = 8192;

struct layout {
  size_t plan, cum[2], jobs[2], seq_jobs, prefix_jobs, seen, where, ml, o, total;
  int64_t pieces[2];
  int cap, workers[2], m[2], piece_pairs[2];
};

// Lists: 0 narrow, 1 wide.  All sizes grow with each of the arguments.
layout lay_out(int dtype, bool q8, int rows, int heads, int kv_heads, int D, int n_seq, int n_prefix) {
  layout y{};
  const int64_t pairs = (int64_t)rows * (heads / kv_heads);
  y.cap = (int)std::min<int64_t>(2 * (pairs / 16) + n_seq + n_prefix + 2, INT32_MAX);
  const int cus = 256;
  y.workers[0] = cus * 4 * (dtype == SG_F32 ? 1 : 2);
  y.workers[1] = cus * (D == 256 || (dtype == SG_F32 && D == 128) ? 1 : 2);
  y.m[0] = 16;
  y.m[1] = sgk::attn_wide_pairs(D, dtype == SG_F32, q8);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  y.plan = take(2 * sizeof(sg_attn_plan));
  for (int i = 0; i < 2; i++) {
    y.cum[i] = take(sizeof(int64_t) * ((size_t)y.cap + 1));
    y.jobs[i] = take(sizeof(sg_attn_job) * (size_t)y.cap);
  }
  y.seq_jobs = take(sizeof(int32_t) * ((size_t)n_seq + 1));
  y.prefix_jobs = take(sizeof(int32_t) * ((size_t)n_prefix + 1));
  y.seen = take(sizeof(int2) * (size_t)rows);
  y.where = take(sizeof(int4) * (size_t)rows);
  // Rows whose jobs may lie in two lists, each with a place of its own for a (row, head): none where
  // nothing is shared or sequences fill several jobs themselves (all_keys), so no more than those that
  // such sequences may have.
  const int64_t apart = n_prefix == 0 ? 0 : std::min<int64_t>(rows, (int64_t)kFullJobs * y.m[1] * n_seq / (heads / kv_heads));
  int64_t rows_of_o = 2 * apart * heads;
  for (int i = 0; i < 2; i++) {
    y.pieces[i] = rows_of_o;
    y.piece_pairs[i] = (int)std::min<int64_t>(y.m[i], pairs);
    rows_of_o += (int64_t)y.workers[i] * 2 * y.piece_pairs[i];
  }
  y.ml = take(sizeof(float2) * (size_t)rows_of_o);
  y.o = take(sizeof(float) * (size_t)rows_of_o * D);
  y.total = at;
  return y;
}

template <typename T, int D>
hipError_t join(const sg_attn_shared_args& a, const sg_attn_list& la, const sg_attn_list& lb, int all_keys, hipStream_t s) {
  const int64_t n = (int64_t)a.rows * a.heads;
  if (n <= kJoinFew) return sgp::run_kernel(k_attn_join<T, D, 16>, dim3(n), dim3(64 * 16), 0, s, a, la, lb);
  if (n <= kJoinSome) return sgp::run_kernel(k_attn_join<T, D, 4>, dim3(n), dim3(64 * 4), 0, s, a, la, lb);
  hipError_t e = sgp::run_kernel(k_attn_join_split<T, D>, dim3(lb.workers, lb.m / 16), dim3(256), 0, s, a, lb);
  if (e != hipSuccess || all_keys) return e;
  return sgp::run_kernel(k_attn_join<T, D, 1>, dim3(std::min<int64_t>((n + 3) / 4, kJoinBlocks)), dim3(256), 0, s, a, la, lb);
}
template <typename T>
hipError_t join_dims(const sg_attn_shared_args& a, const sg_attn_list& la, const sg_attn_list& lb, int all_keys, int D,
                     hipStream_t s) {
  if (D == 64) return join<T, 64>(a, la, lb, all_keys, s);
  if (D == 128) return join<T, 128>(a, la, lb, all_keys, s);
  return join<T, 256>(a, la, lb, all_keys, s);
}

}  // namespace

namespace sgk {

size_t attn_shared_work_bytes(int dtype, bool q8, int rows, int heads, int kv_heads, int D, int n_seq, int n_prefix) {
  return lay_out(dtype, q8, rows, heads, kv_heads, D, n_seq, n_prefix).total;
}

hipError_t attn_shared(sg_attn_shared_args a, sg_attn_batch b, int dtype, bool q8, int D, void* work, hipStream_t s) {
  const layout y = lay_out(dtype, q8, a.rows, a.heads, a.kv_heads, D, b.n_seq, b.n_prefix);
  char* w = static_cast<char*>(work);
  int2* seen = reinterpret_cast<int2*>(w + y.seen);
  int4* where = reinterpret_cast<int4*>(w + y.where);
  a.seen = seen;
  a.where = where;
  a.part_o = reinterpret_cast<float*>(w + y.o);
  a.part_ml = reinterpret_cast<float2*>(w + y.ml);
  b.seq_jobs = reinterpret_cast<int32_t*>(w + y.seq_jobs);
  b.prefix_jobs = reinterpret_cast<int32_t*>(w + y.prefix_jobs);
  sg_attn_list lists[2];
  for (int i = 0; i < 2; i++) {
    sg_attn_list& l = lists[i];
    l.plan = reinterpret_cast<sg_attn_plan*>(w + y.plan) + i;
    l.cum = reinterpret_cast<int64_t*>(w + y.cum[i]);
    l.jobs = reinterpret_cast<sg_attn_job*>(w + y.jobs[i]);
    l.piece0 = y.pieces[i];
    l.piece_pairs = y.piece_pairs[i];
    l.m = y.m[i];
    l.workers = y.workers[i];
    l.blocks = i ? l.workers : l.workers / 4;
    l.wide = i;
    l.cap = y.cap;
    l.unit_cost = unit_cost(dtype, q8, D, i);
    // A worker's least, so that the join has fewer pieces (one query behind 1536 places of float32, 256 dims:
    // 23 us with 1, 28 with 2, 40 with 4; a wide list with 16: 64 tokens of codes 72 for 64); and what a
    // job costs beside its tiles (40 passages of float32 with 0: 214 for 206).
    l.min_units = i ? (dtype == SG_F32 && !q8 ? 3 : 8) : dtype == SG_F32 && D == 256 ? 1 : 2;
    l.job_cost = i ? 4 : dtype == SG_F32 && D == 256 ? 1 : 2;
  }
  const int64_t pairs = (int64_t)a.rows * a.group;
  // A job for each M pairs of a sequence, over prefix and own keys in one go, where no prefix is
  // shared or sequences fill several jobs themselves; otherwise the plan weighs it by the lengths.
  // (lay_out counts on it.)
  b.all_keys = b.n_seq <= b.n_prefix || b.n_prefix == 0 || pairs >= (int64_t)kFullJobs * y.m[1] * b.n_seq;
  const int wide_own = pairs > (int64_t)kNarrowPairs * b.n_seq;
  const int64_t narrow_pairs = dtype != SG_F32 && !q8 ? kNarrowPairs / 2 : kNarrowPairs;
  const int wide_prefix = b.all_keys ? wide_own : pairs > narrow_pairs * b.n_prefix;
  const sg_attn_list& lb = lists[wide_own];
  const sg_attn_list& la = lists[wide_prefix];
  const int one_list = &la == &lb;
  const int join_rows = (int64_t)a.rows * a.heads <= kJoinSome;  // one by one
  // Few rows and sequences: four waves, which meet sooner than sixteen (64 tokens: 49 and 54 us a call; 300
  // and more alike).
  const int threads = a.rows > 512 || b.n_seq > 512 || b.n_prefix > 512 ? 1024 : 256;
  hipError_t e =
      sgp::run_kernel(threads == 1024 ? k_attn_plan<1024> : k_attn_plan<256>, dim3(1), dim3(threads), 0, s, a, b, la, lb, one_list,
                      join_rows, seen, where);
  auto run = [&](const sg_attn_list& l) {
    if (e != hipSuccess) return;
    e = dtype == SG_F32   ? attn_shared_f32(a, l, q8, D, s)
        : dtype == SG_F16 ? attn_shared_f16(a, l, q8, D, s)
                          : attn_shared_bf16(a, l, q8, D, s);
  };
  run(la);
  if (!one_list) run(lb);
  if (e != hipSuccess) return e;
  if (dtype == SG_F32) return join_dims<float>(a, la, lb, b.all_keys, D, s);
  if (dtype == SG_F16) return join_dims<_Float16>(a, la, lb, b.all_keys, D, s);
  return join_dims<sgp::bf16_t>(a, la, lb, b.all_keys, D, s);
}

}  // namespace sgk
