// A label drawn from each column of scores.
//
// For a column l of m scores, M = max l and a temperature T, the weights are
// w_i = exp((l_i - M) / T).  Of the labels in the order of falling scores
// (ties by rising index) the first k are kept (top-k), of these the shortest
// beginning whose weights sum to p times theirs (top-p), and of these the
// ones with w_i >= q, that is q times the largest (min-p).  The label is the
// first, by rising index, at which the sum of the kept weights passes u
// times their total.
//
// Every cut keeps a beginning of that order, so it is a pair (tau, r): the
// labels above tau and the first r of those at tau.  Sums of weights are
// taken in integers, w 2^shift rounded to the nearest with the shift as
// large as m of them allow (2^45 at m = 131072): integer sums do not hang on
// their order, so a drawn label depends neither on how a column is split
// over threads nor on the order of atomics, and they keep small weights that
// sums of 32-bit floats would lose.  What a unit cannot hold they lose too:
// m / 2 units at most in all, 2^-29 of the largest weight at m = 131072 and
// 2^-17 at kSampleMostLabels, where the entry point ends.
//
// A cut is found from a short list.  The lanes that share a column each hold
// the largest of their part of it; an order statistic of those maxima is a
// bound with a known number of scores at or above it, and not many more.
// The scores above the bound are gathered with their indices and sorted;
// the cuts are then prefixes of the sorted list.  Where the list does not
// hold (very many equal scores, a nucleus of thousands) the cut comes from
// a search over the whole column.  The draw itself goes by rising index: a
// prefix sum over the kept labels.
#include "answer_launch.hpp"
#include "answer_limits.hpp"
#include "answer_types.hpp"
#include "answer_wave.hpp"
#include "common.hpp"

namespace sdca_gpu {
namespace {

constexpr int kBins = 2048;
constexpr u64 kOne52 = 0x4330000000000000ull;  // 2^52 as a double

// A NaN counts as a label that cannot be drawn (the larger of a NaN and a
// number is the number).
__device__ inline float score(float x) { return fmaxf(x, -INFINITY); }

struct Weights {
  float max, inv_t;
  double scale;
  // (The smaller of NaN and 0 is 0: an infinite maximum has weight 1.)
  __device__ float of(float l) const { return expf(fminf((l - max) * inv_t, 0.f)); }
  // w 2^shift to the nearest integer, plus the pattern of 2^52: the sum
  // w 2^shift + 2^52 has its integer part in the lowest bits.  Sums of
  // these carry a known multiple of the pattern.
  __device__ u64 raw(float w) const {
    return static_cast<u64>(__double_as_longlong(__builtin_fma(static_cast<double>(w), scale, 4503599627370496.0)));
  }
  __device__ u64 fixed(float w) const { return raw(w) - kOne52; }
};

// ---------------------------------------------------------------------------
// Settings and results of a column.
// ---------------------------------------------------------------------------
struct SampleArgs {
  int m;
  int64_t n, lds;
  const float* u;
  PerColumn<float> temperature, top_p, min_p;
  PerColumn<int64_t> top_k;
  int64_t* labels;
  float* prob;
  int64_t* kept;
  double scale;
};

template <class T>
__device__ inline T setting(const PerColumn<T>& c, int64_t col) {
  return c.each ? c.each[col] : c.value;
}

struct Settings {
  float t, p, q;
  int k;  // 0: off
  bool greedy, cut;
  __device__ Settings(const SampleArgs& a, int64_t col) {
    t = fminf(setting(a.temperature, col), 3.402823466e38f);
    greedy = !(setting(a.temperature, col) >= 1.17549435e-38f);
    p = setting(a.top_p, col);
    p = p < 1.f ? fmaxf(p, 0.f) : 1.f;
    q = setting(a.min_p, col);
    q = q > 0.f ? fminf(q, 1.f) : 0.f;
    const int64_t kk = setting(a.top_k, col);
    k = kk > 0 && kk < a.m ? static_cast<int>(kk) : 0;
    cut = k || p < 1.f;
  }
};

__device__ inline void answer(const SampleArgs& a, int64_t col, int64_t label, float prob,
                              int64_t kept) {
  a.labels[col] = label;
  if (a.prob) a.prob[col] = prob;
  if (a.kept) a.kept[col] = kept;
}

// The shortest beginning with at least p of the mass, and at least one
// label: the least integer sum that it reaches.
__device__ inline u64 top_p_target(float p, u64 mass) {
  const u64 t = static_cast<u64>(ceil(static_cast<double>(p) * static_cast<double>(mass)));
  return t < 1 ? 1 : t > mass ? mass : t;
}
// The label is the first whose sum exceeds this.
__device__ inline u64 draw_target(float u, u64 total) {
  u = u > 0.f ? (u < 1.f ? u : 0.99999994f) : 0.f;
  const u64 t = static_cast<u64>(static_cast<double>(u) * static_cast<double>(total));
  return t < total ? t : total - 1;
}
__device__ inline float share(float w, double scale, u64 total) {
  return static_cast<float>(static_cast<double>(w) * scale / static_cast<double>(total));
}
// Scores below this have weight 0: exp(-105) is below half the smallest
// float.  (Rounded down, so that no score of nonzero weight is below.)
__device__ inline float live_floor(float max, float t) {
  const float f = max - 106.f * t;
  return f == f ? f : -INFINITY;  // an infinite maximum
}

// ---------------------------------------------------------------------------
// A column in a wave's registers: lane t holds the values 256 g + 4 t + e.
// ---------------------------------------------------------------------------

// The cut (tau, ties) by a search over the keys' bits, for a column whose
// short list does not do: each step counts or sums what is at least a
// trial key.
template <int E>
__device__ inline void wave_search(const float (&l)[E], const Weights& wt, const Settings& c,
                                         unsigned* tau_out, int* ties_out) {
  unsigned tau = 0;
  int ties = 0;
  if (c.k) {
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned trial = tau | (1u << bit);
      int count = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) count += __popcll(__ballot(key_of(l[e]) >= trial));
      if (count >= c.k) tau = trial;
    }
    int above = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) above += __popcll(__ballot(key_of(l[e]) > tau));
    ties = c.k - above;
  }
  if (c.p < 1.f) {
    const u64 f_tau = ties ? wt.fixed(wt.of(score_of(tau))) : 0;
    u64 mass = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) mass += key_of(l[e]) > tau ? wt.fixed(wt.of(l[e])) : 0;
    mass = wave_sum(mass) + ties * f_tau;
    const u64 target = top_p_target(c.p, mass);
    unsigned cut = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned trial = cut | (1u << bit);
      u64 sum = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) sum += key_of(l[e]) >= trial ? wt.fixed(wt.of(l[e])) : 0;
      if (wave_sum(sum) >= target) cut = trial;
    }
    u64 above = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) above += key_of(l[e]) > cut ? wt.fixed(wt.of(l[e])) : 0;
    above = wave_sum(above);
    const u64 f = wt.fixed(wt.of(score_of(cut)));
    const u64 need = f ? (target - above + f - 1) / f : 1;
    ties = cut == tau && ties && need > static_cast<u64>(ties) ? ties : static_cast<int>(need);
    tau = cut;
  }
  *tau_out = tau;
  *ties_out = ties;
}

// The draw from a column in registers: the labels above tau and the first
// `ties` at it, those with a weight of at least q.
template <int E>
__device__ inline void wave_draw(const float (&l)[E], const Weights& wt, const Settings& c,
                                 const SampleArgs& a, int64_t col, unsigned tau, int ties) {
  const int lane = threadIdx.x & 63;
  const float w_tau = ties ? wt.of(score_of(tau)) : 0.f;
  u64 mass = 0;
  int count = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float w = wt.of(l[e]);
    const bool in = (tau == 0 || key_of(l[e]) > tau) && w >= c.q && w > 0.f;
    mass += in ? wt.fixed(w) : 0;
    count += in;
  }
  const bool tied = ties && w_tau >= c.q && w_tau > 0.f;
  int left = 0;  // of the ties
  if (tied) {
    int at = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) at += __popcll(__ballot(key_of(l[e]) == tau));
    left = at < ties ? at : ties;
  }
  const u64 total = wave_sum(mass) + left * (tied ? wt.fixed(w_tau) : 0);
  const int many = wave_sum(count) + left;
  const u64 target = draw_target(a.u[col], total);
  u64 base = 0;
  bool done = false;
#pragma unroll
  for (int g = 0; g < E / 4; ++g) {
    if (done) continue;
    int own = 0;
    if (tied) {
#pragma unroll
      for (int e = 0; e < 4; ++e) own += key_of(l[4 * g + e]) == tau;
    }
    const int before = tied ? wave_scan(own) - own : 0;
    int rank = before;
    u64 f[4];
    float w[4];
    u64 sum = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = l[4 * g + e];
      w[e] = wt.of(v);
      bool in = (tau == 0 || key_of(v) > tau);
      if (tied && key_of(v) == tau) in = rank++ < left;
      f[e] = in && w[e] >= c.q ? wt.fixed(w[e]) : 0;
      sum += f[e];
    }
    const u64 incl = wave_scan(sum) + base;
    const u64 passed = __ballot(incl > target);
    if (passed) {
      if (lane == __ffsll(passed) - 1) {
        u64 s = incl - sum;
        int pick = 3;
        float wp = w[3];
#pragma unroll
        for (int e = 2; e >= 0; --e) {
          u64 upto = s;
#pragma unroll
          for (int b = 0; b <= e; ++b) upto += f[b];
          if (upto > target) {
            pick = e;
            wp = w[e];
          }
        }
        answer(a, col, 256 * g + 4 * lane + pick, share(wp, wt.scale, total), many);
      }
      done = true;
    }
    base = read_lane64(incl, 63);
    if (tied) {
      const int used = __builtin_amdgcn_readlane(before + own, 63);
      left = left > used ? left - used : 0;
    }
  }
}

constexpr int kWaveList = 256;

template <int E>
__device__ inline int count_at_least(const float (&l)[E], float b) {
  int n = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) n += __popcll(__ballot(l[e] >= b));
  return n;
}


// The cuts and the draw from a list of `count` (at most 64 R) entries by
// rising index.  mass: of all labels, or 0 for that of the list after its
// top-k; the list holds the nucleus.
template <int R>
__device__ inline void wave_list_draw(const u64* list, int count, u64 mass, const Weights& wt,
                                      const Settings& c, const SampleArgs& a, int64_t col) {
  const int lane = threadIdx.x & 63;
  u64 mine[R], entry[R], incl[R];
  bool keep[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    mine[r] = 64 * r + lane < count ? list[64 * r + lane] : 0;
    entry[r] = mine[r];
  }
  sort_wave<false>(entry);
  const int first = c.k && c.k < count ? c.k : count;
  u64 all = 0;
  float w[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool in = 64 * r + lane < first;
    w[r] = in ? wt.of(score_of(static_cast<unsigned>(entry[r] >> 32))) : 0.f;
    incl[r] = wave_scan(in ? wt.fixed(w[r]) : 0) + all;
    all = read_lane64(incl[r], 63);
    keep[r] = w[r] >= c.q && w[r] > 0.f;
  }
  if (c.p < 1.f) {
    const u64 target = top_p_target(c.p, mass ? mass : all);
#pragma unroll
    for (int r = 0; r < R; ++r) keep[r] = keep[r] && incl[r] - wt.fixed(w[r]) < target;
  }
  // The kept labels are a prefix; the last of them bounds them in the list by
  // index.
  int many = 0;
  u64 last = 0, total = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const u64 kept = __ballot(keep[r]);
    const int n = many == 64 * r ? (~kept ? __ffsll(~kept) - 1 : 64) : 0;
    if (n) {
      last = read_lane64(entry[r], n - 1);
      total = read_lane64(incl[r], n - 1);
      many += n;
    }
  }
  const u64 target = draw_target(a.u[col], total);
  u64 base = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float wm = wt.of(score_of(static_cast<unsigned>(mine[r] >> 32)));
    const u64 sum = wave_scan(mine[r] >= last ? wt.fixed(wm) : 0) + base;
    const u64 passed = __ballot(sum > target);
    if (passed) {
      if (lane == __ffsll(passed) - 1)
        answer(a, col, index_of(mine[r]), share(wm, wt.scale, total), many);
      return;
    }
    base = read_lane64(sum, 63);
  }
}

template <class T, int E>
__global__ __launch_bounds__(256, E <= 16 ? 5 : 3) void sample_wave_kernel(
    const T* __restrict__ S, SampleArgs a) {
  __shared__ u64 lists[4][kWaveList];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  if (col >= a.n) return;
  const T* row = S + col * a.lds;

  float l[E];
  float most = -INFINITY;
#pragma unroll
  for (int g = 0; g < E / 4; ++g) {
    float v[4];
    load_vec<4>(row, 256 * g + 4 * lane, a.m, v, -INFINITY);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      l[4 * g + e] = score(v[e]);
      most = fmaxf(most, l[4 * g + e]);
    }
  }
  const Settings c(a, col);
  Weights wt;
  wt.max = wave_max<false>(most);
  if (wt.max == -INFINITY) {
    if (lane == 0) answer(a, col, -1, 0.f, 0);
    return;
  }
  if (c.greedy) {
#pragma unroll
    for (int g = 0; g < E / 4; ++g) {
      const bool here = l[4 * g] == wt.max || l[4 * g + 1] == wt.max || l[4 * g + 2] == wt.max ||
                        l[4 * g + 3] == wt.max;
      const u64 any = __ballot(here);
      if (any) {
        if (lane == __ffsll(any) - 1) {
          const int e = l[4 * g] == wt.max ? 0 : l[4 * g + 1] == wt.max ? 1 : l[4 * g + 2] == wt.max ? 2 : 3;
          answer(a, col, 256 * g + 4 * lane + e, 1.f, 1);
        }
        return;
      }
    }
  }
  wt.inv_t = 1.f / c.t;
  wt.scale = a.scale;
  if (!c.cut) {
    wave_draw<E>(l, wt, c, a, col, 0, 0);
    return;
  }

  // A bound with few enough scores at or above it for a list, and enough of
  // them for the cut: `count` of them.
  // (Scores of weight 0 need not be in it; nor are those at -infinity.)
  const float floor_live = fmaxf(live_floor(wt.max, c.t), -3.402823466e38f);
  const float sorted = sort_wave<false>(most, true);
  float from = floor_live;
  int count = 0;
  u64 mass = 0;  // of all labels, where the list is not the whole of them
  if (c.k) {
    // The k-th largest lane maximum has k scores or more.  Where that is no
    // bound, or one with too many, halving the keys' interval finds one.
    if (c.k <= 64) from = fmaxf(read_lane(sorted, c.k - 1), floor_live);
    count = count_at_least(l, from);
    if (count > kWaveList && c.k <= kWaveList) {
      unsigned low = key_of(from), high = key_of(wt.max) + 1;
      while (count > kWaveList && high - low > 1) {
        const unsigned mid = low + (high - low) / 2;
        const int n = count_at_least(l, score_of(mid));
        if (n < c.k) {
          high = mid;
        } else {
          low = mid;
          count = n;
        }
      }
      from = score_of(low);
    }
  } else {
    // A nucleus: bounds that leave some 44, 97 and 200 of 1000 scores, the
    // first whose scores hold the mass.
    float w[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      w[e] = wt.of(l[e]);
      mass += wt.raw(w[e]);
    }
    mass = wave_sum(mass - E * kOne52);
    const u64 target = top_p_target(c.p, mass);
    for (int t = 0; t < 3; ++t) {
      const float bound = read_lane(sorted, t == 0 ? 31 : t == 1 ? 49 : 61);
      from = fmaxf(bound, floor_live);
      u64 sum = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) sum += wt.raw(l[e] >= from ? w[e] : 0.f);
      count = kWaveList + 1;
      if (wave_sum(sum - E * kOne52) >= target) {
        count = count_at_least(l, from);
        break;
      }
    }
  }
  if (count <= kWaveList) {
    u64* list = lists[wave];
    int placed = 0;
#pragma unroll
    for (int g = 0; g < E / 4; ++g) {
      bool in[4];
      u64 mask[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        in[e] = l[4 * g + e] >= from;
        mask[e] = __ballot(in[e]);
      }
      if ((mask[0] | mask[1] | mask[2] | mask[3]) == 0) continue;
      int at = placed;  // by rising index: the lanes before, then the lane's own before
#pragma unroll
      for (int e = 0; e < 4; ++e)
        at = __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(mask[e] >> 32),
                                       __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(mask[e]), at));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (in[e]) list[at] = entry_of(l[4 * g + e], 256 * g + 4 * lane + e);
        at += in[e];
        placed += __popcll(mask[e]);
      }
    }
    wave_lds_sync();
    if (count <= 64) wave_list_draw<1>(list, count, mass, wt, c, a, col);
    else if (count <= 128) wave_list_draw<2>(list, count, mass, wt, c, a, col);
    else wave_list_draw<4>(list, count, mass, wt, c, a, col);
    return;
  }
  unsigned tau;
  int ties;
  wave_search<E>(l, wt, c, &tau, &ties);
  wave_draw<E>(l, wt, c, a, col, tau, ties);
}

// ---------------------------------------------------------------------------
// A column to a workgroup, and to several.
// ---------------------------------------------------------------------------
constexpr int kList = 1024;  // entries of a short list

template <int THREADS>
struct Shared {
  static constexpr int kWaves = THREADS / 64;
  static constexpr int kEntries = THREADS < kList ? THREADS : kList;
  union {
    u64 hist[kBins];
    unsigned guide[kBins];
    struct {
      u64 entry[kEntries];
      u64 swap[THREADS];
    } list;
  };
  u64 sum[kWaves], sum2[kWaves], sum3[kWaves];
  float value[kWaves], value2[kWaves], value3[kWaves];
  int number[kWaves];
  u64 found_above;
  int found_bin, count;
};

template <int W>
__device__ inline u64 total_of(const u64 (&part)[W]) {
  u64 s = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) s += part[w];
  return s;
}

// A bound with `want` scores or more at or above it: of `units` waves that
// each know their j-th largest lane maximum, r = three quarters reach the
// r-th largest of these, which makes j r scores.  For a nucleus, whose size
// is not known, j stops at half the lanes.
struct Order {
  int j, r;
  __device__ Order(int units, int k, int nucleus) {
    r = (3 * units + 3) / 4;
    j = ((k ? k : nucleus) + r - 1) / r;
    if (!k) j = min(j, 32);
  }
  __device__ bool fits() const { return j <= 40; }
};
// The r-th largest of the units' values (at most 64 units), in every wave.
__device__ inline float unit_bound(const float* value, int units, int r) {
  const int lane = threadIdx.x & 63;
  return read_lane(sort_wave<true>(lane < units ? value[lane] : -INFINITY, true), r - 1);
}
// How many labels the list of a nucleus is made for: first a short one, and
// a longer one where that holds too little.
constexpr int kNucleus = 128, kNucleusLong = 320;

// f(score, index) over the entries [begin, end) of a row in memory, by
// `threads` lanes.
template <class T, class F>
__device__ inline void each_of(const T* row, int begin, int end, int t, int threads, F f) {
  constexpr int V = 8;
  for (int64_t at = begin + int64_t(t) * V; at < end; at += int64_t(threads) * V) {
    float v[V];
    load_vec<V>(row, at, end, v);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (at + e < end) f(score(v[e]), static_cast<int>(at) + e);
  }
}

// The bin at which the running sum over falling bins, `sum` before the
// highest, first reaches `target`, and the sum above it: in s.found_bin and
// s.found_above (the lowest bin where none does).
template <int THREADS>
__device__ void find_bin(int bins, u64 sum, u64 target, Shared<THREADS>& s) {
  constexpr int kOwn = kBins / THREADS;  // bins of a thread
  __syncthreads();
  const int hi = bins - 1 - kOwn * static_cast<int>(threadIdx.x);
  u64 own = 0;
  for (int b = 0; b < kOwn; ++b) own += hi - b >= 0 ? s.hist[hi - b] : 0;
  u64 before = wave_scan(own);
  if ((threadIdx.x & 63) == 63) s.sum[threadIdx.x >> 6] = before;
  if (threadIdx.x == 0) {
    s.found_bin = 0;
    s.found_above = sum;
  }
  __syncthreads();
  for (int w = 0; w < static_cast<int>(threadIdx.x >> 6); ++w) before += s.sum[w];
  before += sum - own;
  if (before < target && before + own >= target) {
    for (int b = 0; b < kOwn; ++b) {
      const u64 here = s.hist[hi - b];
      if (before + here >= target) {
        s.found_bin = hi - b;
        s.found_above = before;
        break;
      }
      before += here;
    }
  }
  __syncthreads();
}

// The key at which the running sum over falling keys, from `floor_key` up,
// first reaches `target` (counts, or with MASS fixed weights), and the sum
// above it: three digits of the key, a histogram each.
template <bool MASS, int THREADS, class T>
__device__ void descend(const T* row, int m, const Weights& wt, unsigned floor_key, u64 target,
                        Shared<THREADS>& s, unsigned* tau, u64* above) {
  unsigned prefix = 0;
  u64 sum = 0;
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
    const int bits = level == 2 ? 10 : 11;
    const int bins = 1 << bits;
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += THREADS) s.hist[i] = 0;
    __syncthreads();
    each_of(row, 0, m, threadIdx.x, THREADS, [&](float l, int) {
      const unsigned key = key_of(l);
      if (key < floor_key || (level && (key >> (shift + bits)) != prefix)) return;
      const u64 add = MASS ? wt.fixed(wt.of(l)) : 1;
      if (add) atomicAdd(&s.hist[(key >> shift) & (bins - 1)], add);
    });
    find_bin(bins, sum, target, s);
    prefix = (prefix << bits) | static_cast<unsigned>(s.found_bin);
    sum = s.found_above;
  }
  *tau = prefix;
  *above = sum;
}

// The draw within [begin, end) of a row: the labels above tau and the first
// `ties` of the whole row at it, those with a weight of at least q.  The
// stretch is narrowed to the one that holds the label, a wave's share at a
// time.  total: of the whole row, with `base` and `tie_base` ties before
// `begin`, and `many` kept; or 0 where [begin, end) is the whole row, which
// gives them then.
template <int THREADS, class T>
__device__ void narrow_and_draw(const T* row, int begin, int end, u64 base, u64 tie_base,
                                u64 total, u64 many, unsigned tau, u64 ties, const Weights& wt,
                                const Settings& c,
                                const SampleArgs& a, int64_t col, Shared<THREADS>& s) {
  constexpr int kWaves = THREADS / 64;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const float w_tau = ties ? wt.of(score_of(tau)) : 0.f;
  const u64 f_tau = w_tau >= c.q ? wt.fixed(w_tau) : 0;
  u64 target = total ? draw_target(a.u[col], total) : 0;
  // The sums below are those that the caller's total is made of (the same
  // weights under the same cuts, as integers), so one stretch passes the
  // target at each step.  Each step leaves a sixteenth, or a quarter with four
  // waves, or 64 scores: the stretch is down to 64 after eight steps, and the
  // loop ends whatever the sums are.
  for (int step = 0; step < 8; ++step) {
    const int part = ((end - begin + kWaves - 1) / kWaves + 63) / 64 * 64;
    const int b = begin + wave * part, e = b + part < end ? b + part : end;
    u64 n_tie = 0, mass = 0, count = 0;
    if (b < e)
      each_of(row, b, e, lane, 64, [&](float l, int) {
        const unsigned key = key_of(l);
        const float w = wt.of(l);
        if (key > tau && w >= c.q && w > 0.f) {
          mass += wt.fixed(w);
          ++count;
        }
        n_tie += ties && key == tau;
      });
    n_tie = wave_sum(n_tie);
    mass = wave_sum(mass);
    count = wave_sum(count);
    __syncthreads();
    if (lane == 0) {
      s.sum[wave] = n_tie;
      s.sum2[wave] = mass;
      s.sum3[wave] = count;
    }
    __syncthreads();
    if (total == 0) {
      u64 tied = total_of(s.sum);
      tied = tied < ties ? tied : ties;
      total = total_of(s.sum2) + tied * f_tau;
      many = total_of(s.sum3) + (w_tau >= c.q && w_tau > 0.f ? tied : 0);
      target = draw_target(a.u[col], total);
    }
    int pick = begin;
    for (int w = 0; w < kWaves; ++w) {
      const u64 left = ties > tie_base ? ties - tie_base : 0;
      const u64 t = s.sum[w] < left ? s.sum[w] : left;
      const u64 here = s.sum2[w] + t * f_tau;
      if (base + here > target) break;
      base += here;
      tie_base += s.sum[w];
      pick += part;
    }
    begin = pick;
    end = pick + part < end ? pick + part : end;
    if (part <= 64) break;
  }
  if (wave == 0) {
    const bool in = begin + lane < end;
    const float l = in ? score(to_float(row[begin + lane])) : -INFINITY;
    const unsigned key = key_of(l);
    const float w = wt.of(l);
    const bool tied = in && ties && key == tau;
    const u64 rank = wave_scan(tied ? u64(1) : u64(0)) + tie_base;
    const bool keep = in && w >= c.q && (key > tau || (tied && rank <= ties));
    const u64 sum = wave_scan(keep ? wt.fixed(w) : 0) + base;
    const u64 passed = __ballot(sum > target);
    if (passed && lane == __ffsll(passed) - 1)
      answer(a, col, begin + lane, share(w, wt.scale, total), static_cast<int64_t>(many));
  }
}

// Sorts the first P (a power of two from 64 to THREADS) of the workgroup's
// values, one a thread, falling.
template <int THREADS>
__device__ inline u64 sort_block(u64 v, int P, u64* swap) {
  const int i = threadIdx.x;
  if (i < P) v = sort_wave<true>(v, (i & 64) == 0 || P == 64);
  for (int size = 128; size <= P; size <<= 1) {
    const bool falling = (i & size) == 0 || size == P;
    for (int stride = size >> 1; stride >= 64; stride >>= 1) {
      __syncthreads();
      if (i < P) swap[i] = v;
      __syncthreads();
      if (i < P) {
        const u64 o = swap[i ^ stride];
        const bool larger = ((i & stride) == 0) == falling;
        v = (o > v) == larger ? o : v;
      }
    }
    if (i < P) v = sort_merge<32, true>(v, falling);
  }
  return v;
}

// The inclusive sum over the workgroup's threads.
template <int THREADS>
__device__ inline u64 block_scan(u64 v, u64 (&part)[THREADS / 64], u64* total) {
  v = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 all = 0, before = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w == static_cast<int>(threadIdx.x >> 6)) before = all;
    all += part[w];
  }
  *total = all;
  return v + before;
}

// The nucleus of a column with very many labels in it takes two passes over
// the column.  The first adds the mass up in 2048 even steps of the score,
// which finds the step that the target falls into.  The second gathers the
// few labels of that step, whose sorted list gives the cut, and adds up the
// labels above it by stretches of the column, which gives the draw its
// stretch.
//
// The first pass only guides: it takes hardware exponentials and sums of 32
// bits, and the second one's exact sums check its step.
struct NucleusSteps {
  float low, per, rate, unit, max;
  u64 target;
  __device__ NucleusSteps(u64 mass, const Weights& wt, const Settings& c, int m) {
    target = top_p_target(c.p, mass);
    // Labels of weights below e = (1 - p) mass / m sum to less than what the
    // nucleus leaves out, so it has none of them.
    const float rest = (1.f - c.p) *
                       static_cast<float>(static_cast<double>(mass) / wt.scale) /
                       static_cast<float>(m);
    low = wt.max + (logf(rest) - 0.01f) / wt.inv_t - fabsf(wt.max) * 1e-5f;
    per = static_cast<float>(kBins) / (wt.max - low);
    // Sums of at most 2^30, and a rounding up for each label besides.
    unit = 1073741824.f * static_cast<float>(wt.scale / static_cast<double>(mass));
    rate = wt.inv_t * 1.44269504f;
    max = wt.max;
    share = static_cast<u64>(static_cast<double>(target) / static_cast<double>(mass) * 1073741824.0);
  }
  u64 share;  // the target as the guide has it
  __device__ bool fit() const { return per > 0.f && per < INFINITY && low > -INFINITY; }
  __device__ int of(float l) const {  // rises with l
    return min(static_cast<int>((l - low) * per), kBins - 1);
  }
  __device__ unsigned weight(float l) const {
    return static_cast<unsigned>(__builtin_amdgcn_exp2f((l - max) * rate) * unit + 0.5f);
  }
};

// What the second pass finds in a lane's scores.
struct NucleusSums {
  u64 over = 0, sum = 0, many = 0;  // above the step; sum and many: those that min-p leaves
  template <class F>
  __device__ void add(const NucleusSteps& steps, int step, float l, const Weights& wt,
                      const Settings& c, F in_step) {
    if (!(l >= steps.low)) return;
    const int at = steps.of(l);
    if (at > step) {
      const float w = wt.of(l);
      const u64 f = wt.fixed(w);
      over += f;
      if (w >= c.q) {
        sum += f;
        ++many;
      }
    } else if (at == step) {
      in_step();
    }
  }
};

// The first of `parts` (at most 64; lane i has the mass of part i) at which
// the sum passes the target, else the last, and the sum of those before it.
__device__ inline int part_of(u64 mass, int parts, u64 target, u64* before) {
  const u64 incl = wave_scan(mass);
  const u64 passed = __ballot(incl > target);
  const int part = passed ? min(__ffsll(passed), parts) - 1 : parts - 1;
  *before = read_lane64(incl - mass, part);
  return part;
}

// The cut and the draw behind the second pass.  entry: thread i's of the
// `count` in the step; above: the mass above it; s.sum2 and s.sum3: the mass
// and number of the labels above it that min-p leaves, for each of kWaves
// stretches of `part` scores.  False, and nothing done, where the step was
// not the right one.
template <int THREADS, class T>
__device__ bool finish_nucleus(const T* row, u64 entry, int count, u64 above, u64 target, int part,
                               const Weights& wt, const Settings& c, const SampleArgs& a,
                               int64_t col, Shared<THREADS>& s) {
  constexpr int kWaves = THREADS / 64;
  const int i = threadIdx.x, wave = i >> 6, lane = i & 63;
  if (above >= target) return false;
  int P = 64;
  while (P < count) P <<= 1;
  entry = sort_block<THREADS>(entry, P, s.list.swap);
  const float w = i < count ? wt.of(score_of(static_cast<unsigned>(entry >> 32))) : 0.f;
  const u64 f = i < count ? wt.fixed(w) : 0;
  u64 all;
  const u64 incl = block_scan<THREADS>(f, s.sum, &all);
  if (above + all < target) return false;
  const bool in = i < count && above + incl - f < target;  // a prefix, not empty
  const u64 votes = __ballot(in);
  __syncthreads();
  if (lane == 0) s.number[wave] = __popcll(votes);
  s.list.swap[i] = entry;
  __syncthreads();
  int kept = 0;
  for (int v = 0; v < kWaves; ++v) kept += s.number[v];
  const unsigned tau = static_cast<unsigned>(s.list.swap[kept - 1] >> 32);
  if (in && w >= c.q) {
    atomicAdd(&s.sum2[index_of(entry) / part], f);
    atomicAdd(&s.sum3[index_of(entry) / part], u64(1));
  }
  __syncthreads();
  const u64 total = total_of(s.sum2), draw = draw_target(a.u[col], total), many = total_of(s.sum3);
  u64 base;
  const int pick = part_of(lane < kWaves ? s.sum2[lane] : 0, kWaves, draw, &base);
  // The ties that are kept, in all and before the stretch.
  const bool tie = in && static_cast<unsigned>(entry >> 32) == tau;
  const u64 tied = __ballot(tie), early = __ballot(tie && index_of(entry) < pick * part);
  __syncthreads();
  if (lane == 0) {
    s.sum[wave] = __popcll(tied);
    s.number[wave] = __popcll(early);
  }
  __syncthreads();
  const u64 ties = total_of(s.sum);
  u64 tie_base = 0;
  for (int v = 0; v < kWaves; ++v) tie_base += s.number[v];
  narrow_and_draw<THREADS>(row, pick * part, min(a.m, pick * part + part), base, tie_base, total,
                           many, tau, ties, wt, c, a, col, s);
  return true;
}

// The nucleus by one workgroup, of the labels with keys from floor_key up.
// False, and nothing done, where the step is not the right one or holds more
// labels than the list.
template <int THREADS, class T>
__device__ bool nucleus_and_draw(const T* row, u64 mass, unsigned floor_key, const Weights& wt,
                                 const Settings& c, const SampleArgs& a, int64_t col,
                                 Shared<THREADS>& s) {
  constexpr int kWaves = THREADS / 64, kEntries = Shared<THREADS>::kEntries;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const NucleusSteps steps(mass, wt, c, a.m);
  if (!steps.fit()) return false;
  for (int i = threadIdx.x; i < kBins; i += THREADS) s.guide[i] = 0;
  __syncthreads();
  each_of(row, 0, a.m, threadIdx.x, THREADS, [&](float l, int) {
    if (l >= steps.low && key_of(l) >= floor_key) atomicAdd(&s.guide[steps.of(l)], steps.weight(l));
  });
  __syncthreads();
  u64 own[kBins / THREADS];
#pragma unroll
  for (int b = 0; b < kBins / THREADS; ++b) own[b] = s.guide[threadIdx.x + b * THREADS];
  __syncthreads();
#pragma unroll
  for (int b = 0; b < kBins / THREADS; ++b) s.hist[threadIdx.x + b * THREADS] = own[b];
  find_bin(kBins, 0, steps.share, s);
  const int step = s.found_bin;
  __syncthreads();
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();

  const int part = ((a.m + kWaves - 1) / kWaves + 63) / 64 * 64;
  const int begin = wave * part, end = min(a.m, begin + part);
  NucleusSums sums;
  if (begin < end)
    each_of(row, begin, end, lane, 64, [&](float l, int i) {
      sums.add(steps, step, l, wt, c, [&] {
        if (key_of(l) < floor_key) return;
        const int at = atomicAdd(&s.count, 1);
        if (at < kEntries) s.list.entry[at] = entry_of(l, i);
      });
    });
  const u64 over = wave_sum(sums.over), sum = wave_sum(sums.sum), many = wave_sum(sums.many);
  if (lane == 0) {
    s.sum[wave] = over;
    s.sum2[wave] = sum;
    s.sum3[wave] = many;
  }
  __syncthreads();
  const int count = s.count;
  const u64 above = total_of(s.sum);
  __syncthreads();
  if (count > kEntries) return false;
  const u64 entry = static_cast<int>(threadIdx.x) < count ? s.list.entry[threadIdx.x] : 0;
  return finish_nucleus<THREADS>(row, entry, count, above, steps.target, part, wt, c, a, col, s);
}

// The cut by searches over the whole column, and the draw: for columns whose
// short list does not do.  mass: of all labels, where it is known; steps:
// whether a nucleus is first searched in even steps.
template <int THREADS, class T>
__device__ void search_and_draw(const T* row, u64 mass, const Weights& wt, const Settings& c,
                                const SampleArgs& a, int64_t col, Shared<THREADS>& s,
                                bool steps = true) {
  unsigned tau = 0;
  u64 ties = 0;  // labels at tau that are kept
  if (c.k) {
    u64 above;
    descend<false>(row, a.m, wt, 0, static_cast<u64>(c.k), s, &tau, &above);
    ties = c.k - above;
  }
  if (c.p < 1.f) {
    if (c.k || mass == 0) {
      mass = 0;
      each_of(row, 0, a.m, threadIdx.x, THREADS, [&](float l, int) {
        if (key_of(l) > tau) mass += wt.fixed(wt.of(l));
      });
      mass = wave_sum(mass);
      __syncthreads();
      if ((threadIdx.x & 63) == 0) s.sum[threadIdx.x >> 6] = mass;
      __syncthreads();
      mass = total_of(s.sum);
      if (ties) mass += ties * wt.fixed(wt.of(score_of(tau)));
      __syncthreads();
    }
    if (steps && nucleus_and_draw<THREADS>(row, mass, tau, wt, c, a, col, s)) return;
    const u64 target = top_p_target(c.p, mass);
    unsigned cut;
    u64 above;
    descend<true>(row, a.m, wt, tau, target, s, &cut, &above);
    const u64 w = wt.fixed(wt.of(score_of(cut)));
    u64 need = w ? (target - above + w - 1) / w : 1;
    if (cut == tau && ties && need > ties) need = ties;
    tau = cut;
    ties = need;
  }
  narrow_and_draw<THREADS>(row, 0, a.m, 0, 0, 0, 0, tau, ties, wt, c, a, col, s);
}

// A stretch [begin, end) of a column, for the workgroup's waves: each has
// the same number of groups of 64 V neighbouring scores, lane t the values
// V t .. V t + V - 1 of each group.  R: a lane's scores that are kept in
// registers; R = 0 reads them from memory each time, 16 scores at once.
template <class T, int THREADS, int R>
struct Column {
  static constexpr int V = sizeof(T) == 2 ? 8 : 4;
  static constexpr int kGroups = R / V;
  static constexpr bool kHalf = sizeof(T) == 2;
  const T* row;
  int groups, from, end;  // from: this lane's first score; end: of the wave's
  int length;
  unsigned raw[kGroups ? kGroups * (kHalf ? V / 2 : V) : 1];

  __device__ Column(const T* r, int begin, int end_, int groups_)
      : row(r), groups(groups_), length(end_ - begin) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first = begin + wave * groups * 64 * V;
    from = first + (threadIdx.x & 63) * V;
    end = min(end_, first + groups * 64 * V);
    if constexpr (R > 0) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        if (g >= groups) break;
        T v[V];
        const int at = from + g * 64 * V;
        if (at + V <= end) {
          __builtin_memcpy(v, row + at, sizeof(v));
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] = at + e < end ? row[at + e] : T(-INFINITY);
        }
        if constexpr (kHalf) {
          __builtin_memcpy(&raw[g * V / 2], v, sizeof(v));
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) raw[g * V + e] = __float_as_uint(to_float(v[e]));
        }
      }
    }
  }
  // Waves whose lanes all hold a score.
  __device__ int full_waves() const {
    return min(THREADS / 64, max(length - 64 * V, 0) / (groups * 64 * V) + 1);
  }
  __device__ void group(int g, float (&l)[V]) const {
    if constexpr (R > 0) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if constexpr (kHalf) {
          const unsigned short b = static_cast<unsigned short>(raw[(g * V + e) / 2] >> (16 * (e & 1)));
          T t;
          __builtin_memcpy(&t, &b, 2);
          l[e] = score(to_float(t));
        } else {
          l[e] = score(__uint_as_float(raw[g * V + e]));
        }
      }
    } else {
      load_vec<V>(row, int64_t(from) + int64_t(g) * 64 * V, end, l, -INFINITY);
#pragma unroll
      for (int e = 0; e < V; ++e) l[e] = score(l[e]);
    }
  }
  // f(scores, index of the first) for each of the lane's groups, until it
  // gives false (in all lanes of a wave alike).
  template <class F>
  __device__ void groups_until(F f) {
    if constexpr (R > 0) {
      // Each pass makes its own floats of the registers, and one group's work
      // ends before the next one's begins: floats kept from one pass to the
      // next, or indices, or many groups' exponentials in flight, spill.
#pragma unroll
      for (unsigned& r : raw) asm volatile("" : "+v"(r));
      asm volatile("" : "+v"(from));
      bool go = true;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        if (g < groups && go) {
          float l[V];
          group(g, l);
          go = f(l, from + g * 64 * V);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      constexpr int kBatch = 16 / V;
      for (int g = 0; g < groups; g += kBatch) {
        float l[kBatch][V];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) group(g + b, l[b]);
        bool go = true;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          if (go) go = f(l[b], from + (g + b) * 64 * V);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (!go) break;
      }
    }
  }
  template <class F>
  __device__ void each(F f) {
    groups_until([&](const float (&l)[V], int at) {
#pragma unroll
      for (int e = 0; e < V; ++e) f(l[e], at + e);
      return true;
    });
  }
};

// The fixed weights of a group of scores.
template <int V>
__device__ inline u64 mass_of(const Weights& wt, const float (&l)[V]) {
  u64 sum = 0;
#pragma unroll
  for (int e = 0; e < V; ++e) sum += wt.raw(wt.of(l[e]));
  return sum - V * kOne52;
}

// The fixed weights of those of a group that min-p leaves, and their number.
template <int V>
__device__ inline void add_kept(const Weights& wt, float q, const float (&l)[V], u64* mass,
                                int* count) {
  u64 sum = 0;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float w = wt.of(l[e]);
    w = w >= q ? w : 0.f;
    sum += wt.raw(w);
    *count += w > 0.f;
  }
  *mass += sum - V * kOne52;
}

// Appends the scores of a group that are at least `from` to a list in LDS
// (it counts those beyond its room too).  Most groups have none.
template <int V>
__device__ inline void push_from(float from, const float (&l)[V], int at, u64* list, int room,
                                 int* count) {
  float most = l[0];
#pragma unroll
  for (int e = 1; e < V; ++e) most = fmaxf(most, l[e]);
  if (!(most >= from && most > -INFINITY)) return;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if (l[e] >= from && l[e] > -INFINITY) {
      const int i = atomicAdd(count, 1);
      if (i < room) list[i] = entry_of(l[e], at + e);
    }
  }
}

// The cuts and the draw from a list of `count` (at most THREADS) entries,
// thread i's in `entry`.  mass: of all labels, or 0 for that of the list
// (after its top-k).  False, and nothing done, where the list holds less
// than the nucleus.
template <int THREADS>
__device__ bool list_and_draw(u64 entry, int count, u64 mass, const Weights& wt,
                              const Settings& c, const SampleArgs& a, int64_t col,
                              Shared<THREADS>& s) {
  constexpr int kWaves = THREADS / 64;
  const int i = threadIdx.x, lane = i & 63, wave = i >> 6;
  const auto weight = [&] {
    return i < count ? wt.of(score_of(static_cast<unsigned>(entry >> 32))) : 0.f;
  };
  if (mass && !c.k) {  // before the sort, which a nucleus of thousands need not wait for
    u64 held;
    block_scan<THREADS>(i < count ? wt.fixed(weight()) : 0, s.sum, &held);
    if (held < top_p_target(c.p, mass)) return false;
  }
  int P = 64;
  while (P < count) P <<= 1;
  entry = sort_block<THREADS>(entry, P, s.list.swap);
  const float w = weight();
  const u64 f = i < count ? wt.fixed(w) : 0;
  const int first = c.k && c.k < count ? c.k : count;
  u64 all;
  const u64 incl = block_scan<THREADS>(i < first ? f : 0, s.sum, &all);
  bool keep = i < first && w >= c.q && w > 0.f;
  if (c.p < 1.f) {
    const u64 target = top_p_target(c.p, mass ? mass : all);
    if (all < target) return false;
    keep = keep && incl - f < target;
  }
  // The kept labels are a prefix of the list; they are sorted again by index
  // (its complement falls), each with its place in the list behind it.
  const u64 votes = __ballot(keep);
  const int own = ~votes ? __ffsll(~votes) - 1 : 64;
  if (lane == 0) s.number[wave] = own;
  s.list.swap[i] = entry;
  __syncthreads();
  int many = 0;
  for (int v = 0; v < kWaves; ++v) {
    many += s.number[v];
    if (s.number[v] < 64) break;
  }
  int P2 = 64;
  while (P2 < many) P2 <<= 1;
  u64 by = i < many ? (static_cast<u64>(static_cast<unsigned>(entry)) << 32) | static_cast<unsigned>(i) : 0;
  by = sort_block<THREADS>(by, P2, s.list.entry);
  const float wk =
      i < many ? wt.of(score_of(static_cast<unsigned>(s.list.swap[static_cast<unsigned>(by)] >> 32))) : 0.f;
  const u64 fk = i < many ? wt.fixed(wk) : 0;
  u64 total;
  const u64 sum = block_scan<THREADS>(fk, s.sum2, &total);
  const u64 target = draw_target(a.u[col], total);
  if (sum > target && sum - fk <= target)
    answer(a, col, index_of(by >> 32), share(wk, wt.scale, total), many);
  return true;
}

// (Four waves to a SIMD: they hide the loads and the exponentials' latencies.)
template <class T, int THREADS, int R>
__global__ __launch_bounds__(THREADS, 4) void sample_block_kernel(const T* __restrict__ S,
                                                               SampleArgs a) {
  constexpr int kWaves = THREADS / 64;
  constexpr int kEntries = Shared<THREADS>::kEntries;
  __shared__ Shared<THREADS> s;
  const int64_t col = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const T* row = S + col * a.lds;
  typedef Column<T, THREADS, R> Col;
  Col column(row, 0, a.m, (a.m + THREADS * Col::V - 1) / (THREADS * Col::V));
  const Settings c(a, col);

  float most = -INFINITY;
  column.each([&](float l, int) { most = fmaxf(most, l); });
  const int full = column.full_waves();
  const Order brief(full, c.k, kNucleus), longer(full, 0, kNucleusLong);
  const bool list_does = c.cut && brief.fits();
  const bool again = !c.k && THREADS >= kList && longer.j > brief.j;
  const float top = wave_max<true>(most);
  if (lane == 0) s.value[wave] = top;
  if (list_does) {
    const float sorted = sort_wave<true>(most, true);
    const float x = read_lane(sorted, brief.j - 1), y = read_lane(sorted, again ? longer.j - 1 : 0);
    if (lane == 0) {
      s.value2[wave] = x;
      s.value3[wave] = y;
    }
  }
  __syncthreads();
  Weights wt;
  wt.max = s.value[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) wt.max = fmaxf(wt.max, s.value[w]);
  if (wt.max == -INFINITY) {
    if (threadIdx.x == 0) answer(a, col, -1, 0.f, 0);
    return;
  }
  if (c.greedy) {
    int best = a.m;
    column.each([&](float l, int i) { best = l == wt.max && i < best ? i : best; });
#pragma unroll
    for (int d = 32; d; d >>= 1) best = min(best, __shfl_xor(best, d));
    if (lane == 0) s.number[wave] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 0; w < kWaves; ++w) best = min(best, s.number[w]);
      answer(a, col, best, 1.f, 1);
    }
    return;
  }
  wt.inv_t = 1.f / c.t;
  wt.scale = a.scale;

  if (!c.cut) {
    // Each wave's sum and count; then the wave whose stretch holds the label
    // goes through it group by group.
    u64 mass = 0;
    int count = 0;
    column.groups_until([&](const float (&l)[Col::V], int) {
      add_kept(wt, c.q, l, &mass, &count);
      return true;
    });
    mass = wave_sum(mass);
    count = wave_sum(count);
    if (lane == 0) {
      s.sum[wave] = mass;
      s.number[wave] = count;
    }
    __syncthreads();
    const u64 total = total_of(s.sum);
    const u64 target = draw_target(a.u[col], total);
    u64 base = 0;
    for (int w = 0; w < wave; ++w) base += s.sum[w];
    if (base > target || base + s.sum[wave] <= target) return;
    int many = 0;
    for (int w = 0; w < kWaves; ++w) many += s.number[w];
    column.groups_until([&](const float (&l)[Col::V], int at) {
      u64 f[Col::V], sum = 0;
#pragma unroll
      for (int e = 0; e < Col::V; ++e) {
        const float w = wt.of(l[e]);
        f[e] = w >= c.q ? wt.fixed(w) : 0;
        sum += f[e];
      }
      const u64 incl = wave_scan(sum) + base;
      const u64 passed = __ballot(incl > target);
      base = read_lane64(incl, 63);
      if (!passed) return true;
      if (lane == __ffsll(passed) - 1) {
        u64 upto = incl - sum;
        int pick = -1;
        float w = 0.f;
#pragma unroll
        for (int e = 0; e < Col::V; ++e) {
          upto += f[e];
          if (pick < 0 && upto > target) {
            pick = at + e;
            w = wt.of(l[e]);
          }
        }
        answer(a, col, pick, share(w, wt.scale, total), many);
      }
      return false;
    });
    return;
  }

  const float floor_live = live_floor(wt.max, c.t);
  u64 mass = 0;
  for (int attempt = 0; list_does && attempt < (again ? 2 : 1); ++attempt) {
    __syncthreads();
    if (threadIdx.x == 0) s.count = 0;
    const float bound = attempt ? unit_bound(s.value3, full, longer.r)
                                : unit_bound(s.value2, full, brief.r);
    // Whether the list holds every label of nonzero weight.
    const bool whole = bound <= floor_live;
    const bool sum_all = c.p < 1.f && !c.k && !whole;
    const float from = whole ? floor_live : bound;
    __syncthreads();
    const bool sum_now = sum_all && mass == 0;
    column.groups_until([&](const float (&l)[Col::V], int at) {
      if (sum_now) mass += mass_of(wt, l);
      push_from(from, l, at, s.list.entry, kEntries, &s.count);
      return true;
    });
    if (sum_now) {
      mass = wave_sum(mass);
      if (lane == 0) s.sum3[wave] = mass;
    }
    __syncthreads();
    if (sum_all) mass = total_of(s.sum3);
    const int count = s.count;
    if (count > kEntries) break;
    const u64 entry = static_cast<int>(threadIdx.x) < count ? s.list.entry[threadIdx.x] : 0;
    if (list_and_draw<THREADS>(entry, count, sum_all ? mass : 0, wt, c, a, col, s)) return;
  }
  __syncthreads();
  search_and_draw<THREADS>(row, mass, wt, c, a, col, s);
}

// ---------------------------------------------------------------------------
// A column to several workgroups: with few columns one workgroup each leaves
// most of the device idle.  Three kernels: the parts' maxima and order
// statistics; then, with the column's maximum known, their sums and entries
// of the list; then the draw.  Where a nucleus can be larger than the list,
// three more take the columns that the draw has left: the two passes, and
// the draw behind them.  (For the others they end at once, at 2 us each; one
// workgroup takes 50 us for the two passes over 10^5 scores.)
// ---------------------------------------------------------------------------
constexpr int kPartThreads = 256, kPartWaves = kPartThreads / 64;
constexpr int kMaxParts = 64 / kPartWaves;  // unit_bound takes 64 waves
constexpr int kPartStep = 2048;             // parts are multiples of it: whole groups of any type

struct PartsOf {  // one column's
  u64 mass[kMaxParts];
  float top[kMaxParts], jth[kMaxParts * kPartWaves];
  int count[kMaxParts], first[kMaxParts];
  int listed, gathered;
  // Of a nucleus that the list does not hold: whether it is one, the guide
  // to its step, and its sums by parts.
  int large, unused;
  NucleusSums sums[kMaxParts];
  unsigned guide[kBins];
  u64 entry[kList];
  // (A part to a lane: one after the other the loads of 16 parts took 2 us.)
  __device__ u64 total(int parts) const {
    const int lane = threadIdx.x & 63;
    return wave_sum(lane < parts ? mass[lane] : 0);
  }
};
static_assert(kMaxParts == kList / 64, "finish_nucleus takes the parts as the waves' stretches");

struct PartArgs {
  PartsOf* of;
  int parts, part;  // how many, and the scores of each but the last
  bool large;       // whether the kernels for large nuclei follow
};

template <class T>
__device__ inline Column<T, kPartThreads, 0> part_column(const T* row, int m, const PartArgs& p) {
  typedef Column<T, kPartThreads, 0> Col;
  const int begin = blockIdx.x * p.part;
  return Col(row, begin, min(m, begin + p.part), p.part / (kPartThreads * Col::V));
}
// Waves of all parts whose lanes all hold a score.
template <int V>
__device__ inline int full_units(int m, const PartArgs& p) {
  return min(p.parts * kPartWaves, max(m - 64 * V, 0) / (p.part / kPartWaves) + 1);
}

template <class T>
__global__ __launch_bounds__(kPartThreads) void sample_parts_kernel(const T* __restrict__ S,
                                                                    SampleArgs a, PartArgs p) {
  __shared__ float tops[kPartWaves];
  const int64_t col = blockIdx.y;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  PartsOf& of = p.of[col];
  auto column = part_column(S + col * a.lds, a.m, p);
  const Settings c(a, col);
  float most = -INFINITY;
  column.each([&](float l, int) { most = fmaxf(most, l); });
  const float top = wave_max<true>(most);
  if (lane == 0) tops[wave] = top;
  const Order order(full_units<decltype(column)::V>(a.m, p), c.k, kNucleusLong);
  if (c.cut && order.fits()) {
    const float x = read_lane(sort_wave<true>(most, true), order.j - 1);
    if (lane == 0) of.jth[blockIdx.x * kPartWaves + wave] = x;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = tops[0];
    for (int w = 1; w < kPartWaves; ++w) t = fmaxf(t, tops[w]);
    of.top[blockIdx.x] = t;
    if (blockIdx.x == 0) of.listed = of.gathered = of.large = 0;
  }
}

// What the second and third kernel know of a column.
struct PartsKnown {
  float max, bound, floor_live;
  bool list_does, whole, sum_all;
  PartsKnown() = default;
  __device__ PartsKnown(const PartsOf& of, const PartArgs& p, const Settings& c, int units) {
    const int lane = threadIdx.x & 63;
    max = wave_max<true>(lane < p.parts ? of.top[lane] : -INFINITY);
    const Order order(units, c.k, kNucleusLong);
    list_does = c.cut && !c.greedy && order.fits();
    floor_live = live_floor(max, c.t);
    bound = list_does ? unit_bound(of.jth, units, order.r) : 0.f;
    whole = list_does && bound <= floor_live;
    sum_all = list_does && c.p < 1.f && !c.k && !whole;
  }
};

__device__ inline Weights weights_of(const PartsOf& of, const PartArgs& p, const Settings& c,
                                     const SampleArgs& a) {
  const int lane = threadIdx.x & 63;
  Weights wt;
  wt.max = wave_max<true>(lane < p.parts ? of.top[lane] : -INFINITY);
  wt.inv_t = 1.f / c.t;
  wt.scale = a.scale;
  return wt;
}

template <class T>
__global__ __launch_bounds__(kPartThreads) void sample_lists_kernel(const T* __restrict__ S,
                                                                    SampleArgs a, PartArgs p) {
  __shared__ u64 sums[kPartWaves], entries[kList];
  __shared__ int numbers[kPartWaves], counted, placed;
  const int64_t col = blockIdx.y;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  PartsOf& of = p.of[col];
  const Settings c(a, col);
  auto column = part_column(S + col * a.lds, a.m, p);
  __shared__ PartsKnown shared_known;
  if (wave == 0) {
    const PartsKnown k(of, p, c, full_units<decltype(column)::V>(a.m, p));
    if (lane == 0) shared_known = k;
  }
  if (threadIdx.x == 0) counted = 0;
  __syncthreads();
  const PartsKnown known = shared_known;
  if (known.max == -INFINITY || (c.cut && !known.list_does && !c.greedy)) return;
  Weights wt;
  wt.max = known.max;
  wt.inv_t = 1.f / c.t;
  wt.scale = a.scale;

  const bool mine = of.top[blockIdx.x] == known.max;  // the column's maximum is in this part
  u64 mass = 0;
  int number = c.greedy ? a.m : 0;
  const float from = known.whole ? known.floor_live : known.bound;
  if (c.greedy) {
    if (mine) column.each([&](float l, int i) { number = l == wt.max && i < number ? i : number; });
#pragma unroll
    for (int d = 32; d; d >>= 1) number = min(number, __shfl_xor(number, d));
  } else if (!c.cut) {
    column.groups_until([&](const float (&l)[decltype(column)::V], int) {
      add_kept(wt, c.q, l, &mass, &number);
      return true;
    });
    number = wave_sum(number);
  } else {
    column.groups_until([&](const float (&l)[decltype(column)::V], int at) {
      if (known.sum_all) mass += mass_of(wt, l);
      push_from(from, l, at, entries, kList, &counted);
      return true;
    });
  }
  mass = wave_sum(mass);
  if (lane == 0) {
    sums[wave] = mass;
    numbers[wave] = number;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = numbers[0];
    for (int w = 1; w < kPartWaves; ++w) n = c.greedy ? min(n, numbers[w]) : n + numbers[w];
    of.mass[blockIdx.x] = total_of(sums);
    (c.greedy ? of.first : of.count)[blockIdx.x] = n;
    // The order of the parts' entries in the list does not matter: it is
    // sorted.
    placed = counted ? atomicAdd(&of.listed, counted) : 0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < counted && i < kList; i += kPartThreads)
    if (placed + i < kList) of.entry[placed + i] = entries[i];
}

template <class T>
__global__ __launch_bounds__(kList) void sample_draw_kernel(const T* __restrict__ S, SampleArgs a,
                                                            PartArgs p) {
  __shared__ Shared<kList> s;
  const int64_t col = blockIdx.x;
  const T* row = S + col * a.lds;
  const PartsOf& of = p.of[col];
  const Settings c(a, col);
  const PartsKnown known(of, p, c, full_units<Column<T, kPartThreads, 0>::V>(a.m, p));
  if (known.max == -INFINITY) {
    if (threadIdx.x == 0) answer(a, col, -1, 0.f, 0);
    return;
  }
  if (c.greedy) {
    if (threadIdx.x == 0) {
      int best = a.m;
      for (int i = 0; i < p.parts; ++i) best = min(best, of.first[i]);
      answer(a, col, best, 1.f, 1);
    }
    return;
  }
  Weights wt;
  wt.max = known.max;
  wt.inv_t = 1.f / c.t;
  wt.scale = a.scale;
  if (!c.cut) {
    const int lane = threadIdx.x & 63;
    const u64 mass = lane < p.parts ? of.mass[lane] : 0, total = wave_sum(mass);
    const int many = wave_sum(lane < p.parts ? of.count[lane] : 0);
    u64 base;
    const int begin = p.part * part_of(mass, p.parts, draw_target(a.u[col], total), &base);
    narrow_and_draw<kList>(row, begin, min(a.m, begin + p.part), base, 0, total,
                           static_cast<u64>(many), 0u, 0, wt, c, a, col, s);
    return;
  }
  const u64 mass = known.sum_all ? of.total(p.parts) : 0;
  if (known.list_does && of.listed <= kList) {
    const int count = of.listed;
    const u64 entry = static_cast<int>(threadIdx.x) < count ? of.entry[threadIdx.x] : 0;
    if (list_and_draw<kList>(entry, count, mass, wt, c, a, col, s)) return;
  }
  if (p.large && known.sum_all && NucleusSteps(mass, wt, c, a.m).fit()) {
    for (int i = threadIdx.x; i < kBins; i += kList) p.of[col].guide[i] = 0;
    if (threadIdx.x == 0) p.of[col].large = 1;
    return;
  }
  __syncthreads();
  search_and_draw<kList>(row, mass, wt, c, a, col, s);
}

template <class T>
__global__ __launch_bounds__(kPartThreads) void sample_guide_kernel(const T* __restrict__ S,
                                                                    SampleArgs a, PartArgs p) {
  const int64_t col = blockIdx.y;
  PartsOf& of = p.of[col];
  if (!of.large) return;
  __shared__ unsigned guide[kBins];
  auto column = part_column(S + col * a.lds, a.m, p);
  const Settings c(a, col);
  const Weights wt = weights_of(of, p, c, a);
  const NucleusSteps steps(of.total(p.parts), wt, c, a.m);
  for (int i = threadIdx.x; i < kBins; i += kPartThreads) guide[i] = 0;
  __syncthreads();
  column.each([&](float l, int) {
    if (l >= steps.low) atomicAdd(&guide[steps.of(l)], steps.weight(l));
  });
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kPartThreads)
    if (guide[i]) atomicAdd(&of.guide[i], guide[i]);
}

template <class T>
__global__ __launch_bounds__(kPartThreads) void sample_gather_kernel(const T* __restrict__ S,
                                                                     SampleArgs a, PartArgs p) {
  const int64_t col = blockIdx.y;
  PartsOf& of = p.of[col];
  if (!of.large) return;
  __shared__ Shared<kPartThreads> s;
  __shared__ u64 entries[kList];
  __shared__ int placed;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  auto column = part_column(S + col * a.lds, a.m, p);
  const Settings c(a, col);
  const Weights wt = weights_of(of, p, c, a);
  const NucleusSteps steps(of.total(p.parts), wt, c, a.m);
  for (int i = threadIdx.x; i < kBins; i += kPartThreads) s.hist[i] = of.guide[i];
  if (threadIdx.x == 0) s.count = 0;
  find_bin(kBins, 0, steps.share, s);
  const int step = s.found_bin;
  NucleusSums sums;
  column.each([&](float l, int i) {
    sums.add(steps, step, l, wt, c, [&] {
      const int at = atomicAdd(&s.count, 1);
      if (at < kList) entries[at] = entry_of(l, i);
    });
  });
  const u64 over = wave_sum(sums.over), sum = wave_sum(sums.sum), many = wave_sum(sums.many);
  __syncthreads();
  if (lane == 0) {
    s.sum[wave] = over;
    s.sum2[wave] = sum;
    s.sum3[wave] = many;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    NucleusSums& to = of.sums[blockIdx.x];
    to.over = total_of(s.sum);
    to.sum = total_of(s.sum2);
    to.many = total_of(s.sum3);
    placed = s.count ? atomicAdd(&of.gathered, s.count) : 0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < s.count && i < kList; i += kPartThreads)
    if (placed + i < kList) of.entry[placed + i] = entries[i];
}

template <class T>
__global__ __launch_bounds__(kList) void sample_finish_kernel(const T* __restrict__ S,
                                                              SampleArgs a, PartArgs p) {
  const int64_t col = blockIdx.x;
  const PartsOf& of = p.of[col];
  if (!of.large) return;
  __shared__ Shared<kList> s;
  const T* row = S + col * a.lds;
  const Settings c(a, col);
  const Weights wt = weights_of(of, p, c, a);
  const u64 mass = of.total(p.parts);
  const int i = threadIdx.x, count = of.gathered;
  if (count <= kList) {
    const int lane = threadIdx.x & 63;
    const u64 above = wave_sum(lane < p.parts ? of.sums[lane].over : 0);
    if (i < kMaxParts) {
      s.sum2[i] = i < p.parts ? of.sums[i].sum : 0;
      s.sum3[i] = i < p.parts ? of.sums[i].many : 0;
    }
    __syncthreads();
    const u64 entry = i < count ? of.entry[i] : 0;
    if (finish_nucleus<kList>(row, entry, count, above, top_p_target(c.p, mass), p.part, wt, c, a,
                              col, s))
      return;
  }
  __syncthreads();
  search_and_draw<kList>(row, mass, wt, c, a, col, s, false);
}

// The arguments of the n columns from `first` on.
SampleArgs columns_of(const SampleArgs& a, int64_t first, int64_t n) {
  SampleArgs part = a;
  const auto from = [&](auto& p) {
    if (p) p += first;
  };
  part.n = n;
  from(part.u);
  from(part.temperature.each);
  from(part.top_p.each);
  from(part.min_p.each);
  from(part.top_k.each);
  from(part.labels);
  from(part.prob);
  from(part.kept);
  return part;
}

template <class T, int THREADS, int R>
void start_block(const SampleLaunch& l, const SampleArgs& a) {
  each_slice(l.n, 1, THREADS, [&](int64_t first, int64_t n) {
    sample_block_kernel<T, THREADS, R><<<static_cast<unsigned>(n), THREADS, 0, l.stream>>>(
        static_cast<const T*>(l.S) + first * l.lds, columns_of(a, first, n));
  });
}
template <class T, int E>
void start_wave(const SampleLaunch& l, const SampleArgs& a) {
  each_slice(l.n, 4, 256, [&](int64_t first, int64_t n) {
    sample_wave_kernel<T, E><<<static_cast<unsigned>((n + 3) / 4), 256, 0, l.stream>>>(
        static_cast<const T*>(l.S) + first * l.lds, columns_of(a, first, n));
  });
}

template <class T>
void start_parts(const SampleLaunch& l, const SampleArgs& a) {
  PartArgs p;
  p.of = static_cast<PartsOf*>(l.work);
  p.part = (a.m / kMaxParts + kPartStep) / kPartStep * kPartStep;
  p.parts = (a.m + p.part - 1) / p.part;
  // A column with a top-k has its nucleus in the list, or none at all.
  p.large = (a.top_k.each || a.top_k.value == 0) && (a.top_p.each || a.top_p.value < 1.f);
  const T* S = static_cast<const T*>(l.S);
  const dim3 grid(static_cast<unsigned>(p.parts), static_cast<unsigned>(l.n));
  sample_parts_kernel<T><<<grid, kPartThreads, 0, l.stream>>>(S, a, p);
  sample_lists_kernel<T><<<grid, kPartThreads, 0, l.stream>>>(S, a, p);
  sample_draw_kernel<T><<<static_cast<unsigned>(l.n), kList, 0, l.stream>>>(S, a, p);
  if (!p.large) return;
  sample_guide_kernel<T><<<grid, kPartThreads, 0, l.stream>>>(S, a, p);
  sample_gather_kernel<T><<<grid, kPartThreads, 0, l.stream>>>(S, a, p);
  sample_finish_kernel<T><<<static_cast<unsigned>(l.n), kList, 0, l.stream>>>(S, a, p);
}

// Columns that one workgroup's registers do not hold go to several workgroups
// each where one apiece leaves compute units idle.  Measured in us, one
// workgroup / several, for n columns of m scores:
//
//             m        n = 16     64       128      256      512
//   top-k 5   40000 f32  15/18    16/18    17/21    21/31    39/50
//             65537 f32  18/17    21/20    23/25    29/39    61/71
//            128000 f32  22/19    32/24    36/34    51/60   100/109
//            128000 f16  20/18    22/21    24/26    29/40    58/75
//   top-p .95 40000 f32  25/29    37/39    28/36    47/58    77/89
//             65537 f32  32/31    83/62    84/71    90/88   133/137
//            128000 f32  68/42   130/69   134/83   146/117  249/189
//            128000 f16  69/39   126/65   128/76   131/100  221/163
//   uncut     40000 f32  20/17    21/20    22/24    26/34    47/58
//             65537 f32  29/19    33/24    34/32    40/47    81/86
//            128000 f32  45/21    54/29    58/40    71/68   135/122
//            128000 f16  42/19    44/26    45/35    50/52   100/99
//
// The limits on n are the nucleus's, which differs most and which settings of
// each column's own may hold.  They cost a top-k or an uncut draw of 128 to
// 256 columns up to 11 us (20/31 for 256 of 65537 f16), and a nucleus of
// more than 256 columns of 128000 the 60 us that several would save.
bool in_parts(int64_t m, int64_t n) { return m > 32768 && n <= (m > 65536 ? 256 : 64); }

template <class T>
hipError_t sample(const SampleLaunch& l) {
  SampleArgs a;
  a.m = static_cast<int>(l.m);
  a.n = l.n;
  a.lds = l.lds;
  a.u = l.u;
  a.temperature = l.temperature;
  a.top_p = l.top_p;
  a.min_p = l.min_p;
  a.top_k = l.top_k;
  a.labels = l.labels;
  a.prob = l.prob;
  a.kept = l.kept;
  int bits = 0;
  while ((int64_t(1) << bits) < l.m) ++bits;
  a.scale = static_cast<double>(u64(1) << (62 - bits < 46 ? 62 - bits : 46));
  // Else by the column's length: a wave up to 2048 scores (8000 columns of
  // 2000: 31 us with a top-k, 110 by a workgroup; one column 7.4 and 9.3), a
  // workgroup that holds the column in registers above, 16 scores to a
  // thread (with four waves the arguments and settings lie in 224 to 260 bytes
  // of scratch, read again for each group), and one that reads it twice from
  // there on.  (32 to a thread spill:
  // a top-k of 32000 floats took 18 us, against 14 read twice; 12000 take 11
  // held, 12 read.)
  if (in_parts(l.m, l.n)) start_parts<T>(l, a);
  else if (l.m <= 256) start_wave<T, 4>(l, a);
  else if (l.m <= 1024) start_wave<T, 16>(l, a);
  else if (l.m <= 2048) start_wave<T, 32>(l, a);
  else if (l.m <= 256 * 16) start_block<T, 256, 16>(l, a);
  else if (l.m <= 1024 * 16) start_block<T, 1024, 16>(l, a);
  else start_block<T, 1024, 0>(l, a);
  return hipGetLastError();
}

}  // namespace

size_t sample_work_bytes(int64_t m, int64_t n) {
  return in_parts(m, n) ? static_cast<size_t>(n) * sizeof(PartsOf) : 0;
}

hipError_t launch_sample(const SampleLaunch& a) {
  switch (a.data) {
    case SDCA_F32: return sample<float>(a);
    case SDCA_F64: return sample<double>(a);
    case SDCA_F16: return sample<__half>(a);
    default: return sample<__hip_bfloat16>(a);
  }
}

}  // namespace sdca_gpu
