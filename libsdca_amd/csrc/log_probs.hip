// Log-probabilities of given labels, and their gradient.
//
// For a column of m scores s with the largest M and a temperature T, the
// weights are w_j = exp((s_j - M) / T) (1 where s_j = M), Z their sum and
// p_j = w_j / Z the probabilities; a label's log-probability is log p_label,
// the entropy H = log Z - sum w_j log w_j / Z, and with a gradient g of the
// log-probability and h of the entropy the scores' gradient is
//   d_j = (g ([j = label] - p_j) - h p_j (log p_j + H)) / T.
//
// A column goes by once: each lane keeps a running maximum with Z and
// sum w log w relative to it, and brings them to a larger maximum when one
// comes.  Exponents are in base 2, relative to a reference rather than to
// the maximum itself: with c = log2(e) / T and ref = M c rounded and held
// within +-2^24, e_j = fma(s_j, c, -ref) is one instruction, and the same
// reference in every term cancels in the differences that are the results.
// Up to 2^24 the rounding is half a unit at most: the weights' largest is
// between 2^-1/2 and 2^1/2.  (At 2^32 it is 2^7 or more, and the weights
// infinite or 0.)  Scores masked at -1e9, at the type's lowest value or at
// -infinity then have weight 0 beside any ordinary score.  Where a maximum is
// far, M c beyond 2^24 (large scores, a temperature near nothing, +infinity, or
// nothing but masks), exponents are (s_j - M) c instead.  Log-probabilities
// then take a second pass, over the column or a workgroup's part of it, from
// the caches; the gradient's kernels have them in the pass that they make.
// (64 columns of 128000 bfloat16, top 20, us: ordinary 17.4, one all masks
// 22.9, all such 23.7, all but 100 scores of each at -1e9 23.4.  With such
// exponents in the first pass 17.6, 20.9, 21.6 and 21.8, but 600 x 64000 19.2
// where it is 18.2, and 64 x 128000 with masks in some columns 21.7, not 20.9.)
#include <type_traits>

#include "answer_launch.hpp"
#include "answer_limits.hpp"
#include "answer_types.hpp"
#include "answer_wave.hpp"
#include "common.hpp"

namespace sdca_gpu {
namespace {

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
constexpr float kFar = 16777216.f;
constexpr float kLowest = -3.402823466e38f;
// Exponents below this have weight 0, and 0 times this is 0.
constexpr float kGone = -200.f;

__device__ inline float exp2_of(float e) { return __builtin_amdgcn_exp2f(e); }
__device__ inline float ref_of(float max, float c) { return fminf(fmaxf(max * c, -kFar), kFar); }
__device__ inline bool is_far(float max, float c) { return fabsf(max * c) > kFar && max > -INFINITY; }
// s - max where infinities are equal, and NaN stays.
__device__ inline float below(float s, float max) { return s == max ? 0.f : s - max; }

// 16 bytes of a column as words, and as floats.  (Held as elements, 16-bit
// scores take a register each.)
template <class T>
__device__ inline unsigned bits_of(T x) {
  unsigned b = 0;
  __builtin_memcpy(&b, &x, sizeof(T));
  return b;
}
// The scores from `at` on, -infinity before `begin` and from `end` on.
template <class T>
__device__ inline void load_words(const T* row, int64_t at, int64_t begin, int64_t end,
                                  unsigned (&w)[4]) {
  constexpr int V = 16 / static_cast<int>(sizeof(T)), kIn = V / 4;
  if (at >= begin && at + V <= end) {
    __builtin_memcpy(w, row + at, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int e = 0; e < kIn; ++e) {
        const int64_t k = at + i * kIn + e;
        w[i] |= bits_of(k >= begin && k < end ? row[k] : from_float<T>(-INFINITY)) << (16 * e);
      }
    }
  }
}
// How many values a column's first value is behind a multiple of 16 bytes:
// vectors are taken from there on (2048 columns of 100003 halves at 2 bytes'
// alignment 91 us, of 100000 84).
template <class T>
__device__ inline int behind_16(const T* row) {
  return static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
}
// What exponents are relative to: the maximum itself where it is far, or a
// reference.
struct Origin {
  float from, ref;
  __device__ Origin(float max, float c) {
    const bool far = is_far(max, c);
    from = far ? max : 0.f;
    ref = far ? 0.f : ref_of(max, c);
  }
  __device__ float exponent(float s, float c) const { return fmaf(below(s, from), c, -ref); }
};
// The weights of some scores: their largest, and the sums of 2^e and e 2^e
// with exponents relative to its origin.  (A NaN among the scores makes the
// sums NaN and leaves max.)
struct Mass {
  float max = -INFINITY, sum = 0.f, weighted = 0.f;

  __device__ void shift(float by) {
    const float f = exp2_of(by);
    weighted = f * fmaf(fmaxf(by, kGone), sum, weighted);
    sum *= f;
  }
  // To a larger or equal maximum.
  template <bool ANY>
  __device__ void rise(float to, float c) {
    if constexpr (ANY) {
      const Origin old(max, c), now(to, c);
      // (By 1/2 at most where there is a weight; without one it can be large.)
      shift(fminf(fmaf(below(old.from, now.from), c, old.ref - now.ref), 1.f));
    } else {
      shift(ref_of(max, c) - ref_of(to, c));
    }
    max = to;
  }
  // A lane's scores (as words); returns their largest.  Without ANY as if no
  // maximum were far: a negative one's weights are then too small, and a
  // positive one's mean nothing.
  template <class T, bool ANY, int N>
  __device__ float add(const unsigned (&raw)[N][4], float c) {
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    float v[N][V], most = -INFINITY;
#pragma unroll
    for (int u = 0; u < N; ++u) unpack<T>(raw[u], v[u]);
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) most = fmaxf(most, v[u][e]);
    if (most > max) rise<ANY>(most, c);
    const Origin origin(max, c);
    if (!ANY || !__ballot(origin.from != 0.f)) {
      const float ref = ref_of(max, c);
      weigh(v, [&](float x) { return fmaf(x, c, -ref); });
    } else {
      weigh(v, [&](float x) { return origin.exponent(x, c); });
    }
    return most;
  }
  // A vector of a lane's scores beside a far maximum that is not below them.
  template <class T>
  __device__ void add_below(const unsigned (&raw)[4], float c) {
    float v[1][16 / sizeof(T)];
    unpack<T>(raw, v[0]);
    weigh(v, [&](float x) { return below(x, max) * c; });
  }
  // All lanes' together, in every lane; `most` is their largest.
  template <bool ANY>
  __device__ void over_wave(float c) { over_wave<ANY>(wave_max<true>(max), c); }
  template <bool ANY>
  __device__ void over_wave(float most, float c) {
    rise<ANY>(most, c);
    sum = wave_total(sum);
    weighted = wave_total(weighted);
  }

 private:
  template <int N, int V, class Exponent>
  __device__ void weigh(const float (&v)[N][V], Exponent exponent) {
    float s = 0.f, w_e = 0.f;
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x = exponent(v[u][e]), w = exp2_of(x);
        s += w;
        w_e = fmaf(w, fmaxf(x, kGone), w_e);
      }
    sum += s;
    weighted += w_e;
  }
};

// ---------------------------------------------------------------------------
// The best of a column: a wave's 64 entries (score, index) by lane, falling.
// Candidates, which are entries of at least a bound, gather in LDS; 64 of
// them are sorted and merged into the list.  The bound has an index too: of
// very many equal scores (a mask of the lowest value) only those of low index
// are candidates (64 rows of 128000, some so masked: 63 us with the score
// alone, 16 with both).
// ---------------------------------------------------------------------------
struct Best {
  u64 list = 0;
  float bound = kLowest;  // a score below it, or -infinity or NaN, is none
  int index = 0x7fffffff;  // the last index at which the bound itself is one
  int waiting = 0;

  __device__ void merge_sorted(u64 rising) {
    list = rising > list ? rising : list;
    list = sort_merge<32, true>(list, true);
  }
  __device__ void at_least(u64 entry) {
    if (!entry) return;
    bound = score_of(static_cast<unsigned>(entry >> 32));
    index = index_of(entry);
  }
  __device__ void merge(u64 some, int top) {
    merge_sorted(sort_wave<true>(some, false));
    at_least(read_lane64(list, top - 1));
  }
  __device__ void take(float s, int at, u64* room, int top) {
    if (!__ballot(s >= bound)) return;
    const bool candidate = s > bound || (s == bound && at <= index);
    const u64 mask = __ballot(candidate);
    if (!mask) return;
    const int lane = threadIdx.x & 63;
    if (candidate) {
      const int before = __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(mask >> 32),
                                                   __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(mask), 0));
      room[waiting + before] = entry_of(s, at);
    }
    waiting += __popcll(mask);
    if (waiting < 64) return;
    wave_lds_sync();
    const u64 first = room[lane], rest = room[64 + lane];
    wave_lds_sync();
    room[lane] = rest;
    wave_lds_sync();
    waiting -= 64;
    merge(first, top);
  }
  __device__ void finish(u64* room, int top) {
    if (!waiting) return;
    const int lane = threadIdx.x & 63;
    wave_lds_sync();
    merge(lane < waiting ? room[lane] : 0, top);
    waiting = 0;
  }
};

struct LogProbsArgs {
  int m;
  int64_t n, lds;
  const int64_t* labels;
  float inv_t;
  int top;
  float *logp, *entropy, *stats, *top_logp;
  int64_t* top_index;
  // Columns in parts: `length` scores each, their masses and best.
  int parts, length;
  Mass* masses;
  u64* lists;
};

// A column's label and its score, read before the column goes by.
struct Own {
  int64_t label = -1;
  float score = 0.f;
  template <class T>
  __device__ Own(const T* row, int64_t col, const LogProbsArgs& a) {
    if (a.logp) label = a.labels[col];
    if (label >= 0 && label < a.m) score = to_float(row[label]);
  }
};

// A column's results, by one wave.
__device__ inline void finish(int64_t col, const Mass& mass, u64 list, const Own& own, const LogProbsArgs& a) {
  const int lane = threadIdx.x & 63;
  const float c = a.inv_t * kLog2e, max = mass.max;
  const Origin origin(max, c);
  const auto exponent = [&](float s) { return origin.exponent(s, c); };
  const bool none = max == -INFINITY && mass.sum == 0.f;
  const float log_sum = log2f(mass.sum);
  float entropy = none ? 0.f : (log_sum - mass.weighted / mass.sum) * kLn2;
  if (entropy < 0.f) entropy = 0.f;
  const auto logp = [&](float s) { return none ? -INFINITY : (exponent(s) - log_sum) * kLn2; };
  if (lane == 0) {
    if (a.logp)
      a.logp[col] = own.label == -1 ? 0.f : own.label < 0 || own.label >= a.m ? NAN : logp(own.score);
    if (a.entropy) a.entropy[col] = entropy;
    if (a.stats) {
      float* out = a.stats + 3 * col;
      out[0] = max;
      // The sum relative to the maximum, not to the reference.
      out[1] = none ? -INFINITY : (log_sum - exponent(max)) * kLn2;
      out[2] = entropy;
    }
  }
  if (lane < a.top) {
    const float s = score_of(static_cast<unsigned>(list >> 32));
    if (a.top_logp) a.top_logp[col * a.top + lane] = list ? logp(s) : -INFINITY;
    if (a.top_index) a.top_index[col * a.top + lane] = list ? index_of(list) : -1;
  }
}

// The masses of WAVES waves, and their best, in the first.  again(max) sees the
// largest of all, and returns in all waves whether it has changed the masses.
template <int WAVES, bool TOP, class Again>
__device__ inline void join_waves(Mass& mass, u64& list, u64 (*room)[128], float c, int wave, Again again) {
  __shared__ float of_wave[WAVES][3];
  const int lane = threadIdx.x & 63;
  const auto give = [&] {
    if (lane == 0) {
      of_wave[wave][0] = mass.max;
      of_wave[wave][1] = mass.sum;
      of_wave[wave][2] = mass.weighted;
    }
  };
  Mass all;  // a wave's by lane
  const auto take = [&] {
    if (lane < WAVES) {
      all.max = of_wave[lane][0];
      all.sum = of_wave[lane][1];
      all.weighted = of_wave[lane][2];
    }
  };
  float most = 0.f;
  give();
#pragma unroll
  for (int s = 1; s < WAVES; s *= 2) {
    if (TOP && (wave & (2 * s - 1)) == s) room[wave][lane] = list;
    if (TOP || s == 1) __syncthreads();
    if (s == 1) {
      if constexpr (TOP) {  // (few registers beside the lists: 20 x 166617 halves 17.6 us, 18.2 as below)
        most = of_wave[0][0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) most = fmaxf(most, of_wave[w][0]);
      } else {
        take();
        most = wave_max<true>(all.max);
      }
      if (again(most)) {
        __syncthreads();
        give();
        __syncthreads();
        take();
      }
    }
    if (TOP && (wave & (2 * s - 1)) == 0) {
      Best b;
      b.list = list;
      b.merge_sorted(room[wave + s][63 - lane]);
      list = b.list;
    }
  }
  if (wave == 0) {
    if (TOP) take();
    mass = all;
    mass.over_wave<true>(most, c);
  }
}

// WAVES waves to a column, or to a part of it; with one wave, four columns to
// a workgroup.  A wave takes 64 kLoads vectors of 16 bytes at a time.
template <class T, int WAVES, bool TOP>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void log_probs_kernel(
    const T* __restrict__ S, LogProbsArgs a) {
  constexpr int V = 16 / static_cast<int>(sizeof(T)), kLoads = 4, kStep = 64 * V * kLoads;
  constexpr int kColumns = WAVES == 1 ? 4 : 1;
  __shared__ u64 room[TOP ? kColumns * WAVES : 1][128];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kColumns + (WAVES == 1 ? wave : 0);
  if (WAVES == 1 && col >= a.n) return;  // whole waves, and no barrier below
  const T* row = S + col * a.lds;
  const float c = a.inv_t * kLog2e;
  const int first = blockIdx.y * a.length, end = min(a.m, first + a.length);
  const Own own(row, col, a);

  Mass mass;
  Best best;
  bool started = false;
  const int64_t begin = first - behind_16(row + first) + (WAVES == 1 ? 0 : wave) * kStep;
  for (int64_t at = begin; at < end; at += WAVES * kStep) {
    unsigned raw[kLoads][4];
    if (at >= first && at + kStep <= end) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) __builtin_memcpy(raw[u], row + at + (u * 64 + lane) * V, 16);
    } else {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) load_words(row, at + (u * 64 + lane) * V, first, end, raw[u]);
    }
    const float most = mass.add<T, false>(raw, c);
    if constexpr (TOP) {
      if (!started) {
        // `top` lanes have a score of at least this.
        best.bound = fmaxf(read_lane(sort_wave<true>(most, true), a.top - 1), kLowest);
        started = true;
      }
      if (__ballot(most >= best.bound)) {
        float v[kLoads][V];
#pragma unroll
        for (int u = 0; u < kLoads; ++u) unpack<T>(raw[u], v[u]);
#pragma unroll
        for (int u = 0; u < kLoads; ++u)
#pragma unroll
          for (int e = 0; e < V; ++e)
            best.take(v[u][e], static_cast<int>(at) + (u * 64 + lane) * V + e, room[wave], a.top);
      }
    }
  }
  if constexpr (TOP) best.finish(room[wave], a.top);
  mass.over_wave<false>(c);
  // Where the largest of the column, or of the workgroup's part, is far: the
  // weights once more, from differences.
  const auto again = [&](float most) {
    if (!__builtin_amdgcn_readfirstlane(is_far(most, c))) return false;
    mass.max = most;
    mass.sum = mass.weighted = 0.f;
    // (A loop keeps the kernels with alternatives short: 20 x 166617 halves 17.6 us,
    // 18.3 with it unrolled; 2048 x 100003 halves without 82.5, unrolled 81.1.)
    constexpr int kInLine = TOP || WAVES == 1 ? 1 : kLoads;
    for (int64_t at = begin; at < end; at += WAVES * kStep) {
#pragma unroll kInLine
      for (int u = 0; u < kLoads; ++u) {
        unsigned raw[4];
        load_words(row, at + (u * 64 + lane) * V, first, end, raw);
        mass.add_below<T>(raw, c);
      }
    }
    mass.over_wave<true>(c);
    return true;
  };
  if constexpr (WAVES == 1) {
    again(mass.max);
  } else {
    join_waves<WAVES, TOP>(mass, best.list, room, c, wave, again);
    if (wave) return;
  }
  if (a.parts == 1) {
    finish(col, mass, best.list, own, a);
  } else {
    const int64_t part = col * a.parts + blockIdx.y;
    if (lane == 0) a.masses[part] = mass;
    if (TOP && lane < a.top) a.lists[part * a.top + lane] = best.list;
  }
}

// A column from its parts (64 of them at most).
constexpr int kJoinWaves = 4;
template <class T, bool TOP>
__global__ __launch_bounds__(64 * kJoinWaves) void log_probs_join_kernel(const T* __restrict__ S,
                                                                         LogProbsArgs a) {
  __shared__ u64 room[TOP ? kJoinWaves : 1][128];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t col = blockIdx.x;
  const float c = a.inv_t * kLog2e;
  const Own own(S + col * a.lds, col, a);
  Mass mass;
  const int mine = wave + lane * kJoinWaves;
  if (mine < a.parts) mass = a.masses[col * a.parts + mine];
  mass.over_wave<true>(c);
  Best best;
  if constexpr (TOP) {
    for (int p = wave; p < a.parts; p += kJoinWaves)
      best.merge_sorted(63 - lane < a.top ? a.lists[(col * a.parts + p) * a.top + 63 - lane] : 0);
  }
  join_waves<kJoinWaves, TOP>(mass, best.list, room, c, wave, [](float) { return false; });
  if (wave == 0) finish(col, mass, best.list, own, a);
}

// How a launch takes the columns: waves to a part, parts to a column.
struct LogProbsPlan {
  int waves, parts, length;
};
LogProbsPlan plan_log_probs(int64_t m, int64_t n) {
  const auto split = [&](int64_t parts) {
    const int64_t length = ((m + parts - 1) / parts + 2047) / 2048 * 2048;
    return LogProbsPlan{4, static_cast<int>((m + length - 1) / length), static_cast<int>(length)};
  };
  // us without and with 10 alternatives: 500 x 2000 floats 7.2, 9.1 by one wave
  // to a column, 7.4, 13.9 by sixteen; 5000 x 4000 16, 22 by one, 16, 31 by
  // four, but 4 x 4000 4.8, 11.5 and by sixteen 4.0, 7.9.
  if (m <= 2048 || (m <= 8192 && n >= 2048)) return {1, 1, static_cast<int>(m)};
  // 300 x 64000 bfloat16 14.4, 22.3 in parts, 13.7, 29.3 by four waves; 600 x
  // 64000 20.4, 32.0 and 18.2, 33.1.
  if (n < 512 && m > 32768) {
    const int64_t parts = (1024 + n - 1) / n, most = (m + 8191) / 8192;
    return split(parts < most ? (parts < 64 ? parts : 64) : (most < 64 ? most : 64));
  }
  // 1 x 16000 floats 4.3, 9.1 by sixteen waves, 4.9, 12.0 by four; 300 x 16000
  // bfloat16 7.3, 16.6 and 6.4, 12.2.
  if (n < 256) return {16, 1, static_cast<int>(m)};
  return {4, 1, static_cast<int>(m)};
}

template <class T, int WAVES, bool TOP>
void start(const LogProbsLaunch& l, LogProbsArgs a) {
  constexpr int64_t kColumns = WAVES == 1 ? 4 : 1;
  constexpr int kThreads = WAVES == 1 ? 256 : 64 * WAVES;
  const int64_t n = a.n;
  each_slice(n, kColumns, static_cast<int64_t>(kThreads) * a.parts, [&](int64_t first, int64_t count) {
    LogProbsArgs s = a;
    s.n = count;
    s.labels = a.labels + first;
    if (a.logp) s.logp = a.logp + first;
    if (a.entropy) s.entropy = a.entropy + first;
    if (a.stats) s.stats = a.stats + 3 * first;
    if (a.top_logp) s.top_logp = a.top_logp + first * a.top;
    if (a.top_index) s.top_index = a.top_index + first * a.top;
    s.masses = a.masses + first * a.parts;
    s.lists = a.lists + first * a.parts * a.top;
    const T* S = static_cast<const T*>(l.S) + first * a.lds;
    log_probs_kernel<T, WAVES, TOP>
        <<<dim3(static_cast<unsigned>((count + kColumns - 1) / kColumns), a.parts), kThreads, 0, l.stream>>>(S, s);
    if (a.parts > 1)
      log_probs_join_kernel<T, TOP><<<static_cast<unsigned>(count), 64 * kJoinWaves, 0, l.stream>>>(S, s);
  });
}

template <class T, bool TOP>
void log_probs(const LogProbsLaunch& l) {
  const LogProbsPlan plan = plan_log_probs(l.m, l.n);
  LogProbsArgs a = {};
  a.m = static_cast<int>(l.m);
  a.n = l.n;
  a.lds = l.lds;
  a.labels = l.labels;
  a.inv_t = l.inv_t;
  a.top = l.top;
  a.logp = l.logp;
  a.entropy = l.entropy;
  a.stats = l.stats;
  a.top_logp = l.top_logp;
  a.top_index = l.top_index;
  a.parts = plan.parts;
  a.length = plan.length;
  a.masses = static_cast<Mass*>(l.work);
  a.lists = reinterpret_cast<u64*>(static_cast<char*>(l.work) +
                                   (plan.parts > 1 ? (l.n * plan.parts * sizeof(Mass) + 15) / 16 * 16 : 0));
  switch (plan.waves) {
    case 1: return start<T, 1, TOP>(l, a);
    case 4: return start<T, 4, TOP>(l, a);
    default: return start<T, 16, TOP>(l, a);
  }
}

template <class T>
hipError_t log_probs(const LogProbsLaunch& l) {
  l.top ? log_probs<T, true>(l) : log_probs<T, false>(l);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// The gradient.
// ---------------------------------------------------------------------------
struct GradArgs {
  int m;
  int64_t n, lds, ldd;
  const int64_t* labels;
  const float *g, *h, *stats;
  float inv_t;
  float* logp;
};

// A column's own numbers.  With weights w = 2^e whose sum is 2^log2_sum, the
// gradient of a score that is not the label's is w (c1 + c2 e).  The constants
// have 1 / T in them, or where they could then pass the largest float
// (`apart`: of a weight of 0 they would make NaN) it is multiplied last.
struct GradColumn {
  float log2_sum, c1, c2, g, h;
  int label;
  bool none, apart;

  __device__ GradColumn(const GradArgs& a, int64_t col) {
    const int64_t l = a.labels[col];
    // (Far below the first vector, which starts up to 15 before the column.)
    label = l >= 0 && l < a.m ? static_cast<int>(l) : -0x7fffffff;
    g = l == -1 ? 0.f : label < 0 ? NAN : a.g[col];
    h = a.h ? a.h[col] : 0.f;
    // (log p and e are below 256 in size where there is a weight.)
    apart = !((fabsf(g) + 512.f * fabsf(h)) * a.inv_t < 1e38f);
    if (!apart) g *= a.inv_t, h *= a.inv_t;
    if (a.logp && label < 0 && threadIdx.x % 64 == 0) a.logp[col] = l == -1 ? 0.f : NAN;
  }
  __device__ void set(float log_sum, float entropy, bool empty) {
    log2_sum = log_sum;
    none = empty;
    const float one = exp2_of(-log2_sum);
    c1 = none ? g * 0.f : -one * fmaf(h, fmaf(-log2_sum, kLn2, entropy), g);
    c2 = none ? 0.f : -one * h * kLn2;
  }
  template <bool H>
  __device__ float of(float e) const {
    const float w = exp2_of(e);
    return H ? w * fmaf(c2, fmaxf(e, kGone), c1) : w * c1;
  }
};

// V scores of a column, from `at` on, to their gradients; the lane that has
// the label's writes its log-probability.  (S and D may be one matrix: a lane
// has read what it writes.)
template <bool H, bool APART, class T, int V, class Exponent>
__device__ inline void grad_vec(const unsigned (&raw)[4], int at, int m, const GradColumn& c, float last,
                                Exponent exponent, float* logp, T* d) {
  const auto result = [&](float x) { return from_float<T>(APART ? x * last : x); };
  float s[V];
  unpack<T>(raw, s);
  T out[V];
#pragma unroll
  for (int e = 0; e < V; ++e) out[e] = result(c.of<H>(exponent(s[e])));
  if (c.label >= at && c.label < at + V) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (c.label == at + e) {
        const float x = exponent(s[e]);
        if (!c.none) out[e] = result(c.of<H>(x) + c.g);
        if (logp) *logp = c.none ? -INFINITY : (x - c.log2_sum) * kLn2;
      }
  }
  if (at >= 0 && at + V <= m) {
    unsigned words[4];  // (one store; of elements it would be four)
    __builtin_memcpy(words, out, 16);
    __builtin_memcpy(d + at, words, 16);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (at + e >= 0 && at + e < m) d[at + e] = out[e];
  }
}

// From the columns' statistics.  A workgroup takes 256 kLoads vectors of a
// column (ROWS = 1), or each of its waves a column of its own.
template <class T, int ROWS, bool H>
__global__ __launch_bounds__(256) void log_probs_grad_kernel(const T* S, T* D, GradArgs a) {
  constexpr int V = 16 / static_cast<int>(sizeof(T)), kLoads = 4, kLanes = 256 / ROWS;
  const int lane = threadIdx.x % kLanes;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / kLanes;
  if (col >= a.n) return;
  GradColumn c(a, col);
  const float* stats = a.stats + 3 * col;
  const float max = stats[0], by = a.inv_t * kLog2e;
  c.set(stats[1] * kLog2e, stats[2], max == -INFINITY && stats[1] == -INFINITY);
  const auto exponent = [&](float s) { return fminf(s - max, 0.f) * by; };
  const T* s = S + col * a.lds;
  T* d = D + col * a.ldd;
  float* logp = a.logp ? a.logp + col : nullptr;
  constexpr int kStep = kLanes * V * kLoads;
  const float last = c.apart ? a.inv_t : 1.f;
  for (int64_t at0 = static_cast<int64_t>(blockIdx.y) * kStep - behind_16(s); at0 < a.m;
       at0 += static_cast<int64_t>(gridDim.y) * kStep) {
    unsigned raw[kLoads][4];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) load_words(s, at0 + (u * kLanes + lane) * V, 0, a.m, raw[u]);
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int64_t at = at0 + (u * kLanes + lane) * V;
      if (at >= a.m) break;
      grad_vec<H, true, T, V>(raw[u], static_cast<int>(at), a.m, c, last, exponent, logp, d);
    }
  }
}

// The whole column in registers: its statistics and then its gradient from
// one reading.  WAVES waves to a column (with one, four columns to a
// workgroup), NV vectors to a lane.
//
// Scores stay as they came and are converted again for each use, one vector
// after the other: as floats 16-bit ones take twice the registers, which
// leaves one workgroup of 1024 to a compute unit, whose loads and exponentials
// do not overlap.
template <int NV>
__device__ inline void keep_words(unsigned (&raw)[NV][4]) {
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(raw[u][i]));
}
template <class T, int WAVES, int NV, bool H>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES, WAVES == 16 ? 8 : 1) void log_probs_grad_whole_kernel(
    const T* S, T* D, GradArgs a) {
  constexpr int V = 16 / static_cast<int>(sizeof(T)), kLanes = 64 * WAVES;
  constexpr int kColumns = WAVES == 1 ? 4 : 1;
  __shared__ float part[3][WAVES];
  const int lane = threadIdx.x % kLanes;
  const int wave = __builtin_amdgcn_readfirstlane(lane >> 6);
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kColumns + threadIdx.x / kLanes;
  if (WAVES == 1 && col >= a.n) return;
  const T* s = S + col * a.lds;
  const int at0 = lane * V - behind_16(s);
  unsigned raw[NV][4];
#pragma unroll
  for (int u = 0; u < NV; ++u) load_words(s, at0 + u * kLanes * V, 0, a.m, raw[u]);
  GradColumn c(a, col);
  float max = -INFINITY;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    float v[V];
    unpack<T>(raw[u], v);
#pragma unroll
    for (int e = 0; e < V; ++e) max = fmaxf(max, v[e]);
  }
  max = wave_max<true>(max);
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) part[0][wave] = max;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) max = fmaxf(max, part[0][w]);
  }
  keep_words(raw);
  const float by = a.inv_t * kLog2e, ref = ref_of(max, by);
  const Origin origin(max, by);
  const bool odd = is_far(max, by) || c.apart;
  float sum = 0.f, weighted = 0.f;
  const auto add = [&](auto exponent) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      float v[V];
      unpack<T>(raw[u], v);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x = exponent(v[e]), w = exp2_of(x);
        sum += w;
        weighted = fmaf(w, fmaxf(x, kGone), weighted);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (odd) add([&](float x) { return origin.exponent(x, by); });
  else add([&](float x) { return fmaf(x, by, -ref); });
  sum = wave_total(sum);
  weighted = wave_total(weighted);
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) part[1][wave] = sum, part[2][wave] = weighted;
    __syncthreads();
    sum = weighted = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += part[1][w], weighted += part[2][w];
  }
  keep_words(raw);
  const float log2_sum = log2f(sum);
  float entropy = (log2_sum - weighted / sum) * kLn2;
  if (entropy < 0.f) entropy = 0.f;
  c.set(log2_sum, entropy, max == -INFINITY && sum == 0.f);
  T* d = D + col * a.ldd;
  float* logp = a.logp ? a.logp + col : nullptr;
  const auto write = [&](auto apart, auto exponent) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int at = at0 + u * kLanes * V;
      if (at >= a.m) break;
      grad_vec<H, apart, T, V>(raw[u], at, a.m, c, c.apart ? a.inv_t : 1.f, exponent, logp, d);
      __builtin_amdgcn_sched_barrier(0);  // (all vectors' temporaries at once do not fit)
    }
  };
  if (odd) write(std::true_type(), [&](float x) { return origin.exponent(x, by); });
  else write(std::false_type(), [&](float x) { return fmaf(x, by, -ref); });
}

// A longer column by one workgroup that goes through it twice: for the
// statistics, and backwards for the gradient, which finds the column's end in
// the L2 and the rest in the last-level cache.
constexpr int kTwiceWaves = 16;
template <class T, bool H>
__global__ __launch_bounds__(64 * kTwiceWaves, 8) void log_probs_grad_twice_kernel(const T* S, T* D, GradArgs a) {
  constexpr int V = 16 / static_cast<int>(sizeof(T)), kLoads = 4, kLanes = 64 * kTwiceWaves;
  constexpr int kStep = kLanes * V * kLoads;
  __shared__ float part[3][kTwiceWaves];
  const int lane = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(lane >> 6);
  const int64_t col = blockIdx.x;
  const T* s = S + col * a.lds;
  T* d = D + col * a.ldd;
  const float by = a.inv_t * kLog2e;
  GradColumn c(a, col);
  const int64_t begin = -static_cast<int64_t>(behind_16(s));
  const int64_t steps = (a.m - begin + kStep - 1) / kStep;
  const auto load = [&](int64_t step, unsigned (&raw)[kLoads][4]) {
    const int64_t at0 = begin + step * kStep;
    if (at0 >= 0 && at0 + kStep <= a.m) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) __builtin_memcpy(raw[u], s + at0 + (u * kLanes + lane) * V, 16);
    } else {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) load_words(s, at0 + (u * kLanes + lane) * V, 0, a.m, raw[u]);
    }
  };
  Mass mass;
  for (int64_t step = 0; step < steps; ++step) {
    unsigned raw[kLoads][4];
    load(step, raw);
    mass.add<T, true>(raw, by);
  }
  mass.over_wave<true>(by);
  if ((lane & 63) == 0) part[0][wave] = mass.max, part[1][wave] = mass.sum, part[2][wave] = mass.weighted;
  __syncthreads();
  mass = Mass();
  if ((lane & 63) < kTwiceWaves) {
    mass.max = part[0][lane & 63];
    mass.sum = part[1][lane & 63];
    mass.weighted = part[2][lane & 63];
  }
  mass.over_wave<true>(by);
  const float max = mass.max, ref = ref_of(max, by);
  const Origin origin(max, by);
  const bool odd = is_far(max, by) || c.apart;
  const float log2_sum = log2f(mass.sum);
  float entropy = (log2_sum - mass.weighted / mass.sum) * kLn2;
  if (entropy < 0.f) entropy = 0.f;
  c.set(log2_sum, entropy, max == -INFINITY && mass.sum == 0.f);
  float* logp = a.logp ? a.logp + col : nullptr;
  for (int64_t step = steps - 1; step >= 0; --step) {
    unsigned raw[kLoads][4];
    load(step, raw);
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int64_t at = begin + step * kStep + (u * kLanes + lane) * V;
      if (at >= a.m) break;
      if (odd) {
        grad_vec<H, true, T, V>(raw[u], static_cast<int>(at), a.m, c, c.apart ? a.inv_t : 1.f,
                                [&](float x) { return origin.exponent(x, by); }, logp, d);
      } else {
        grad_vec<H, false, T, V>(raw[u], static_cast<int>(at), a.m, c, 1.f,
                                 [&](float x) { return fmaf(x, by, -ref); }, logp, d);
      }
    }
  }
}

// From so many columns on they go to a workgroup each.
constexpr int64_t kTwiceColumns = 256;

// Columns that the whole-column kernel holds, wherever they start.
template <class T>
constexpr int64_t whole_most(int vectors = 1024 * 4) {
  return (vectors - 1) * int64_t(16) / static_cast<int64_t>(sizeof(T)) + 1;
}

template <class T>
GradArgs args_of(const LogProbsGradLaunch& l, int64_t first, int64_t count) {
  GradArgs a;
  a.m = static_cast<int>(l.m);
  a.n = count;
  a.lds = l.lds;
  a.ldd = l.ldd;
  a.labels = l.labels + first;
  a.g = l.g + first;
  a.h = l.h ? l.h + first : nullptr;
  a.stats = l.stats ? l.stats + 3 * first : nullptr;
  a.inv_t = l.inv_t;
  a.logp = l.logp ? l.logp + first : nullptr;
  return a;
}

template <class T, int WAVES, int NV>
void start_whole(const LogProbsGradLaunch& l) {
  constexpr int64_t kColumns = WAVES == 1 ? 4 : 1;
  constexpr int kThreads = WAVES == 1 ? 256 : 64 * WAVES;
  each_slice(l.n, kColumns, kThreads, [&](int64_t first, int64_t count) {
    const auto kernel = l.h ? log_probs_grad_whole_kernel<T, WAVES, NV, true>
                            : log_probs_grad_whole_kernel<T, WAVES, NV, false>;
    kernel<<<static_cast<unsigned>((count + kColumns - 1) / kColumns), kThreads, 0, l.stream>>>(
        static_cast<const T*>(l.S) + first * l.lds, static_cast<T*>(l.D) + first * l.ldd,
        args_of<T>(l, first, count));
  });
}

template <class T>
void start_twice(const LogProbsGradLaunch& l) {
  each_slice(l.n, 1, 64 * kTwiceWaves, [&](int64_t first, int64_t count) {
    const auto kernel = l.h ? log_probs_grad_twice_kernel<T, true> : log_probs_grad_twice_kernel<T, false>;
    kernel<<<static_cast<unsigned>(count), 64 * kTwiceWaves, 0, l.stream>>>(
        static_cast<const T*>(l.S) + first * l.lds, static_cast<T*>(l.D) + first * l.ldd,
        args_of<T>(l, first, count));
  });
}

template <class T, int ROWS>
void start_grad(const LogProbsGradLaunch& l) {
  constexpr int64_t kEach = 256 / ROWS * (16 / sizeof(T)) * 4;
  const int64_t parts = ROWS > 1 ? 1 : (l.m + kEach - 1) / kEach;
  const unsigned across = static_cast<unsigned>(parts < 1024 ? parts : 1024);
  each_slice(l.n, ROWS, 256 * static_cast<int64_t>(across), [&](int64_t first, int64_t count) {
    const auto kernel = l.h ? log_probs_grad_kernel<T, ROWS, true> : log_probs_grad_kernel<T, ROWS, false>;
    kernel<<<dim3(static_cast<unsigned>((count + ROWS - 1) / ROWS), across), 256, 0, l.stream>>>(
        static_cast<const T*>(l.S) + first * l.lds, static_cast<T*>(l.D) + first * l.ldd,
        args_of<T>(l, first, count));
  });
}

template <class T>
hipError_t log_probs_grad(LogProbsGradLaunch l) {
  constexpr int64_t V = 16 / sizeof(T);
  if (!l.stats) {
    const bool aligned = reinterpret_cast<uintptr_t>(l.S) % 16 == 0 && (l.n == 1 || l.lds % V == 0);
    const auto holds = [&](int vectors) {
      return l.m <= whole_most<T>(vectors) || (aligned && l.m <= vectors * V);
    };
    if (holds(64)) return start_whole<T, 1, 1>(l), hipGetLastError();
    if (holds(64 * 4)) return start_whole<T, 1, 4>(l), hipGetLastError();
    if (holds(256 * 4)) return start_whole<T, 4, 4>(l), hipGetLastError();
    if (holds(256 * 8)) return start_whole<T, 4, 8>(l), hipGetLastError();
    if (holds(1024 * 4)) return start_whole<T, 16, 4>(l), hipGetLastError();
    // (4096 columns of 65536 bfloat16: 231 us, with the statistics in a launch
    // of their own 302; but a few columns leave most of the device idle.)
    if (l.n >= kTwiceColumns) return start_twice<T>(l), hipGetLastError();
    LogProbsLaunch s = {};
    s.data = l.data;
    s.m = l.m;
    s.n = l.n;
    s.S = l.S;
    s.lds = l.lds;
    s.labels = l.labels;
    s.inv_t = l.inv_t;
    s.stats = static_cast<float*>(l.work);
    s.work = static_cast<char*>(l.work) + (3 * l.n * sizeof(float) + 15) / 16 * 16;
    s.stream = l.stream;
    l.stats = s.stats;
    const hipError_t e = launch_log_probs(s);
    if (e != hipSuccess) return e;
  }
  if (l.m <= 64 * V * 4) start_grad<T, 4>(l);
  else start_grad<T, 1>(l);
  return hipGetLastError();
}

}  // namespace

size_t log_probs_work_bytes(int, int64_t m, int64_t n, int top) {
  const LogProbsPlan plan = plan_log_probs(m, n);
  if (plan.parts == 1) return 0;
  return (static_cast<size_t>(n) * plan.parts * sizeof(Mass) + 15) / 16 * 16 +
         static_cast<size_t>(n) * plan.parts * top * sizeof(u64);
}

hipError_t launch_log_probs(const LogProbsLaunch& l) {
  switch (l.data) {
    case SDCA_F32: return log_probs<float>(l);
    case SDCA_F16: return log_probs<__half>(l);
    default: return log_probs<__hip_bfloat16>(l);
  }
}

size_t log_probs_grad_work_bytes(int data, int64_t m, int64_t n, bool stats) {
  if (stats || n >= kTwiceColumns || m <= (data == SDCA_F32 ? whole_most<float>() : whole_most<__half>())) return 0;
  return (3 * static_cast<size_t>(n) * sizeof(float) + 15) / 16 * 16 + log_probs_work_bytes(data, m, n, 0);
}

hipError_t launch_log_probs_grad(const LogProbsGradLaunch& l) {
  switch (l.data) {
    case SDCA_F32: return log_probs_grad<float>(l);
    case SDCA_F16: return log_probs_grad<__half>(l);
    default: return log_probs_grad<__hip_bfloat16>(l);
  }
}

}  // namespace sdca_gpu
