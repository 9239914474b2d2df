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
// over threads nor on the order of atomics, and they are exact where sums of
// 32-bit floats would lose the tail's small weights.
#include "answer_launch.hpp"
#include "answer_types.hpp"

namespace sdca_gpu {
namespace {

typedef unsigned long long u64;

constexpr int kBlock = 1024;
constexpr int kWaves = kBlock / 64;
constexpr int kVec = 4;
constexpr int kBins = 2048;

// A NaN counts as a label that cannot be drawn; -0 and 0 are one value.
__device__ inline float score(float x) { return x == x ? x + 0.f : -INFINITY; }

// Order-preserving integer of a score.
__device__ inline unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ inline float score_of(unsigned key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

struct Weights {
  float max, inv_t, scale;
  __device__ float of(float l) const { return l == max ? 1.f : expf((l - max) * inv_t); }
  __device__ u64 fixed(float w) const { return static_cast<u64>(rintf(w * scale)); }
};

struct Shared {
  u64 hist[kBins];
  u64 wave[kWaves], wave2[kWaves], wave3[kWaves];
  u64 found_above;
  int found_bin;
};

__device__ inline u64 shfl_up64(u64 v, int d) {
  const unsigned lo = __shfl_up(static_cast<unsigned>(v), d);
  const unsigned hi = __shfl_up(static_cast<unsigned>(v >> 32), d);
  return (static_cast<u64>(hi) << 32) | lo;
}
__device__ inline u64 shfl_xor64(u64 v, int d) {
  const unsigned lo = __shfl_xor(static_cast<unsigned>(v), d);
  const unsigned hi = __shfl_xor(static_cast<unsigned>(v >> 32), d);
  return (static_cast<u64>(hi) << 32) | lo;
}
__device__ inline u64 wave_scan(u64 v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u64 o = shfl_up64(v, d);
    if (lane >= d) v += o;
  }
  return v;
}
__device__ inline u64 wave_sum(u64 v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += shfl_xor64(v, d);
  return v;
}
__device__ inline u64 block_sum(u64 v, u64* part) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 s = 0;
  for (int w = 0; w < kWaves; ++w) s += part[w];
  return s;
}

// f(score, index) over the row's entries from `begin` on, a stride of
// `threads` lanes.
template <class T, class F>
__device__ inline void each(const T* row, int64_t begin, int64_t end, int t, int threads, F f) {
  for (int64_t at = begin + int64_t(t) * kVec; at < end; at += int64_t(threads) * kVec) {
    float v[kVec];
    load_vec<kVec>(row, at, end, v);
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      if (at + e < end) f(score(v[e]), at + e);
  }
}

// The key at which the running sum over falling keys, from `floor_key` up,
// first reaches `target` (counts, or with MASS fixed weights), and the sum
// above it: three digits of the key, a histogram each.
template <bool MASS, class T>
__device__ void descend(const T* row, int64_t m, const Weights& wt, unsigned floor_key, u64 target,
                        Shared& s, unsigned* tau, u64* above) {
  unsigned prefix = 0;
  u64 sum = 0;
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
    const int bits = level == 2 ? 10 : 11;
    const int bins = 1 << bits;
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kBlock) s.hist[i] = 0;
    if (threadIdx.x == 0) {
      s.found_bin = 0;
      s.found_above = sum;
    }
    __syncthreads();
    each(row, 0, m, threadIdx.x, kBlock, [&](float l, int64_t) {
      const unsigned key = key_of(l);
      if (key < floor_key || (level && (key >> (shift + bits)) != prefix)) return;
      const u64 add = MASS ? wt.fixed(wt.of(l)) : 1;
      if (add) atomicAdd(&s.hist[(key >> shift) & (bins - 1)], add);
    });
    __syncthreads();
    const int hi = bins - 1 - 2 * static_cast<int>(threadIdx.x);
    const u64 a = hi >= 1 ? s.hist[hi] : 0, b = hi >= 1 ? s.hist[hi - 1] : 0;
    u64 incl = wave_scan(a + b);
    if ((threadIdx.x & 63) == 63) s.wave[threadIdx.x >> 6] = incl;
    __syncthreads();
    for (int w = 0; w < static_cast<int>(threadIdx.x >> 6); ++w) incl += s.wave[w];
    const u64 before = sum + incl - a - b;
    if (before < target && before + a + b >= target) {
      const bool first = before + a >= target;
      s.found_bin = first ? hi : hi - 1;
      s.found_above = first ? before : before + a;
    }
    __syncthreads();
    prefix = (prefix << bits) | static_cast<unsigned>(s.found_bin);
    sum = s.found_above;
  }
  *tau = prefix;
  *above = sum;
}

template <class T>
__device__ inline T setting(const PerColumn<T>& c, int64_t col) {
  return c.each ? c.each[col] : c.value;
}

struct SampleArgs {
  int64_t m, lds;
  const float* u;
  PerColumn<float> temperature, top_p, min_p;
  PerColumn<int64_t> top_k;
  int64_t* labels;
  float* prob;
  int64_t* kept;
  float scale;
};

// A column per workgroup, read from memory on every pass.
template <class T>
__global__ __launch_bounds__(kBlock) void sample_column_kernel(const T* __restrict__ S,
                                                               SampleArgs a) {
  __shared__ Shared s;
  const int64_t col = blockIdx.x, m = a.m;
  const T* row = S + col * a.lds;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;

  u64 best = 0;  // (key, falling index) of the first maximum
  each(row, 0, m, threadIdx.x, kBlock, [&](float l, int64_t i) {
    const u64 c = (static_cast<u64>(key_of(l)) << 32) | (0xffffffffu - static_cast<unsigned>(i));
    best = c > best ? c : best;
  });
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const u64 o = shfl_xor64(best, d);
    best = o > best ? o : best;
  }
  if (lane == 0) s.wave[wave] = best;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) best = s.wave[w] > best ? s.wave[w] : best;

  const float T_ = setting(a.temperature, col);
  Weights wt;
  wt.max = score_of(static_cast<unsigned>(best >> 32));
  const bool greedy = !(T_ >= 1.17549435e-38f), none = wt.max == -INFINITY;
  if (greedy || none) {
    if (threadIdx.x == 0) {
      a.labels[col] = none ? -1 : static_cast<int64_t>(0xffffffffu - static_cast<unsigned>(best));
      if (a.prob) a.prob[col] = none ? 0.f : 1.f;
      if (a.kept) a.kept[col] = none ? 0 : 1;
    }
    return;
  }
  wt.inv_t = 1.f / fminf(T_, 3.402823466e38f);
  wt.scale = a.scale;
  const float p = setting(a.top_p, col);
  float q = setting(a.min_p, col);
  q = q > 0.f ? fminf(q, 1.f) : 0.f;
  const int64_t k = setting(a.top_k, col);

  unsigned tau = 0;
  u64 ties = 0;  // labels at tau that are kept
  if (k > 0 && k < m) {
    u64 above;
    descend<false>(row, m, wt, 0, static_cast<u64>(k), s, &tau, &above);
    ties = k - above;
  }
  if (p < 1.f) {
    u64 mass = 0;
    each(row, 0, m, threadIdx.x, kBlock, [&](float l, int64_t) {
      if (key_of(l) > tau) mass += wt.fixed(wt.of(l));
    });
    mass = block_sum(mass, s.wave2);
    if (ties) mass += ties * wt.fixed(wt.of(score_of(tau)));
    // The shortest beginning with a sum of at least p mass, and of at least
    // one label.
    u64 target = static_cast<u64>(ceil(static_cast<double>(p) * static_cast<double>(mass)));
    target = p > 0.f ? target : 1;
    target = target < 1 ? 1 : target > mass ? mass : target;
    unsigned cut;
    u64 above;
    descend<true>(row, m, wt, tau, target, s, &cut, &above);
    const u64 w = wt.fixed(wt.of(score_of(cut)));
    u64 need = w ? (target - above + w - 1) / w : 1;
    if (cut == tau && ties && need > ties) need = ties;
    tau = cut;
    ties = need;
  }

  // The draw.  The row is narrowed to the stretch that holds the label, a
  // sixteenth at a time; the first narrowing also gives the total.
  const float w_tau = ties ? wt.of(score_of(tau)) : 0.f;
  const u64 f_tau = w_tau >= q ? wt.fixed(w_tau) : 0;
  int64_t begin = 0, end = m;
  u64 total = 0, target = 0, tie_base = 0, mass_base = 0;
  while (true) {
    const int64_t part = ((end - begin + kWaves - 1) / kWaves + 63) / 64 * 64;
    const int64_t b = begin + wave * part, e = b + part < end ? b + part : end;
    u64 n_tie = 0, mass = 0, many = 0;
    if (b < e)
      each(row, b, e, lane, 64, [&](float l, int64_t) {
        const unsigned key = key_of(l);
        const float w = wt.of(l);
        if (key > tau && w >= q && w > 0.f) {
          mass += wt.fixed(w);
          ++many;
        }
        n_tie += ties && key == tau;
      });
    n_tie = wave_sum(n_tie);
    mass = wave_sum(mass);
    many = wave_sum(many);
    __syncthreads();
    if (lane == 0) {
      s.wave[wave] = n_tie;
      s.wave2[wave] = mass;
      s.wave3[wave] = many;
    }
    __syncthreads();
    if (begin == 0 && end == m && total == 0) {
      u64 all = 0, tied = 0, count = 0;
      for (int w = 0; w < kWaves; ++w) {
        all += s.wave2[w];
        tied += s.wave[w];
        count += s.wave3[w];
      }
      tied = tied < ties ? tied : ties;
      total = all + tied * f_tau;
      count += w_tau >= q && w_tau > 0.f ? tied : 0;
      float u = a.u[col];
      u = u > 0.f ? (u < 1.f ? u : 0.99999994f) : 0.f;
      target = static_cast<u64>(static_cast<double>(u) * static_cast<double>(total));
      target = target < total ? target : total - 1;
      if (threadIdx.x == 0 && a.kept) a.kept[col] = static_cast<int64_t>(count);
    }
    int64_t pick = begin;
    for (int w = 0; w < kWaves; ++w) {
      const u64 left = ties > tie_base ? ties - tie_base : 0;
      const u64 t = s.wave[w] < left ? s.wave[w] : left;
      const u64 here = s.wave2[w] + t * f_tau;
      if (mass_base + here > target) break;
      mass_base += here;
      tie_base += s.wave[w];
      pick += part;
    }
    begin = pick;
    end = pick + part < end ? pick + part : end;
    if (part == 64) break;
  }
  if (wave == 0) {
    const bool in = begin + lane < end;
    const float l = in ? score(to_float(row[begin + lane])) : -INFINITY;
    const unsigned key = key_of(l);
    const float w = wt.of(l);
    const bool tied = in && ties && key == tau;
    const u64 ranked = wave_scan(tied ? 1 : 0) + tie_base;
    const bool keep = in && w >= q && (key > tau || (tied && ranked <= ties));
    const u64 sum = wave_scan(keep ? wt.fixed(w) : 0) + mass_base;
    const u64 passed = __ballot(sum > target);
    if (passed && lane == __ffsll(passed) - 1) {
      a.labels[col] = begin + lane;
      if (a.prob)
        a.prob[col] = static_cast<float>(static_cast<double>(w) * wt.scale / static_cast<double>(total));
    }
  }
}

template <class T>
hipError_t sample(const SampleLaunch& l) {
  SampleArgs a;
  a.m = l.m;
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
  a.scale = static_cast<float>(u64(1) << (62 - bits < 46 ? 62 - bits : 46));
  sample_column_kernel<T><<<static_cast<unsigned>(l.n), kBlock, 0, l.stream>>>(
      static_cast<const T*>(l.S), a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_sample(const SampleLaunch& a) {
  switch (a.data) {
    case SDCA_F32: return sample<float>(a);
    case SDCA_F64: return sample<double>(a);
    case SDCA_F16: return sample<__half>(a);
    default: return sample<__hip_bfloat16>(a);
  }
}

}  // namespace sdca_gpu
