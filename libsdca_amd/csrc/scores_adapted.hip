// Scores from shared 8-bit weights with a low-rank adapter for each example:
// S_i = sx_i sw (q(X_i) W') + T_i B_a', T_i = scale_a X_i A_a', a = index_i.
//
// The product is the 8-bit one (scores_i8.hpp); the adapter's part is added
// to a score in 32 bits where it leaves the registers, so that S is written
// once and rounded once.  T comes from a kernel before (adapters.hip).
#include "scores_i8.hpp"

namespace sdca_gpu {
namespace {

// Sixteen ranks of the terms (rows of 32-bit floats) and of B as the operands
// of 16 x 16 products.  A lane has its example's, or its class's, part.
//
// 32 bits: four products of 16 x 16 x 4; lane group g holds ranks 4 g on.
template <class T>
struct Ranks {
  static constexpr unsigned kInfinite = 0;  // (no parts)
  static constexpr int kEach = 4;
  static __device__ int from(int lane) { return lane / 16 * 4; }
  float v[4];
  static constexpr float back = 1.f;
  __device__ void take(const float* t, int lane) { __builtin_memcpy(v, t + from(lane), 16); }
  __device__ v4f times(const T (&b)[4]) const {
    v4f sum = {};
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(b[e], v[e], sum, 0, 0, 0);
    return sum;
  }
};

// Two 32-bit floats' first digits as 16-bit ones, in a word, and what is left
// of them.  Cut off rather than rounded: a part beyond its term would be an
// infinity where the term is the largest, and would cost the instruction's sum,
// which cuts as well, a digit.
__device__ inline unsigned cut(__half, float& x, float& y) {
  const auto both = __builtin_amdgcn_cvt_pkrtz(x, y);
  x = fmaf(static_cast<float>(both[0]), -1.f, x);
  y = fmaf(static_cast<float>(both[1]), -1.f, y);
  return __builtin_bit_cast(unsigned, both);
}
__device__ inline unsigned cut(__hip_bfloat16, float& x, float& y) {
  const unsigned u = __float_as_uint(x), v = __float_as_uint(y);
  x -= __uint_as_float(u & 0xffff0000u);
  y -= __uint_as_float(v & 0xffff0000u);
  return __builtin_amdgcn_perm(v, u, 0x07060302);
}

// 16 bits: a term is the sum of three parts, which hold its 24 digits, eight and
// more at a time.  Products of 16 x 16 x 32 take the first 16 of their 32 places
// for one part and the others for the next, with B's ranks in both: lane groups
// 0 and 1 hold ranks 0 to 7 and 8 to 15, groups 2 and 3 again.
//
// Halves have few exponents: the 16 ranks are brought to below 2^14 first, so
// that the parts of the largest are ordinary numbers (what is below 2^-24 then,
// 2^-37 of the largest, is lost), and their products back (by the power of two
// `back`, itself at least 2^-126).  (Two halves, in one instruction, held 23
// digits and took as long: 1024 x 14336, rank 32, 95 us and 94.)
template <class T>
struct RanksInParts {
  static constexpr bool kHalf = std::is_same<T, __half>::value;
  static constexpr unsigned kInfinite = kHalf ? 0x7c00 : 0x7f80;
  static constexpr int kEach = 8;
  static __device__ int from(int lane) { return lane / 16 % 2 * 8; }
  unsigned first[4], last[4];
  float back = 1.f;

  __device__ void take(const float* t, int lane) {
    float v[8], most = 0.f;
    __builtin_memcpy(v, t + from(lane), 32);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
    if constexpr (kHalf) {
      most = fmaxf(most, __shfl_xor(most, 16));
      // (Beside an infinite term the largest finite one must not become another.)
      const int down = max((most < INFINITY ? __builtin_amdgcn_frexp_expf(most) : 128) - 14, -126);
      back = __builtin_amdgcn_ldexpf(1.f, down);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __builtin_amdgcn_ldexpf(v[e], -down);
    }
    if (__ballot(most == INFINITY)) split<true>(v, lane);
    else split<false>(v, lane);
    // (Made here: the compiler would keep the terms and split them at each use.)
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(first[i]), "+v"(last[i]));
  }
  // An infinity is its first part alone.
  template <bool INFINITE>
  __device__ void split(const float (&v)[8], int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = v[2 * i], y = v[2 * i + 1];
      const unsigned one = cut(T(), x, y);
      if (INFINITE && fabsf(v[2 * i]) == INFINITY) x = 0.f;
      if (INFINITE && fabsf(v[2 * i + 1]) == INFINITY) y = 0.f;
      const unsigned two = cut(T(), x, y), three = cut(T(), x, y);
      first[i] = lane < 32 ? one : two;
      last[i] = lane < 32 ? three : 0;
    }
  }
  __device__ v4f times(const T (&b)[8]) const {
    return multiply_16<T>(b, first, multiply_16<T>(b, last, v4f{}));
  }
};
template <>
struct Ranks<__half> : RanksInParts<__half> {};
template <>
struct Ranks<__hip_bfloat16> : RanksInParts<__hip_bfloat16> {};

// The adapters that 16 FN examples have, one after the other, and -1.
template <int FN>
struct Turns {
  unsigned long long left[FN];
  __device__ explicit Turns(const int (&mine)[FN]) {
#pragma unroll
    for (int j = 0; j < FN; ++j) left[j] = __ballot(mine[j] >= 0);
  }
  __device__ int next(const int (&mine)[FN]) {
    int a = -1;
#pragma unroll
    for (int j = FN - 1; j >= 0; --j)
      if (left[j]) a = __builtin_amdgcn_readlane(mine[j], __builtin_ctzll(left[j]));
#pragma unroll
    for (int j = 0; j < FN; ++j) left[j] &= ~__ballot(mine[j] == a);
    return a;
  }
};

// The adapters' part of a wave's scores: products of classes by ranks with
// ranks by examples, whose layout is that of the integer product's sums.
// Examples of different adapters take turns: for each adapter the products
// are made for 16 examples at a time, and each example keeps those of its
// own, so that one adapter's infinities reach no other example.  B is loaded
// for some adapters at once: with an adapter for each example the loads'
// latency is what this takes.
//
// A term's parts can be 0 where the term is not, and times an infinity of B
// that is NaN: where a wave's B holds one, its products are left out, and made
// from the terms themselves at the end.
template <class T>
struct Adapted {
  static constexpr bool some = true;
  const float* terms;
  int pitch;
  const int64_t* index;
  const T* B;
  int64_t apart;  // from one adapter's B to the next one's
  int rank, count;
  const int *order, *ids;  // or NULL

  Adapted from(int64_t n0, int64_t m0) const {
    Adapted a = *this;
    a.terms += n0 * pitch;
    if (order) {
      a.order += n0;
      a.ids += n0;
    } else {
      a.index += n0;
    }
    a.B += m0 * rank;
    return a;
  }
  int64_t first_row(int64_t n0) const { return order ? 0 : n0; }
  __device__ int64_t row(int64_t i) const { return order ? order[i] : i; }
  // -1: none, -2: no adapter's number
  __device__ static int adapter(int64_t a, int count) {
    return a >= -1 && a < count ? static_cast<int>(a) : -2;
  }

  // Where a lane's examples and classes are.
  template <int FM, int FN>
  struct Place {
    int mine[FN];       // its examples' adapters, -1: none
    int row[FN];        // of terms
    bool bad[FN];       // no adapter's number
    int64_t at[FM];
  };
  template <int FM, int FN, int Q>
  __device__ inline void find(Place<FM, FN>& place, int64_t row0, int64_t n, int first, int m, int lane) const {
    int of[FN];
    auto& [mine, row, bad, at] = place;
    // (Without conditions, for the loads to be on their way together.)
    if (ids) {
#pragma unroll
      for (int j = 0; j < FN; ++j) of[j] = ids[min(row0 + j * 16 + (lane & 15), n - 1)];
    } else {
      int64_t given[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) given[j] = index[min(row0 + j * 16 + (lane & 15), n - 1)];
#pragma unroll
      for (int j = 0; j < FN; ++j) of[j] = adapter(given[j], count);
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int64_t i = row0 + j * 16 + (lane & 15);
      const int given = i < n ? of[j] : -1;
      bad[j] = given < -1;
      mine[j] = max(given, -1);
      row[j] = static_cast<int>(i < n ? i : n - 1);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int c = first + ((lane & 15) >> 2) * (4 * Q) + (lane & 3) + i / Q * 16 * Q + i % Q * 4;
      at[i] = static_cast<int64_t>(min(c, m - 1)) * rank;
    }
  }

  template <int FM, int FN, int Q>
  __device__ inline void add(v4f (&scores)[FM][FN], int64_t row0, int64_t n, int first, int m,
                             int lane) const {
    using R = Ranks<T>;
    constexpr int kOnce = FM > 2 ? 1 : FN > 2 ? 2 : 4;
    Place<FM, FN> place;
    find<FM, FN, Q>(place, row0, n, first, m, lane);
    auto& [mine, row, bad, at] = place;
    bool again = false;
    // Terms of 64 examples at most in registers, and B for each such part of the
    // examples.  (128 do not fit beside the scores: 1024 x 14336 halves, rank 32, 99
    // us, so 95.)
    constexpr int kExamples = FN > 4 ? FN / 2 : FN;
#pragma unroll
    for (int j0 = 0; j0 < FN; j0 += kExamples) {
      for (int k0 = 0; k0 < rank; k0 += 16) {
        int these[kExamples];
#pragma unroll
        for (int j = 0; j < kExamples; ++j) these[j] = mine[j0 + j];
        Turns<kExamples> turns(these);
        R terms_of[kExamples];
#pragma unroll
        for (int j = 0; j < kExamples; ++j)
          terms_of[j].take(terms + static_cast<int64_t>(row[j0 + j]) * pitch + k0, lane);
        const int k = k0 + R::from(lane);
        int a[kOnce];
        a[0] = turns.next(these);
        while (a[0] >= 0) {
          T b[kOnce][FM][R::kEach];
#pragma unroll
          for (int q = 0; q < kOnce; ++q) {
            if (q) a[q] = turns.next(these);
            const T* from = B + (a[q] < 0 ? a[0] : a[q]) * apart;
#pragma unroll
            for (int i = 0; i < FM; ++i) load(from + at[i], k0, k, b[q][i]);
          }
#pragma unroll
          for (int q = 0; q < kOnce; ++q) {
            if (a[q] < 0) break;
            // (No branch: the products need not wait for this.)
            const bool out = R::kInfinite != 0 && __ballot(infinite(b[q], R::kInfinite));
            again |= out;
#pragma unroll
            for (int j = 0; j < kExamples; ++j) {
              const bool hit = these[j] == a[q];
              if (!__ballot(hit)) continue;
#pragma unroll
              for (int i = 0; i < FM; ++i) {
                const v4f sum = terms_of[j].times(b[q][i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float more = fmaf(sum[e], terms_of[j].back, scores[i][j0 + j][e]);
                  scores[i][j0 + j][e] = hit && !out ? more : scores[i][j0 + j][e];
                }
              }
            }
          }
          a[0] = turns.next(these);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) scores[i][j][e] = bad[j] ? NAN : scores[i][j][e];
    if constexpr (R::kInfinite != 0) {
      if (again) add_whole<FM, FN, Q>(scores, row0, n, first, m, lane);
    }
  }

  // A lane's ranks of a class, from k of the 16 that begin at k0.
  template <int EACH>
  __device__ inline void load(const T* row, int k0, int k, T (&b)[EACH]) const {
    if (k0 + 16 <= rank) {
      __builtin_memcpy(b, row + k, sizeof(b));
    } else {
#pragma unroll
      for (int e = 0; e < EACH; ++e) b[e] = k + e < rank ? row[k + e] : from_float<T>(0.f);
    }
  }

  // Whether one of these is an infinity or NaN: by the largest of their bits.
  template <class Some>
  __device__ static inline bool infinite(const Some& b, unsigned limit) {
    typedef unsigned short v2u __attribute__((ext_vector_type(2)));
    unsigned w[sizeof(b) / 4];
    __builtin_memcpy(w, &b, sizeof(w));
    v2u most = {};
#pragma unroll
    for (unsigned word : w) {
      const unsigned size = word & 0x7fff7fffu;
      v2u two;
      __builtin_memcpy(&two, &size, 4);
      most = __builtin_elementwise_max(most, two);
    }
    return max(static_cast<unsigned>(most[0]), static_cast<unsigned>(most[1])) >= limit;
  }

  // The products that were left out, in 32 bits.
  template <int FM, int FN, int Q>
  __device__ inline void add_whole(v4f (&scores)[FM][FN], int64_t row0, int64_t n, int first, int m, int lane) const {
    using Whole = Ranks<float>;
    // (Found again, so that nothing is kept for this.)
    asm volatile("" : "+v"(lane));
    Place<FM, FN> place;
    find<FM, FN, Q>(place, row0, n, first, m, lane);
    auto& [mine, row, bad, at] = place;
    for (int k0 = 0; k0 < rank; k0 += 16) {
      Turns<FN> turns(mine);
      for (int a = turns.next(mine); a >= 0; a = turns.next(mine)) {
        const T* from = B + a * apart;
        T b[FM][Ranks<T>::kEach];
#pragma unroll
        for (int i = 0; i < FM; ++i) load(from + at[i], k0, k0 + Ranks<T>::from(lane), b[i]);
        if (!__ballot(infinite(b, Ranks<T>::kInfinite))) continue;
        float whole[FM][Whole::kEach];
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          T some[Whole::kEach];
          load(from + at[i], k0, k0 + Whole::from(lane), some);
#pragma unroll
          for (int e = 0; e < Whole::kEach; ++e) whole[i][e] = to_float(some[e]);
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const bool hit = mine[j] == a;
          if (!__ballot(hit)) continue;
          Whole terms_of;
          terms_of.take(terms + static_cast<int64_t>(row[j]) * pitch + k0, lane);
#pragma unroll
          for (int i = 0; i < FM; ++i) {
            const v4f sum = terms_of.times(whole[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) scores[i][j][e] = hit ? scores[i][j][e] + sum[e] : scores[i][j][e];
          }
        }
      }
    }
  }

  __device__ inline float one(int example, int c, int lane) const {
    const int a = adapter(index[example], count);
    if (a < 0) return a == -1 ? 0.f : NAN;
    const float* t = terms + example * pitch;
    const T* b = B + a * apart + static_cast<int64_t>(c) * rank;
    float sum = 0.f;
    for (int k = lane; k < rank; k += 64) sum = fmaf(t[k], to_float(b[k]), sum);
    return wave_total(sum);
  }
};

template <class T, class Out>
hipError_t scores(const ScoresI8Launch& a, const Adapters& ad, const float* terms,
                  const int* order, const int* ids) {
  const Adapted<T> extra = {terms, static_cast<int>(terms_pitch(ad.rank)), ad.index,
                            static_cast<const T*>(ad.B), a.m * ad.rank, static_cast<int>(ad.rank),
                            static_cast<int>(ad.count), order, ids};
  if (a.data == SDCA_I8) start_tiles<Out>(a, extra);
  else if (scores_i8_few(a.n, a.d)) start_few<T, Out>(a, extra);
  else start_strip<T, Out>(a, extra);
  return hipGetLastError();
}
template <class T>
hipError_t scores(const ScoresI8Launch& a, const Adapters& ad, const float* terms,
                  const int* order, const int* ids) {
  switch (a.out) {
    case SDCA_F32: return scores<T, float>(a, ad, terms, order, ids);
    case SDCA_F16: return scores<T, __half>(a, ad, terms, order, ids);
    default: return scores<T, __hip_bfloat16>(a, ad, terms, order, ids);
  }
}

}  // namespace

hipError_t launch_scores_adapted(const ScoresI8Launch& a, const Adapters& ad, const float* terms,
                                 const int* order, const int* ids) {
  switch (ad.data) {
    case SDCA_F32: return scores<float>(a, ad, terms, order, ids);
    case SDCA_F16: return scores<__half>(a, ad, terms, order, ids);
    default: return scores<__hip_bfloat16>(a, ad, terms, order, ids);
  }
}

}  // namespace sdca_gpu
