// Scores from shared 8-bit weights with a low-rank adapter for each example:
// S_i = sx_i sw (q(X_i) W') + T_i B_a', T_i = scale_a X_i A_a', a = index_i.
//
// The product is the 8-bit one (scores_i8.hpp); the adapter's part is added
// to a score in 32 bits where it leaves the registers, so that S is written
// once and rounded once.  T comes from a kernel before (adapters.hip).
#include "scores_i8.hpp"

namespace sdca_gpu {
namespace {

// The adapters' part of 16 examples by 16 FM classes: 16 x 16 x 4 products in
// 32 bits, classes by rank times rank by examples, whose layout is that of
// the integer product's sums.  Examples of different adapters take turns: for
// each adapter among the 16 the products are made for all, and each example
// keeps those of its own, so that one adapter's infinities reach no other
// example.
template <class T>
struct Adapted {
  static constexpr bool some = true;
  const float* terms;
  int pitch;
  const int64_t* index;
  const T* B;
  int64_t apart;  // from one adapter's B to the next one's
  int rank, count;
  const int* order;  // or NULL

  Adapted from(int64_t n0, int64_t m0) const {
    Adapted a = *this;
    if (order) {
      a.order += n0;
    } else {
      a.terms += n0 * pitch;
      a.index += n0;
    }
    a.B += m0 * rank;
    return a;
  }
  int64_t first_row(int64_t n0) const { return order ? 0 : n0; }
  __device__ int64_t row(int64_t i) const { return order ? order[i] : i; }

  template <int FM, int Q>
  __device__ inline void operator()(v4f (&more)[FM], int64_t row0, int64_t n, int first, int m,
                                    int lane) const {
#pragma unroll
    for (int i = 0; i < FM; ++i) more[i] = v4f{0.f, 0.f, 0.f, 0.f};
    const int64_t i = row0 + (lane & 15), at_row = row(i < n ? i : n - 1);
    const int64_t given = i < n ? index[at_row] : -1;
    const bool bad = given < -1 || given >= count;
    const int mine = bad ? -1 : static_cast<int>(given);
    const float* t = terms + at_row * pitch;
    int64_t at[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int c = first + ((lane & 15) >> 2) * (4 * Q) + (lane & 3) + i / Q * 16 * Q + i % Q * 4;
      at[i] = static_cast<int64_t>(min(c, m - 1)) * rank;
    }
    unsigned long long left = __ballot(mine >= 0);
    while (left) {
      const int a = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
      const bool hit = mine == a;
      left &= ~__ballot(hit);
      const T* b = B + a * apart;
      v4f sum[FM] = {};
      for (int k0 = 0; k0 < rank; k0 += 4) {
        const int k = k0 + lane / 16;
        const float tk = t[k];  // (zeros behind the rank)
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          const float bk = k < rank ? to_float(b[at[i] + k]) : 0.f;
          sum[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(bk, tk, sum[i], 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) more[i][e] = hit ? sum[i][e] : more[i][e];
    }
    if (bad) {
#pragma unroll
      for (int i = 0; i < FM; ++i) more[i] = v4f{NAN, NAN, NAN, NAN};
    }
  }

  __device__ inline float one(int example, int c, int lane) const {
    const int64_t a = index[example];
    if (a == -1) return 0.f;
    if (a < 0 || a >= count) return NAN;
    const float* t = terms + example * pitch;
    const T* b = B + a * apart + static_cast<int64_t>(c) * rank;
    float sum = 0.f;
    for (int k = lane; k < rank; k += 64) sum = fmaf(t[k], to_float(b[k]), sum);
    return wave_total(sum);
  }
};

template <class T, class Out>
hipError_t scores(const ScoresI8Launch& a, const Adapters& ad, const float* terms,
                  const int* order) {
  const Adapted<T> extra = {terms, static_cast<int>(terms_pitch(ad.rank)), ad.index,
                            static_cast<const T*>(ad.B), a.m * ad.rank, static_cast<int>(ad.rank),
                            static_cast<int>(ad.count), order};
  if (a.data == SDCA_I8) start_tiles<Out>(a, extra);
  else if (scores_i8_few(a.n, a.d)) start_few<T, Out>(a, extra);
  else start_strip<T, Out>(a, extra);
  return hipGetLastError();
}
template <class T>
hipError_t scores(const ScoresI8Launch& a, const Adapters& ad, const float* terms,
                  const int* order) {
  switch (a.out) {
    case SDCA_F32: return scores<T, float>(a, ad, terms, order);
    case SDCA_F16: return scores<T, __half>(a, ad, terms, order);
    default: return scores<T, __hip_bfloat16>(a, ad, terms, order);
  }
}

}  // namespace

hipError_t launch_scores_adapted(const ScoresI8Launch& a, const Adapters& ad, const float* terms,
                                 const int* order) {
  switch (ad.data) {
    case SDCA_F32: return scores<float>(a, ad, terms, order);
    case SDCA_F16: return scores<__half>(a, ad, terms, order);
    default: return scores<__hip_bfloat16>(a, ad, terms, order);
  }
}

}  // namespace sdca_gpu
