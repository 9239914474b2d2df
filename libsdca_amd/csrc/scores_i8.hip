// Scores by a product in 8-bit integers: S_ij = (sum_k X_ik W_jk) sx_i sw_j.
//
// The sums are exact in 32-bit integers (the entry point bounds d), so they
// do not hang on the order of the terms; each score is rounded three times
// in 32 bits (the sum, and the two scales' products) and once to the
// output's type.
#include "scores_i8.hpp"

namespace sdca_gpu {
namespace {

template <class Out>
hipError_t scores(const ScoresI8Launch& a) {
  if (scores_i8_few(a.n, a.d)) {
    switch (a.data) {
      case SDCA_F32: start_few<float, Out>(a, Nothing()); break;
      case SDCA_F64: start_few<double, Out>(a, Nothing()); break;
      case SDCA_F16: start_few<__half, Out>(a, Nothing()); break;
      case SDCA_BF16: start_few<__hip_bfloat16, Out>(a, Nothing()); break;
      default: start_few<int8_t, Out>(a, Nothing());
    }
    return hipGetLastError();
  }
  switch (a.data) {
    case SDCA_F32: start_strip<float, Out>(a, Nothing()); return hipGetLastError();
    case SDCA_F64: start_strip<double, Out>(a, Nothing()); return hipGetLastError();
    case SDCA_F16: start_strip<__half, Out>(a, Nothing()); return hipGetLastError();
    case SDCA_BF16: start_strip<__hip_bfloat16, Out>(a, Nothing()); return hipGetLastError();
  }
  start_tiles<Out>(a, Nothing());
  return hipGetLastError();
}

}  // namespace

bool scores_i8_quantises(int data, int64_t d, int64_t m, int64_t n) {
  if (scores_i8_few(n, d)) return true;
  // The strip kernel reads all of W for every 32 examples, so W is to be
  // small, and one workgroup does all there is to do for them, which pays
  // while there are few rounds of workgroups.  (us with half-precision
  // examples, against the quantiser and the product one after the other,
  // without the second launch's 2 us: 20011 x 513, m 137: 19.0, 25.0; 20000 x
  // 128, m 128: 10.1, 12.3; m 256: 13.2, 14.6; 100 x 512, m 128: 6.6, 8.9; but
  // 20000 x 1024, m 256: 37, 28; 200000 x 256, m 128: 71, 60.)
  return data != SDCA_I8 && n <= 65536 && m <= 256 && d <= 1024 && m * d <= 98304;
}

hipError_t launch_scores_i8(const ScoresI8Launch& a) {
  switch (a.out) {
    case SDCA_F32: return scores<float>(a);
    case SDCA_F16: return scores<__half>(a);
    default: return scores<__hip_bfloat16>(a);
  }
}

}  // namespace sdca_gpu
