// Host-side launch interface of the kernels that answer from a trained model
// (internal): the 8-bit quantiser, the 8-bit score product and the draw of a
// label from scores.
#ifndef SDCA_HIP_ANSWER_LAUNCH_HPP
#define SDCA_HIP_ANSWER_LAUNCH_HPP

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/sdca_hip.h"

namespace sdca_gpu {

// Columns x (d values, leading dimension ldx) to int8 q and scale s.  q's
// rows are written up to `pad` values, zeros from d on.
struct QuantLaunch {
  int data;  // SDCA_F32, F64, F16, BF16
  int64_t d, n;
  const void* X;
  int64_t ldx;
  int8_t* Q;
  int64_t ldq, pad;
  float* scales;
  hipStream_t stream;
};
hipError_t launch_quantize(const QuantLaunch& a);

// The int8 rows of src again with pitch ldq, zeros from d up to pad.
hipError_t launch_repack_i8(const int8_t* src, int64_t ld, int64_t d, int64_t n, int8_t* dst,
                            int64_t ldq, int64_t pad, hipStream_t stream);

// K bytes of one staged tile row; the tile kernels read X in whole ones.
constexpr int64_t kI8TileK = 128;

// S_ij = (sum_k X_ik W_jk) sx_i sw_j.
struct ScoresI8Launch {
  int data;  // X's type: SDCA_I8, or where scores_i8_quantises holds any of the quantiser's
  int out;   // SDCA_F32, F16, BF16
  int64_t d, m, n;
  // n rows, pitch ldx.  Int8 rows have zeros from d up to a multiple of
  // kI8TileK and 16-byte addresses, but where scores_i8_quantises holds.
  const void* X;
  int64_t ldx;
  const float* sx;
  const int8_t* W;  // m rows, pitch ldw
  int64_t ldw;
  const float* sw;
  void* S;
  int64_t lds;
  hipStream_t stream;
};
// Whether X is taken as the caller has it, quantised on the way.
bool scores_i8_quantises(int data, int64_t d, int64_t m, int64_t n);
hipError_t launch_scores_i8(const ScoresI8Launch& a);

// One setting of the draw: a value for all columns, or one per column.
template <class T>
struct PerColumn {
  T value;
  const T* each;  // device, or NULL
};

// Labels of a column at most.  Weights are added up in units of 2^-shift with
// m 2^shift <= 2^62, and each is off by half a unit at most, so a sum is off by
// m 2^-(shift + 1): here 2^-17 of the largest weight, which is less than the
// weights' own rounding can make of it.  The error grows with the square of m
// (2^-7 at 2^28 labels).
constexpr int64_t kSampleMostLabels = int64_t(1) << 23;

struct SampleLaunch {
  int data;  // SDCA_F32, F64, F16, BF16
  int64_t m, n;
  const void* S;
  int64_t lds;
  const float* u;
  PerColumn<float> temperature, top_p, min_p;
  PerColumn<int64_t> top_k;
  int64_t* labels;
  float* prob;    // or NULL
  int64_t* kept;  // or NULL
  void* work;     // sample_work_bytes of device memory
  hipStream_t stream;
};
size_t sample_work_bytes(int64_t m, int64_t n);
hipError_t launch_sample(const SampleLaunch& a);

}  // namespace sdca_gpu

#endif  // SDCA_HIP_ANSWER_LAUNCH_HPP
