// Host-side launch interface of the kernels that answer from a trained model
// (internal): the 8-bit quantiser, the 8-bit score product, the draw of a
// label from scores, and labels' log-probabilities with their gradient.
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

// Alternatives of a column at most: a wave's sorted list has one to a lane.
constexpr int64_t kMostTop = 64;

struct LogProbsLaunch {
  int data;  // SDCA_F32, F16, BF16
  int64_t m, n;
  const void* S;
  int64_t lds;
  const int64_t* labels;
  float inv_t;
  int top;
  // Results, each or NULL: n, n, 3 n, top n, top n values.
  float *logp, *entropy, *stats, *top_logp;
  int64_t* top_index;
  void* work;  // log_probs_work_bytes of device memory
  hipStream_t stream;
};
size_t log_probs_work_bytes(int data, int64_t m, int64_t n, int top);
hipError_t launch_log_probs(const LogProbsLaunch& a);

struct LogProbsGradLaunch {
  int data;  // SDCA_F32, F16, BF16
  int64_t m, n;
  const void* S;
  int64_t lds;
  const int64_t* labels;
  const float *g, *h;  // n; h or NULL
  const float* stats;  // 3 n, or NULL
  float inv_t;
  void* D;  // S's type; may be S
  int64_t ldd;
  float* logp;  // n, or NULL
  void* work;   // log_probs_grad_work_bytes of device memory
  hipStream_t stream;
};
size_t log_probs_grad_work_bytes(int data, int64_t m, int64_t n, bool stats);
hipError_t launch_log_probs_grad(const LogProbsGradLaunch& a);

// Low-rank adapters: matrices of an example's adapter a = index[i], in the
// examples' type.  -1: none; another index outside [0, count): NaN scores.
struct Adapters {
  int data;  // SDCA_F32, F16, BF16
  int64_t count, rank;
  const void* A;  // count x rank rows of d values
  const void* B;  // count x m rows of `rank` values
  const int64_t* index;
  PerColumn<float> scale;
};
constexpr int64_t kMostRank = 128, kMostAdapters = 65535;
// Rows of terms: rank values of an example, zeros up to whole 16.
constexpr int64_t terms_pitch(int64_t rank) { return (rank + 15) / 16 * 16; }

// terms[i] = scale_a X_i A_a' for the n rows of X (`wide` values of type
// `data`, pitch ldx) with A_a's `rank` rows of `wide` values, adapters
// count apart; rows without an adapter have none written.
struct TermsLaunch {
  int data;
  int64_t wide, n;
  const void* X;
  int64_t ldx;
  const Adapters* adapters;
  const void* A;
  // The rows in the order of their adapters and each adapter's place and
  // number in it, as launch_group leaves them: terms (and Q) are then in that
  // order.  NULL: as they come.
  const int* order;
  const int2* spans;
  float* terms;
  // 1, or with Q terms_parts(n): the wide axis in so many parts, for which
  // `terms` has room n rows apart; the terms are the first part's in the end.
  int parts;
  // NULL, or the rows in 8 bits besides, as launch_quantize gives them with
  // ldq = pad.
  int8_t* Q;
  int64_t pad;
  float* scales;
  hipStream_t stream;
};
// Whether an example has workgroups of its own, or 16 and more share one: then
// the adapters' order is worth finding first.  (us with and without, order and
// product included, m = d = 4096, fp16: rank 16, 8 adapters, n = 1024: 46, 56;
// 2048: 68, 75; 3000: 101, 98; rank 32, 4 adapters, 1024: 52, 58; 2048: 79, 79;
// rank 64, 512: 50, 50; 1024: 81, 66.)
constexpr bool terms_by_rows(int64_t n, int64_t rank) { return n * terms_pitch(rank) <= 32768; }
int terms_parts(int64_t n, int64_t rank);
hipError_t launch_terms(const TermsLaunch& a);

// The n rows in the order of their adapters, rising for each, those without
// one last (`order`, n), each adapter's first place and number of rows
// (`spans`, count + 1: the last is of the rows without), and, or NULL, the
// rows' adapters in that order (`ids`, n: -1 without, -2 where the index is
// none of [-1, count)).
hipError_t launch_group(const Adapters& adapters, int64_t n, int* order, int2* spans, int* ids,
                        hipStream_t stream);

// launch_scores_i8 with adapters: terms are the examples' (of X_i itself, not
// of its 8-bit form).  With an order, 8-bit example i of X, its terms and
// ids[i] are those of row order[i] of S.
hipError_t launch_scores_adapted(const ScoresI8Launch& a, const Adapters& adapters,
                                 const float* terms, const int* order, const int* ids);

struct AdaptedGradLaunch {
  int grad;  // G's type
  int64_t d, m, n;
  const void* G;
  int64_t ldg;
  const void* X;
  int64_t ldx;
  Adapters adapters;
  float *dA, *dB;
  void* work;  // adapted_grad_work_bytes of device memory
  hipStream_t stream;
};
size_t adapted_grad_work_bytes(int grad, int data, int64_t d, int64_t m, int64_t n, int64_t count, int64_t rank);
hipError_t launch_adapted_grad(const AdaptedGradLaunch& a);

}  // namespace sdca_gpu

#endif  // SDCA_HIP_ANSWER_LAUNCH_HPP
