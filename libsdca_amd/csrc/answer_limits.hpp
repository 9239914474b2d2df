// Limits that the answering kernels' launches keep to (host code alone, so
// that it can be checked without a device).
#ifndef SDCA_HIP_ANSWER_LIMITS_HPP
#define SDCA_HIP_ANSWER_LIMITS_HPP

#include <stdint.h>

namespace sdca_gpu {

// A dispatch counts its work-items in 32 bits: of a grid of 2^32 threads or
// more only the remainder runs, without an error (268435461 columns, 16 to a
// workgroup of 256: the first 16 were done).  Half of that is as good as all
// of it: such a launch takes milliseconds.
constexpr int64_t kDispatchThreads = int64_t(1) << 31;

// f(first, count) for slices that make up [0, n) in their order, each of no
// more than one dispatch takes at `threads` threads for `per` of them.
template <class F>
void each_slice(int64_t n, int64_t per, int64_t threads, F f) {
  const int64_t most = kDispatchThreads / threads * per;
  for (int64_t first = 0; first < n; first += most)
    f(first, n - first < most ? n - first : most);
}

}  // namespace sdca_gpu

#endif  // SDCA_HIP_ANSWER_LIMITS_HPP
