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

// Offsets of the 8-bit product's loads into a buffer that holds rows of an
// operand.  A row's own offset is below kI8MostOffset: a tile's 256 rows, and
// up to 32 beyond the last class, of at most kI8MaxPitch, and K up to 131071.
// A buffer has at most 2^31 - 1 bytes, so kOutside added to any row's offset
// lies beyond it, where loads give zeros.  (Unsigned: the sum may pass 2^31,
// which a signed one must not.)
constexpr int64_t kI8MaxPitch = int64_t(1) << 22;
constexpr uint32_t kI8MostOffset = 288 * kI8MaxPitch + (1 << 17);
constexpr uint32_t kOutside = 0x7fffffffu;
constexpr uint32_t i8_offset(uint32_t row, uint32_t k) { return row + k; }
static_assert(i8_offset(kI8MostOffset, kOutside) >= kOutside, "outside of any buffer");

}  // namespace sdca_gpu

#endif  // SDCA_HIP_ANSWER_LIMITS_HPP
