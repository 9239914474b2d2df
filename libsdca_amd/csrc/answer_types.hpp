// Loads and conversions of the element types the answering kernels take.
#ifndef SDCA_HIP_ANSWER_TYPES_HPP
#define SDCA_HIP_ANSWER_TYPES_HPP

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sdca_gpu {

__device__ inline float to_float(float x) { return x; }
__device__ inline float to_float(double x) { return static_cast<float>(x); }
__device__ inline float to_float(__half x) { return __half2float(x); }
__device__ inline float to_float(__hip_bfloat16 x) {
  unsigned short b;
  __builtin_memcpy(&b, &x, 2);
  return __uint_as_float(static_cast<unsigned>(b) << 16);
}

// Values at .. at + V - 1 of a row of `len` as floats, 0 beyond its end.
// The row may start at any multiple of its element: the copy below becomes
// wide loads, which the device takes at any address.
template <int V, class T>
__device__ inline void load_vec(const T* row, int64_t at, int64_t len, float (&v)[V],
                                float beyond = 0.f) {
  if (at + V <= len) {
    T raw[V];
    __builtin_memcpy(raw, row + at, sizeof(raw));
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = to_float(raw[e]);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = at + e < len ? to_float(row[at + e]) : beyond;
  }
}

// Eight values of a column of d for its quantiser: those from `at` on, or the
// last eight where the column ends before at + 8: one load whatever d (20011
// columns of 513 half-precision values 12 us, with a load for each value of
// the end 13.5).
template <class T>
__device__ inline void load_column(const T* x, int64_t at, int64_t d, T (&raw)[8]) {
  if (d >= 8) {
    __builtin_memcpy(raw, x + (at + 8 <= d ? at : d - 8), sizeof(raw));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) raw[e] = at + e < d ? x[at + e] : T(0.f);
  }
}

// The bytes that load_column's values at `at` were quantised to, from `at` on,
// zeros from d on.
__device__ inline void end_column(int64_t at, int64_t d, unsigned (&w)[2]) {
  if (d < 8 || at + 8 <= d) return;
  const int64_t more = at + 8 - d;  // bytes of values before `at`, or beyond d
  uint64_t b;
  __builtin_memcpy(&b, w, 8);
  b = more < 8 ? b >> (8 * more) : 0;
  __builtin_memcpy(w, &b, 8);
}

// |x| as an integer: the order of the bit patterns is that of the values,
// with infinity and the NaNs on top, so one integer maximum finds both the
// largest magnitude and a non-finite value.
__device__ inline unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The scale of a column of that largest magnitude: max |x| (1 / 127).  A
// column of zeros (or of values whose scale is no 32-bit number above zero)
// gets 0 and zeros; one that holds an infinity or a NaN gets NaN and zeros,
// so that every product with it is NaN.
struct ColumnScale {
  float scale;
  bool some;  // whether any value is not quantised to zero
  __device__ explicit ColumnScale(unsigned most) {
    const bool finite = most < 0x7f800000u;
    scale = finite ? __uint_as_float(most) * (1.f / 127.f) : __uint_as_float(0x7fc00000u);
    some = finite && scale > 0.f;
  }
};

// Eight values x / scale to the nearest integers, as bytes: the quotient is
// rounded to 32 bits first, and halves go to even.
//
// x r with r = 1 / scale is within two units (2^-16 below 128) of that
// quotient, and both have the same nearest integer unless one is that near
// to a half: only then, once in some 10^4 values, are the quotients taken.
// The integer comes from adding 1.5 2^23, which leaves it in the low bits.
__device__ inline void quantize8(const float (&v)[8], const ColumnScale& s, unsigned (&w)[2]) {
  w[0] = w[1] = 0;
  if (!s.some) return;
  const float r = 1.f / s.scale;
  unsigned b[8];
  float far = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float q = v[e] * r, shifted = q + 12582912.f;
    b[e] = __float_as_uint(shifted);
    far = fmaxf(far, fabsf(q - (shifted - 12582912.f)));
  }
  // (Below 2^-100 the reciprocal is no ordinary number, and the scale may
  // have lost digits itself: quotients, and a clamp.)
  if (far > 0.4999f || !(s.scale >= 7.9e-31f)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = rintf(v[e] / s.scale);
      b[e] = static_cast<unsigned>(static_cast<int>(fminf(fmaxf(q, -127.f), 127.f)));
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const unsigned low = __builtin_amdgcn_perm(b[4 * h + 1], b[4 * h], 0x0c0c0400);
    const unsigned high = __builtin_amdgcn_perm(b[4 * h + 3], b[4 * h + 2], 0x04000c0c);
    w[h] = low | high;
  }
}

// Rounds to the output's type, to nearest, halves to even.
template <class T> __device__ inline T from_float(float x);
template <> __device__ inline float from_float<float>(float x) { return x; }
template <> __device__ inline __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ inline __hip_bfloat16 from_float<__hip_bfloat16>(float x) {
  return __float2bfloat16(x);
}

}  // namespace sdca_gpu

#endif  // SDCA_HIP_ANSWER_TYPES_HPP
