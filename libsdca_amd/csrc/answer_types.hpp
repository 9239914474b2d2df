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

// Rounds to the output's type, to nearest, halves to even.
template <class T> __device__ inline T from_float(float x);
template <> __device__ inline float from_float<float>(float x) { return x; }
template <> __device__ inline __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ inline __hip_bfloat16 from_float<__hip_bfloat16>(float x) {
  return __float2bfloat16(x);
}

}  // namespace sdca_gpu

#endif  // SDCA_HIP_ANSWER_TYPES_HPP
