// Columns to 8-bit integers with one scale each.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "answer_launch.hpp"
#include "answer_limits.hpp"
#include "answer_types.hpp"

namespace sdca_gpu {
namespace {

constexpr int kVec = 8;  // values a lane takes at a time: 16 bytes of a 16-bit type, 8 of q

template <class T>
__device__ inline void load_values(const T* x, int64_t at, int64_t d, float (&v)[kVec]) {
  T raw[kVec];
  load_column(x, at, d, raw);
#pragma unroll
  for (int e = 0; e < kVec; ++e) v[e] = to_float(raw[e]);
}

// TPC threads share a column and keep it in registers (G vectors of 8 values
// each), so that it is read once; LOOP: a longer column is read twice.
template <class T, int TPC, int G, bool LOOP>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ X, int64_t ldx,
                                                       int64_t d, int64_t n,
                                                       int8_t* __restrict__ Q, int64_t ldq,
                                                       int64_t pad, float* __restrict__ scales) {
  constexpr int kColumns = 256 / TPC;
  __shared__ unsigned part[4];
  const int t = threadIdx.x % TPC;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kColumns + threadIdx.x / TPC;
  if (TPC <= 64 && col >= n) return;  // whole columns, and no barrier below
  const T* x = X + col * ldx;
  int8_t* q = Q + col * ldq;

  float v[G][kVec];
  unsigned most = 0;
  const int64_t sweeps = LOOP ? (d + int64_t(TPC) * G * kVec - 1) / (int64_t(TPC) * G * kVec) : 1;
  for (int64_t sweep = 0; sweep < sweeps; ++sweep) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      load_values(x, (sweep * G + g) * TPC * kVec + int64_t(t) * kVec, d, v[g]);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const unsigned b = magnitude(v[g][e]);
        most = b > most ? b : most;
      }
    }
  }
#pragma unroll
  for (int off = TPC < 64 ? TPC / 2 : 32; off; off >>= 1) {
    const unsigned o = __shfl_xor(most, off);
    most = o > most ? o : most;
  }
  if (TPC > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) most = part[w] > most ? part[w] : most;
  }
  const ColumnScale s(most);
  if (t == 0) scales[col] = s.scale;

  for (int64_t sweep = 0; sweep < sweeps; ++sweep) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int64_t at = (sweep * G + g) * TPC * kVec + int64_t(t) * kVec;
      if (LOOP) load_values(x, at, d, v[g]);
      if (at >= pad) continue;
      unsigned w[2];
      quantize8(v[g], s, w);
      end_column(at, d, w);
      if (at + kVec <= pad) {
        __builtin_memcpy(q + at, w, kVec);
      } else {
        for (int e = 0; at + e < pad; ++e)
          q[at + e] = static_cast<int8_t>(w[e / 4] >> (8 * (e % 4)));
      }
    }
  }
}

template <class T, int TPC, int G, bool LOOP>
void start(const QuantLaunch& a) {
  constexpr int64_t kColumns = 256 / TPC;
  each_slice(a.n, kColumns, 256, [&](int64_t first, int64_t n) {
    quantize_kernel<T, TPC, G, LOOP>
        <<<static_cast<unsigned>((n + kColumns - 1) / kColumns), 256, 0, a.stream>>>(
            static_cast<const T*>(a.X) + first * a.ldx, a.ldx, a.d, n, a.Q + first * a.ldq, a.ldq,
            a.pad, a.scales + first);
  });
}

template <class T>
hipError_t quantize(const QuantLaunch& a) {
  // By the column's length alone: part of a wave for a short column, so that
  // a wave has some KiB to read (200000 columns of 128 floats took 69 us with
  // a wave each, 21 with a quarter, both from the last-level cache; 30 from
  // memory, at 4.3 TB/s; of 512 half-precision values 81 and 51), a workgroup
  // above, with as few registers as hold it (20000 columns of 4096 floats 72 us,
  // 5.7 TB/s).  Columns beyond the registers are read twice (4000 of 40000
  // floats 273 us; 16 of 100000, which leave most of the device idle, 34).
  if (a.pad <= 16 * kVec) start<T, 16, 1, false>(a);
  else if (a.pad <= 16 * 2 * kVec) start<T, 16, 2, false>(a);
  else if (a.pad <= 16 * 4 * kVec) start<T, 16, 4, false>(a);
  else if (a.pad <= 32 * 4 * kVec) start<T, 32, 4, false>(a);
  else if (a.pad <= 256 * 2 * kVec) start<T, 256, 2, false>(a);
  else if (a.pad <= 256 * 6 * kVec) start<T, 256, 6, false>(a);
  else start<T, 256, 6, true>(a);
  return hipGetLastError();
}

__global__ __launch_bounds__(256) void repack_kernel(const int8_t* __restrict__ src, int64_t ld,
                                                     int64_t d, int8_t* __restrict__ dst,
                                                     int64_t ldq, int64_t pad, int64_t total) {
  // A lane writes 16 bytes; the source may start at any byte.
  const int64_t per = pad / 16;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / per, at = (i % per) * 16;
    int w[4] = {0, 0, 0, 0};
    const int8_t* s = src + row * ld + at;
    if (at + 16 <= d) {
      __builtin_memcpy(w, s, 16);
    } else {
      for (int e = 0; at + e < d; ++e) w[e / 4] |= (s[e] & 0xff) << (8 * (e % 4));
    }
    __builtin_memcpy(dst + row * ldq + at, w, 16);
  }
}

}  // namespace

hipError_t launch_quantize(const QuantLaunch& a) {
  switch (a.data) {
    case SDCA_F32: return quantize<float>(a);
    case SDCA_F64: return quantize<double>(a);
    case SDCA_F16: return quantize<__half>(a);
    default: return quantize<__hip_bfloat16>(a);
  }
}

hipError_t launch_repack_i8(const int8_t* src, int64_t ld, int64_t d, int64_t n, int8_t* dst,
                            int64_t ldq, int64_t pad, hipStream_t stream) {
  const int64_t total = n * (pad / 16);
  const int64_t blocks = (total + 255) / 256;
  repack_kernel<<<static_cast<unsigned>(blocks < 8192 ? blocks : 8192), 256, 0, stream>>>(
      src, ld, d, dst, ldq, pad, total);
  return hipGetLastError();
}

}  // namespace sdca_gpu
