// Order, exchanges and sorts of the kernels that answer from scores: integers
// in the order of scores, and a wave's values sorted by its lanes.
#ifndef SDCA_HIP_ANSWER_WAVE_HPP
#define SDCA_HIP_ANSWER_WAVE_HPP

#include <hip/hip_runtime.h>

#include "common.hpp"

namespace sdca_gpu {

typedef unsigned long long u64;

// Order-preserving integer of a score; -0 and 0 are one value.
__device__ inline unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ inline float score_of(unsigned key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}
// Falling scores, ties by rising index, as falling integers (0: no label).
__device__ inline u64 entry_of(float l, int index) {
  return (static_cast<u64>(key_of(l)) << 32) | (0xffffffffu - static_cast<unsigned>(index));
}
__device__ inline int index_of(u64 entry) {
  return static_cast<int>(0xffffffffu - static_cast<unsigned>(entry));
}

// ---------------------------------------------------------------------------
// Waves: 64-bit exchanges, scans and sorts.
// ---------------------------------------------------------------------------
template <int CTRL, int RM>
__device__ inline u64 dpp64(u64 v) {
  const unsigned lo = dpp_bits<CTRL, RM, false>(static_cast<int>(v));
  const unsigned hi = dpp_bits<CTRL, RM, false>(static_cast<int>(v >> 32));
  return (static_cast<u64>(hi) << 32) | lo;
}
// Inclusive sum over the lanes before: rows of 16 by shifts, then the last
// lanes of rows 0 and 2 into 1 and 3, and of the first half into the second.
__device__ inline u64 wave_scan(u64 v) {
  v += dpp64<0x111, 0xF>(v);
  v += dpp64<0x112, 0xF>(v);
  v += dpp64<0x114, 0xF>(v);
  v += dpp64<0x118, 0xF>(v);
  v += dpp64<0x142, 0xA>(v);
  v += dpp64<0x143, 0xC>(v);
  return v;
}
__device__ inline int wave_scan(int v) {
  v += dpp_bits<0x111, 0xF, false>(v);
  v += dpp_bits<0x112, 0xF, false>(v);
  v += dpp_bits<0x114, 0xF, false>(v);
  v += dpp_bits<0x118, 0xF, false>(v);
  v += dpp_bits<0x142, 0xA, false>(v);
  v += dpp_bits<0x143, 0xC, false>(v);
  return v;
}
__device__ inline u64 read_lane64(u64 v, int l) {
  const unsigned lo = __builtin_amdgcn_readlane(static_cast<int>(v), l);
  const unsigned hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), l);
  return (static_cast<u64>(hi) << 32) | lo;
}
__device__ inline u64 wave_sum(u64 v) { return read_lane64(wave_scan(v), 63); }
__device__ inline int wave_sum(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

template <int OFF, bool VALU>
__device__ inline u64 xor_lane64(u64 v) {
  const unsigned lo = xor_lane<OFF, VALU>(static_cast<int>(v));
  const unsigned hi = xor_lane<OFF, VALU>(static_cast<int>(v >> 32));
  return (static_cast<u64>(hi) << 32) | lo;
}
template <int OFF, bool VALU>
__device__ inline u64 other(u64 v) { return xor_lane64<OFF, VALU>(v); }
template <int OFF, bool VALU>
__device__ inline float other(float v) { return xor_lane<OFF, VALU>(v); }

template <bool VALU>
__device__ inline float wave_max(float v) {
  v = fmaxf(v, other<1, VALU>(v));
  v = fmaxf(v, other<2, VALU>(v));
  v = fmaxf(v, other<4, VALU>(v));
  v = fmaxf(v, other<8, VALU>(v));
  v = fmaxf(v, other<16, VALU>(v));
  return fmaxf(v, other<32, VALU>(v));
}

// One step of a bitonic sort: the lane keeps the larger or the smaller of
// its value and lane ^ STRIDE's.
template <int STRIDE, bool VALU, class K>
__device__ inline K sort_step(K v, bool falling) {
  const K o = other<STRIDE, VALU>(v);
  const bool larger = ((threadIdx.x & STRIDE) == 0) == falling;
  return (o > v) == larger ? o : v;
}
template <int STRIDE, bool VALU, class K>
__device__ inline K sort_merge(K v, bool falling) {
  if constexpr (STRIDE >= 32) v = sort_step<32, VALU>(v, falling);
  if constexpr (STRIDE >= 16) v = sort_step<16, VALU>(v, falling);
  if constexpr (STRIDE >= 8) v = sort_step<8, VALU>(v, falling);
  if constexpr (STRIDE >= 4) v = sort_step<4, VALU>(v, falling);
  if constexpr (STRIDE >= 2) v = sort_step<2, VALU>(v, falling);
  return sort_step<1, VALU>(v, falling);
}
// The wave's 64 values by lane, falling or rising.
template <bool VALU, class K>
__device__ inline K sort_wave(K v, bool falling) {
  v = sort_merge<1, VALU>(v, (threadIdx.x & 2) == 0);
  v = sort_merge<2, VALU>(v, (threadIdx.x & 4) == 0);
  v = sort_merge<4, VALU>(v, (threadIdx.x & 8) == 0);
  v = sort_merge<8, VALU>(v, (threadIdx.x & 16) == 0);
  v = sort_merge<16, VALU>(v, (threadIdx.x & 32) == 0);
  return sort_merge<32, VALU>(v, falling);
}

// 64 R values, the i-th in lane i % 64's v[i / 64], falling: within each
// register as above, and between registers without an exchange.
template <int SIZE, int STRIDE, int R, class K>
__device__ inline void sort_registers(K (&v)[R]) {
  if constexpr (STRIDE > 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r & STRIDE) continue;
      const K a = v[r], b = v[r + STRIDE];
      const bool swap = (b > a) == ((r & SIZE) == 0);
      v[r] = swap ? b : a;
      v[r + STRIDE] = swap ? a : b;
    }
    sort_registers<SIZE, STRIDE / 2>(v);
  }
}
template <bool VALU, int SIZE, int R, class K>
__device__ inline void merge_registers(K (&v)[R]) {
  if constexpr (SIZE <= R) {
    sort_registers<SIZE, SIZE / 2>(v);
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = sort_merge<32, VALU>(v[r], (r & SIZE) == 0);
    merge_registers<VALU, SIZE * 2>(v);
  }
}
template <bool VALU, int R, class K>
__device__ inline void sort_wave(K (&v)[R]) {
#pragma unroll
  for (int r = 0; r < R; ++r) v[r] = sort_wave<VALU>(v[r], (r & 1) == 0);
  merge_registers<VALU, 2>(v);
}

}  // namespace sdca_gpu

#endif  // SDCA_HIP_ANSWER_WAVE_HPP
