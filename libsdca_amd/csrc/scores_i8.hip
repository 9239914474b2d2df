// Scores by a product in 8-bit integers: S_ij = (sum_k X_ik W_jk) sx_i sw_j.
//
// The sums are exact in 32-bit integers (the entry point bounds d), so they
// do not hang on the order of the terms; each score is rounded three times
// in 32 bits (the sum, and the two scales' products) and once to the
// output's type.
#include "answer_launch.hpp"
#include "answer_types.hpp"

namespace sdca_gpu {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kTileK = static_cast<int>(kI8TileK);

// An operand's rows from `row` on as a buffer: loads beyond its last byte
// give zeros.
__device__ inline __amdgpu_buffer_rsrc_t rows_buffer(const int8_t* base, int64_t ld, int64_t row,
                                                     int64_t rows, int64_t d) {
  const int64_t left = rows - row;
  int64_t bytes = left > 0 ? (left - 1) * ld + (d + 15) / 16 * 16 : 0;
  if (bytes > 0x7fffffff) bytes = 0x7fffffff;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(base + (left > 0 ? row * ld : 0)),
                                           0, static_cast<int>(bytes), 0x00020000);
}

// 16 bytes of each lane from `offset` in the buffer to LDS: lane i's go to
// dst + 16 i.  (The host pass does not know the builtin's width.)
__device__ inline void load_to_lds(__amdgpu_buffer_rsrc_t from, int8_t* dst, int offset) {
#ifdef __HIP_DEVICE_COMPILE__
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      from, (__attribute__((address_space(3))) void*)(dst), 16, offset, 0, 0, 0);
#endif
}

// A workgroup computes BN examples by BM classes; its WN x WM waves each a
// (BN / WN) x (BM / WM) part in 16 x 16 x 64 matrix instructions.  Classes
// are the instruction's rows and examples its columns, so a lane's four
// results are neighbouring scores of one example.
//
// K goes by in tiles of 128 bytes, two of them in LDS: while one is
// multiplied, the other arrives by loads that write LDS directly.  A tile
// row holds its eight 16-byte pieces in the order piece ^ (row % 8): the 16
// rows that an instruction reads at one place then lie in different banks.
template <class Out, int BN, int BM, int WN, int WM>
__global__ __launch_bounds__(64 * WN * WM) void scores_i8_kernel(
    const int8_t* __restrict__ X, int64_t ldx, const float* __restrict__ sx,
    const int8_t* __restrict__ W, int64_t ldw, const float* __restrict__ sw,
    Out* __restrict__ S, int64_t lds, int d, int m, int n) {
  constexpr int kWaves = WN * WM;
  constexpr int kRows = BN + BM;                // tile rows, the examples' first
  constexpr int kLoads = kRows / 8 / kWaves;    // of a wave: 8 rows each
  constexpr int FN = BN / WN / 16, FM = BM / WM / 16;
  static_assert(kRows % (8 * kWaves) == 0 && BN % 8 == 0, "tile rows per wave");
  __shared__ __align__(128) int8_t tile[2][kRows * kTileK];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave % WN, wm = wave / WN;
  const int64_t n0 = static_cast<int64_t>(blockIdx.y) * BN;
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * BM;
  const __amdgpu_buffer_rsrc_t xb = rows_buffer(X, ldx, n0, n, d);
  const __amdgpu_buffer_rsrc_t wb = rows_buffer(W, ldw, m0, m, d);

  int from[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = (wave * kLoads + i) * 8 + lane / 8;
    const int piece = (lane & 7) ^ (row & 7);
    from[i] = (row < BN ? row * static_cast<int>(ldx) : (row - BN) * static_cast<int>(ldw)) +
              piece * 16;
  }
  auto fetch = [&](int k, int stage) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = (wave * kLoads + i) * 8;
      load_to_lds(row < BN ? xb : wb, &tile[stage][row * kTileK], from[i] + k);
    }
  };

  v4i acc[FM][FN] = {};
  const int tiles = (d + kTileK - 1) / kTileK;
  fetch(0, 0);
  for (int t = 0; t < tiles; ++t) {
    __syncthreads();  // tile t has arrived, and tile t - 1 is no longer read
    if (t + 1 < tiles) fetch((t + 1) * kTileK, (t + 1) & 1);
    const int8_t* base = tile[t & 1];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int piece = k * 4 + lane / 16;
      v4i a[FM], b[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int row = BN + (wm * FM + i) * 16 + (lane & 15);
        a[i] = *reinterpret_cast<const v4i*>(base + row * kTileK + ((piece ^ (row & 7)) * 16));
      }
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int row = (wn * FN + j) * 16 + (lane & 15);
        b[j] = *reinterpret_cast<const v4i*>(base + row * kTileK + ((piece ^ (row & 7)) * 16));
      }
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i], b[j], acc[i][j], 0, 0, 0);
    }
  }

#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const int64_t row = n0 + (wn * FN + j) * 16 + (lane & 15);
    if (row >= n) continue;
    const float s = sx[row];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int64_t at = m0 + (wm * FM + i) * 16 + (lane / 16) * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (at + e < m)
          S[row * lds + at + e] =
              from_float<Out>(static_cast<float>(acc[i][j][e]) * s * sw[at + e]);
    }
  }
}

template <class Out>
hipError_t scores(const ScoresI8Launch& a) {
  constexpr int BN = 64, BM = 128;
  const dim3 grid(static_cast<unsigned>((a.m + BM - 1) / BM),
                  static_cast<unsigned>((a.n + BN - 1) / BN));
  scores_i8_kernel<Out, BN, BM, 2, 2><<<grid, 256, 0, a.stream>>>(
      a.X, a.ldx, a.sx, a.W, a.ldw, a.sw, static_cast<Out*>(a.S), a.lds, static_cast<int>(a.d),
      static_cast<int>(a.m), static_cast<int>(a.n));
  return hipGetLastError();
}

}  // namespace

hipError_t launch_scores_i8(const ScoresI8Launch& a) {
  switch (a.out) {
    case SDCA_F32: return scores<float>(a);
    case SDCA_F16: return scores<__half>(a);
    default: return scores<__hip_bfloat16>(a);
  }
}

}  // namespace sdca_gpu
