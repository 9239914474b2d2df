// The kernels of the 8-bit score product, and what they add to a score on its
// way out: nothing, or a low-rank adapter's part.
#ifndef SDCA_HIP_SCORES_I8_HPP
#define SDCA_HIP_SCORES_I8_HPP

#include <type_traits>

#include "answer_launch.hpp"
#include "answer_limits.hpp"
#include "answer_types.hpp"
#include "common.hpp"

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
__device__ inline void load_to_lds(__amdgpu_buffer_rsrc_t from, int8_t* dst, uint32_t offset) {
#ifdef __HIP_DEVICE_COMPILE__
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      from, (__attribute__((address_space(3))) void*)(dst), 16, offset, 0, 0, 0);
#endif
}

// Blocks go round the eight XCDs in turn, and each XCD has its own L2: block
// `id` takes a tile from its XCD's own eighth of the tiles, which run
// through groups of eight rows of tiles, so that the tiles an XCD works on
// together share their operands' rows.
struct TileAt {
  int n, m;
};
__device__ inline TileAt tile_of(int id, int tiles_n, int tiles_m) {
  const int total = tiles_n * tiles_m, xcd = id & 7, per = total >> 3, more = total & 7;
  const int at = xcd * per + min(xcd, more) + (id >> 3);
  constexpr int kGroup = 8;
  const int group = at / (kGroup * tiles_m);
  const int high = min(kGroup, tiles_n - group * kGroup);
  const int in = at - group * kGroup * tiles_m;
  return {group * kGroup + in % high, in / high};
}

// What is added to a wave's scores before they are rounded: add() to 16 FN
// examples by 16 FM classes in the layout of Turned's acc; one() is it for one
// example and class, from a whole wave.
// from() is the same for a slice that starts at that example and class; the
// slice's example i goes to row row(i) of S from its row first_row() on.
struct Nothing {
  static constexpr bool some = false;
  Nothing from(int64_t, int64_t) const { return {}; }
  int64_t first_row(int64_t n0) const { return n0; }
  __device__ int64_t row(int64_t i) const { return i; }
};

// A wave's scores to memory: 16 examples at a time are turned round in LDS,
// so that stores take the scores of an example in a row, 16 FM of them, at
// any address.  acc[i][j] holds four neighbouring scores of a lane's example;
// for a 16-bit type two of them (Q) take their classes in turn, four and four.
template <class Out, int FM>
struct Turned {
  static constexpr int Q = 4 / static_cast<int>(sizeof(Out));
  static constexpr int kUnit = 16 / static_cast<int>(sizeof(Out));  // scores in 16 bytes
  static constexpr int kPitch = 16 * FM + kUnit;                    // other banks for each row
  static constexpr int kAcross = 16 * FM / kUnit;                   // lanes along an example
  static constexpr int kSize = 16 * kPitch;
  static_assert(FM % Q == 0, "whole units");

  // x_scale(row) is the scale of example rows + row.
  template <int FN, class XScale, class Extra>
  static __device__ inline void store(const v4i (&acc)[FM][FN], Out* turn, XScale x_scale,
                                      const float* sw, Out* S, int64_t lds, int64_t rows,
                                      int first, int m, int64_t n, int lane, const Extra& extra) {
    const int mine = lane / 16 * kUnit;  // this lane's first score of 16 Q
    float scale[FM / Q][kUnit];
#pragma unroll
    for (int g = 0; g < FM / Q; ++g)
#pragma unroll
      for (int e = 0; e < kUnit; ++e) scale[g][e] = sw[min(first + g * 16 * Q + mine + e, m - 1)];
    const auto score = [&](int i, int j, int e, float s) {
      const int g = i / Q, at = i % Q * 4 + e;
      return static_cast<float>(acc[i][j][e]) * s * scale[g][at];
    };
    v4f more[Extra::some ? FM : 1][Extra::some ? FN : 1];
    if constexpr (Extra::some) {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const float s = x_scale(j * 16 + (lane & 15));
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) more[i][j][e] = score(i, j, e, s);
      }
      extra.template add<FM, FN, Q>(more, rows, n, first, m, lane);
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const float s = Extra::some ? 0.f : x_scale(j * 16 + (lane & 15));
#pragma unroll
      for (int g = 0; g < FM / Q; ++g) {
        Out v[kUnit];
#pragma unroll
        for (int e = 0; e < kUnit; ++e) {
          if constexpr (Extra::some) v[e] = from_float<Out>(more[g * Q + e / 4][j][e % 4]);
          else v[e] = from_float<Out>(score(g * Q + e / 4, j, e % 4, s));
        }
        __builtin_memcpy(__builtin_assume_aligned(turn + (lane & 15) * kPitch + g * 16 * Q + mine, 16),
                         v, 16);
      }
      wave_lds_sync();
#pragma unroll
      for (int r = 0; r < 16; r += 64 / kAcross) {
        const int row = r + lane / kAcross, along = lane % kAcross * kUnit;
        Out v[kUnit];
        __builtin_memcpy(v, __builtin_assume_aligned(turn + row * kPitch + along, 16), 16);
        if (rows + j * 16 + row >= n) continue;
        Out* out = S + extra.row(rows + j * 16 + row) * lds + first + along;
        if (first + along + kUnit <= m) {
          __builtin_memcpy(out, v, 16);
        } else {
#pragma unroll
          for (int e = 0; e < kUnit; ++e)
            if (first + along + e < m) out[e] = v[e];
        }
      }
      wave_lds_sync();
    }
  }
};

// A workgroup computes BN examples by BM classes; its WN x WM waves each a
// (BN / WN) x (BM / WM) part in 16 x 16 x 64 matrix instructions.  Classes
// are the instruction's rows and examples its columns, so a lane ends with
// four neighbouring scores of an example (for a 16-bit type eight: two
// instructions, Q = 2, take their classes in turn, four and four).  The wave
// turns 16 examples at a time round in LDS, so that its stores take the
// scores of an example in a row: 16 FM of them, at any address.
//
// K goes by in tiles of 128 bytes, STAGES of them in LDS.  A tile row holds its
// eight 16-byte pieces in the order piece ^ f(row): the rows that an
// instruction reads at one place then lie in different banks.  Loads write
// LDS directly, in the order of the lanes, so the lanes' addresses carry the
// permutation.  While a half tile (64 bytes) is multiplied from registers,
// the next half is read from LDS; between the halves of tile t is the one
// barrier: behind it tile t + 1 has arrived, tile t is in registers, and the
// loads of tile t + STAGES take its place.
template <class Out, class Extra, int BN, int BM, int WN, int WM, int STAGES>
__global__ __launch_bounds__(64 * WN * WM) void scores_i8_kernel(
    const int8_t* __restrict__ X, int64_t ldx, const float* __restrict__ sx,
    const int8_t* __restrict__ W, int64_t ldw, const float* __restrict__ sw,
    Out* __restrict__ S, int64_t lds, int d, int m, int n, int tiles_n, int tiles_m, Extra extra) {
  constexpr int kWaves = WN * WM;
  constexpr int kRows = BN + BM;              // tile rows, the examples' first
  constexpr int kLoads = kRows / 8 / kWaves;  // of a wave: 8 rows each
  constexpr int FN = BN / WN / 16, FM = BM / WM / 16;
  constexpr int Q = 4 / static_cast<int>(sizeof(Out));
  static_assert(kRows % (8 * kWaves) == 0 && BN % 8 == 0 && FM % Q == 0, "tile rows per wave");
  __shared__ __align__(128) int8_t tile[STAGES][kRows * kTileK];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave % WN, wm = wave / WN;
  const TileAt place = tile_of(blockIdx.x, tiles_n, tiles_m);
  const int64_t n0 = static_cast<int64_t>(place.n) * BN;
  const int64_t m0 = static_cast<int64_t>(place.m) * BM;
  const __amdgpu_buffer_rsrc_t xb = rows_buffer(X, ldx, n0, n, d);
  const __amdgpu_buffer_rsrc_t wb = rows_buffer(W, ldw, m0, m, d);

  const auto order = [](int row) {
    return row < BN || Q == 1 ? row & 7 : (row & 3) | ((row >> 3 & 1) << 2);
  };
  uint32_t from[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = (wave * kLoads + i) * 8 + lane / 8;
    const int piece = (lane & 7) ^ order(row);
    from[i] = (row < BN ? row * static_cast<int>(ldx) : (row - BN) * static_cast<int>(ldw)) +
              piece * 16;
  }
  const auto fetch = [&](uint32_t k, int stage) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = (wave * kLoads + i) * 8;
      load_to_lds(row < BN ? xb : wb, &tile[stage][row * kTileK], i8_offset(from[i], k));
    }
  };
  // The lane's first pieces in a tile; its other rows lie at fixed distances
  // (they have the same f), and those of the second half tile at ^ 64.
  const int row_a = BN + wm * (16 * FM) + ((lane & 15) >> 2) * (4 * Q) + (lane & 3);
  const int row_b = wn * (16 * FN) + (lane & 15);
  const int at_a = row_a * kTileK + ((lane / 16) ^ order(row_a)) * 16;
  const int at_b = row_b * kTileK + ((lane / 16) ^ order(row_b)) * 16;

  v4i acc[FM][FN] = {};
  v4i a[2][FM], b[2][FN];
  const auto read = [&](int stage, int h) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
      a[h][i] = *reinterpret_cast<const v4i*>(&tile[stage][(at_a ^ (h * 64)) + (i / Q * 16 * Q + i % Q * 4) * kTileK]);
#pragma unroll
    for (int j = 0; j < FN; ++j)
      b[h][j] = *reinterpret_cast<const v4i*>(&tile[stage][(at_b ^ (h * 64)) + j * 16 * kTileK]);
  };
  const auto multiply = [&](int h) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i)
        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[h][i], b[h][j], acc[i][j], 0, 0, 0);
  };

  // The wave's reads have ended and all but its last `kept` loads have
  // arrived; then the same holds for the workgroup.
  const auto meet = [](auto kept) {
    constexpr int v = decltype(kept)::value;  // vmcnt in bits 0-3 and 14-15, lgkmcnt 0 in 8-11
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((v & 15) | ((v >> 4) << 14) | (7 << 4));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr std::integral_constant<int, (STAGES - 1) * kLoads> first_in;
  constexpr std::integral_constant<int, (STAGES - 2) * kLoads> next_in;

  // Tiles beyond the last are fetched from outside the buffers, which costs
  // no memory access, and are not multiplied: a loop without cases keeps the
  // products in one stream.
  const int tiles = (d + kTileK - 1) / kTileK;
#pragma unroll
  for (int t = 0; t < STAGES; ++t) fetch(t < tiles ? static_cast<uint32_t>(t) * kTileK : kOutside, t);
  meet(first_in);
  read(0, 0);
  int stage = 0;
  for (int t = 0; t < tiles; ++t) {
    read(stage, 1);
    __builtin_amdgcn_sched_barrier(0);  // first the reads, which the products cover
    multiply(0);
    meet(next_in);
    fetch(t + STAGES < tiles ? static_cast<uint32_t>(t + STAGES) * kTileK : kOutside, stage);
    stage = stage + 1 < STAGES ? stage + 1 : 0;
    read(stage, 0);
    __builtin_amdgcn_sched_barrier(0);
    multiply(1);
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();  // no load into LDS is left, and no read of it

  using Turn = Turned<Out, FM>;
  static_assert(kWaves * Turn::kSize * sizeof(Out) <= sizeof(tile), "room to turn");
  const int64_t rows = n0 + wn * FN * 16;
  Turn::store(acc, reinterpret_cast<Out*>(&tile[0][0]) + wave * Turn::kSize,
              [&](int row) { return sx[min(rows + row, static_cast<int64_t>(n - 1))]; }, sw, S, lds,
              rows, static_cast<int>(m0) + wm * (16 * FM), m, n, lane, extra);
}

template <class Out, int BN, int BM, int WN, int WM, int STAGES, class Extra>
void start(const ScoresI8Launch& a, const Extra& extra) {
  constexpr int kThreads = 64 * WN * WM;
  each_slice(a.m, BM, kThreads, [&](int64_t m0, int64_t m) {
    const int tiles_m = static_cast<int>((m + BM - 1) / BM);
    each_slice(a.n, BN, static_cast<int64_t>(kThreads) * tiles_m, [&](int64_t n0, int64_t n) {
      const int tiles_n = static_cast<int>((n + BN - 1) / BN);
      scores_i8_kernel<Out, Extra, BN, BM, WN, WM, STAGES>
          <<<static_cast<unsigned>(tiles_n) * tiles_m, kThreads, 0, a.stream>>>(
              static_cast<const int8_t*>(a.X) + n0 * a.ldx, a.ldx, a.sx + n0, a.W + m0 * a.ldw, a.ldw,
              a.sw + m0, static_cast<Out*>(a.S) + extra.first_row(n0) * a.lds + m0, a.lds, static_cast<int>(a.d),
              static_cast<int>(m), static_cast<int>(n), tiles_n, tiles_m, extra.from(n0, m0));
    });
  });
}

// ---------------------------------------------------------------------------
// One or two examples: W goes by once, and that is what the time is.  Each
// workgroup quantises the examples itself into LDS (which saves a launch
// before it), and its waves take RW classes at a time, 16 neighbouring bytes
// of a class to a lane, with four-byte dot products.  The examples' rows in
// LDS are zero from d on, so what W holds there counts for nothing; a lane
// whose 16 bytes all lie beyond d loads none.
// ---------------------------------------------------------------------------
constexpr int kFewThreads = 256;

template <class T, class Out, class Extra, int NX, int RW>
__global__ __launch_bounds__(kFewThreads) void scores_i8_few_kernel(
    const T* __restrict__ X, int64_t ldx, const float* __restrict__ sx,
    const int8_t* __restrict__ W, int64_t ldw, const float* __restrict__ sw,
    Out* __restrict__ S, int64_t lds, int d, int m, int rows, Extra extra) {
  constexpr int kWaves = kFewThreads / 64, kChunk = 1024;
  extern __shared__ __align__(16) int8_t few_x[];
  __shared__ unsigned part[NX][kWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pad = (d + kChunk - 1) / kChunk * kChunk;
  float scale[NX];
  if constexpr (sizeof(T) == 1) {
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      const int8_t* x = reinterpret_cast<const int8_t*>(X) + i * ldx;
      for (int at = threadIdx.x * 16; at < pad; at += kFewThreads * 16) {
        int w[4] = {0, 0, 0, 0};
        if (at + 16 <= d) {
          __builtin_memcpy(w, x + at, 16);
        } else {
          for (int e = 0; at + e < d; ++e) w[e / 4] |= (x[at + e] & 0xff) << (8 * (e % 4));
        }
        __builtin_memcpy(few_x + i * pad + at, w, 16);
      }
      scale[i] = sx[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      unsigned most = 0;
      for (int at = threadIdx.x * 8; at < d; at += kFewThreads * 8) {
        float v[8];
        load_vec<8>(X + i * ldx, at, d, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = max(most, magnitude(v[e]));
      }
#pragma unroll
      for (int off = 32; off; off >>= 1) most = max(most, static_cast<unsigned>(__shfl_xor(most, off)));
      if (lane == 0) part[i][wave] = most;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      unsigned most = part[i][0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) most = max(most, part[i][w]);
      const ColumnScale s(most);
      scale[i] = s.scale;
      for (int at = threadIdx.x * 8; at < pad; at += kFewThreads * 8) {
        float v[8];
        load_vec<8>(X + i * ldx, at, d, v);
        unsigned w[2];
        quantize8(v, s, w);
        __builtin_memcpy(few_x + i * pad + at, w, 8);
      }
    }
  }
  __syncthreads();

  const int first = blockIdx.x * rows, last = min(m, first + rows);
  for (int r0 = first + wave * RW; r0 < last; r0 += kWaves * RW) {
    const int8_t* row[RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) row[r] = W + min(r0 + r, m - 1) * ldw + lane * 16;
    int acc[RW][NX] = {};
#pragma unroll 4
    for (int at = 0; at < pad; at += kChunk) {
      if (at + lane * 16 >= d) break;
      v4i w[RW];
#pragma unroll
      for (int r = 0; r < RW; ++r) w[r] = *reinterpret_cast<const v4i*>(row[r] + at);
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const v4i x = *reinterpret_cast<const v4i*>(few_x + i * pad + at + lane * 16);
#pragma unroll
        for (int r = 0; r < RW; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r][i] = __builtin_amdgcn_sdot4(w[r][e], x[e], acc[r][i], false);
      }
    }
#pragma unroll
    for (int r = 0; r < RW; ++r)
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const int sum = wave_total(acc[r][i]);
        float more = 0.f;
        if constexpr (Extra::some) more = extra.one(i, min(r0 + r, m - 1), lane);
        if (lane == 0 && r0 + r < last) {
          float score = static_cast<float>(sum) * scale[i] * sw[r0 + r];
          if constexpr (Extra::some) score += more;
          S[i * lds + r0 + r] = from_float<Out>(score);
        }
      }
  }
}

template <class T, class Out, int NX, int RW, class Extra>
void start_few(const ScoresI8Launch& a, const Extra& extra) {
  // About a thousand workgroups: four to a compute unit, which keeps enough
  // loads in flight, and no more than that quantise the examples.
  const int step = kFewThreads / 64 * RW;
  const int64_t share = (a.m + 1023) / 1024;
  const int rows = static_cast<int>((share + step - 1) / step * step);
  const size_t bytes = static_cast<size_t>(NX) * ((a.d + 1023) / 1024 * 1024);
  scores_i8_few_kernel<T, Out, Extra, NX, RW>
      <<<static_cast<unsigned>((a.m + rows - 1) / rows), kFewThreads, bytes, a.stream>>>(
          static_cast<const T*>(a.X), a.ldx, a.sx, a.W, a.ldw, a.sw, static_cast<Out*>(a.S), a.lds,
          static_cast<int>(a.d), static_cast<int>(a.m), rows, extra);
}
template <class T, class Out, class Extra>
void start_few(const ScoresI8Launch& a, const Extra& extra) {
  // Four classes to a wave share the reads of the examples; where that
  // leaves compute units without a workgroup, one class each.
  if (a.m >= 8192) a.n == 1 ? start_few<T, Out, 1, 4>(a, extra) : start_few<T, Out, 2, 4>(a, extra);
  else a.n == 1 ? start_few<T, Out, 1, 1>(a, extra) : start_few<T, Out, 2, 1>(a, extra);
}

// ---------------------------------------------------------------------------
// Few classes: a workgroup takes 32 examples with all the classes.  It
// quantises the examples into LDS, so their 8-bit form never goes to memory
// and there is one launch; then each wave takes 32 classes at a time, whose
// bytes go from W (which stays in the caches) to registers without a barrier,
// the next four steps of K while these four are multiplied.  The examples'
// rows in LDS are zero from d on, and 16 bytes longer than whole steps, so
// that the rows an instruction reads at one place lie in different banks.
// ---------------------------------------------------------------------------
constexpr int kStrip = 32, kStripStep = 64, kStripWaves = 8;

__device__ inline v4i load_buffer(__amdgpu_buffer_rsrc_t from, uint32_t offset) {
  return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(from, offset, 0, 0));
}

__host__ __device__ inline int strip_pitch(int d) {
  return (d + kStripStep - 1) / kStripStep * kStripStep + 16;
}

// G: vectors of eight values that a lane holds of an example.
template <class T, class Out, class Extra, int G>
__global__ __launch_bounds__(64 * kStripWaves, Extra::some ? 4 : 6) void scores_i8_strip_kernel(
    const T* __restrict__ X, int64_t ldx, const int8_t* __restrict__ W, int64_t ldw,
    const float* __restrict__ sw, Out* __restrict__ S, int64_t lds, int d, int m, int n, Extra extra) {
  constexpr int Q = 4 / static_cast<int>(sizeof(Out));
  constexpr int FM = 2, FN = kStrip / 16, kAhead = 2;
  constexpr int kMine = kStrip / kStripWaves;        // a wave's examples,
  constexpr int kOnce = (sizeof(T) == 8 ? 2 : 4) / G;  // so many at once
  static_assert(kMine % kOnce == 0, "whole rounds");
  extern __shared__ __align__(16) int8_t strip[];
  __shared__ __align__(16) Out turned[kStripWaves][Turned<Out, FM>::kSize];
  __shared__ float scales[kStrip];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kStrip;
  const int pitch = strip_pitch(d), steps = (d + kStripStep - 1) / kStripStep;
  const __amdgpu_buffer_rsrc_t wb = rows_buffer(W, ldw, 0, m, d);

  uint32_t from[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int row = ((lane & 15) >> 2) * (4 * Q) + (lane & 3) + i / Q * 16 * Q + i % Q * 4;
    from[i] = row * static_cast<int>(ldw) + lane / 16 * 16;
  }
  v4i next[kAhead][FM];
  const auto fetch = [&](int class0, int step0) {
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
#pragma unroll
      for (int i = 0; i < FM; ++i)
        next[s][i] = load_buffer(
            wb, class0 < m && step0 + s < steps
                    ? i8_offset(from[i], static_cast<uint32_t>(class0 * static_cast<int>(ldw) +
                                                               (step0 + s) * kStripStep))
                    : kOutside);
  };
#pragma unroll
  for (int r0 = 0; r0 < kMine; r0 += kOnce) {
    T raw[kOnce][G][8];
    unsigned most[kOnce] = {};
#pragma unroll
    for (int r = 0; r < kOnce; ++r) {
      const int64_t row = n0 + wave * kMine + r0 + r;
      const T* x = X + (row < n ? row : n - 1) * ldx;
#pragma unroll
      for (int g = 0; g < G; ++g) load_column(x, (g * 64 + lane) * 8, d, raw[r][g]);
    }
#pragma unroll
    for (int r = 0; r < kOnce; ++r)
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) most[r] = max(most[r], magnitude(to_float(raw[r][g][e])));
#pragma unroll
    for (int off = 32; off; off >>= 1)
#pragma unroll
      for (int r = 0; r < kOnce; ++r)
        most[r] = max(most[r], static_cast<unsigned>(__shfl_xor(most[r], off)));
#pragma unroll
    for (int r = 0; r < kOnce; ++r) {
      const ColumnScale s(most[r]);
      const int at_row = wave * kMine + r0 + r;
      if (lane == 0) scales[at_row] = s.scale;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int at = (g * 64 + lane) * 8;
        // Converted again: held as floats since the maximum they spill.
        unsigned words[2 * sizeof(T)];
        __builtin_memcpy(words, raw[r][g], sizeof(words));
#pragma unroll
        for (unsigned& word : words) asm volatile("" : "+v"(word));
        __builtin_memcpy(raw[r][g], words, sizeof(words));
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = to_float(raw[r][g][e]);
        unsigned w[2];
        quantize8(v, s, w);
        end_column(at, d, w);
        if (at < steps * kStripStep) __builtin_memcpy(strip + at_row * pitch + at, w, 8);
      }
    }
  }
  fetch(wave * 16 * FM, 0);
  __syncthreads();

  const int8_t* mine = strip + (lane & 15) * pitch + lane / 16 * 16;
  for (int class0 = wave * 16 * FM; class0 < m; class0 += kStripWaves * 16 * FM) {
    v4i acc[FM][FN] = {};
    for (int step0 = 0; step0 < steps; step0 += kAhead) {
      v4i a[kAhead][FM];
#pragma unroll
      for (int s = 0; s < kAhead; ++s)
#pragma unroll
        for (int i = 0; i < FM; ++i) a[s][i] = next[s][i];
      const bool more = step0 + kAhead < steps;
      fetch(more ? class0 : class0 + kStripWaves * 16 * FM, more ? step0 + kAhead : 0);
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        if (step0 + s >= steps) break;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const v4i b = *reinterpret_cast<const v4i*>(mine + j * 16 * pitch + (step0 + s) * kStripStep);
#pragma unroll
          for (int i = 0; i < FM; ++i)
            acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[s][i], b, acc[i][j], 0, 0, 0);
        }
      }
    }
    Turned<Out, FM>::store(acc, turned[wave], [&](int row) { return scales[row]; }, sw, S, lds, n0,
                           class0, m, n, lane, extra);
  }
}

template <class T, class Out, int G, class Extra>
void start_strip(const ScoresI8Launch& a, const Extra& extra) {
  scores_i8_strip_kernel<T, Out, Extra, G>
      <<<static_cast<unsigned>((a.n + kStrip - 1) / kStrip), 64 * kStripWaves,
         kStrip * static_cast<size_t>(strip_pitch(static_cast<int>(a.d))), a.stream>>>(
          static_cast<const T*>(a.X), a.ldx, a.W, a.ldw, a.sw, static_cast<Out*>(a.S), a.lds,
          static_cast<int>(a.d), static_cast<int>(a.m), static_cast<int>(a.n), extra);
}
template <class T, class Out, class Extra>
void start_strip(const ScoresI8Launch& a, const Extra& extra) {
  if (a.d <= 512) start_strip<T, Out, 1>(a, extra);
  else start_strip<T, Out, 2>(a, extra);
}

// What a tile kernel takes for `tiles` of its tiles, in its time per tile of
// K with one tile and with two tiles to a compute unit (256 of them).
inline double tile_time(int64_t tiles, double one, double two) {
  const int64_t rest = tiles % 512;
  return static_cast<double>(tiles / 512) * two + (rest == 0 ? 0. : rest <= 256 ? one : two);
}

// The tile by its measured microseconds per 128 bytes of K: 256 x 256 does
// the most work per byte read, smaller ones fill the device with fewer
// scores.  (us by tile 256, 128, 64: 16384 x 8192, d 8192: 880, 1030, 1620;
// 1024 x 14336, d 4096: 63, 70, 109; 20000 x 1000, d 4096: 118, 98, 145; 2048
// x 2048, d 2048: 31, 15.6, 19; 512 x 4096, d 4096: 50, 23, 17; 128 x 8192,
// d 4096: 48, 24, 11.5.)
struct TilePlan {
  double us;
  int tile;
};
inline TilePlan plan_tiles(int64_t n, int64_t m, int64_t d) {
  const auto tiles = [&](int64_t t) { return ((n + t - 1) / t) * ((m + t - 1) / t); };
  const double steps = static_cast<double>((d + kTileK - 1) / kTileK);
  const double t256 = steps * tile_time(2 * tiles(256), 1.76, 1.76);
  const double t128 = steps * tile_time(tiles(128), 0.65, 1.07);
  const double t64 = steps * tile_time(tiles(64), 0.33, 0.43);
  if (t256 <= t128 && t256 <= t64) return {t256, 256};
  return t128 <= t64 ? TilePlan{t128, 128} : TilePlan{t64, 64};
}


template <class Out, class Extra>
void start_tile(const ScoresI8Launch& a, const Extra& extra, int tile) {
  if (tile == 256) start<Out, 256, 256, 2, 4, 2>(a, extra);
  else if (tile == 128) start<Out, 128, 128, 2, 4, 2>(a, extra);
  else start<Out, 64, 64, 2, 2, 4>(a, extra);
}

// Tiles of 256 come in rounds of 256, one to a compute unit.  What the last
// whole round leaves of the examples goes to a launch of its own where that,
// by the tile that suits it, takes less than another round: kSecond us are
// the launch's own, with its first loads and last stores.  (us in one launch
// and in two: 17000 x 1024, d 8192: 161, 128; 16640 x 1000, d 4096: 88, 76;
// 200000 x 256, d 4096: 270, 245; 9000 x 8192, d 8192: 521, 503; but 20000 x
// 1000, d 2048: 59, 63.)
constexpr double kSecond = 6.5;
template <class Out, class Extra>
void start_tiles(const ScoresI8Launch& a, const Extra& extra) {
  const TilePlan all = plan_tiles(a.n, a.m, a.d);
  const int64_t across = (a.m + 255) / 256, rounds = (a.n + 255) / 256 * across / 256;
  const int64_t head = rounds * 256 / across * 256;
  if (head > 0 && head < a.n) {
    const double first = static_cast<double>(rounds * ((a.d + kTileK - 1) / kTileK)) * 1.76;
    const TilePlan rest = plan_tiles(a.n - head, a.m, a.d);
    if (first + kSecond + rest.us < all.us) {
      ScoresI8Launch part = a;
      part.n = head;
      start_tile<Out>(part, extra, 256);
      part.n = a.n - head;
      part.X = static_cast<const int8_t*>(a.X) + head * a.ldx;
      part.sx = a.sx + head;
      part.S = static_cast<Out*>(a.S) + extra.first_row(head) * a.lds;
      start_tile<Out>(part, extra.from(head, 0), rest.tile);
      return;
    }
  }
  start_tile<Out>(a, extra, all.tile);
}

// By the examples' room in LDS; shorter rows of W leave most lanes without
// work, and the other kernels do better.
inline bool scores_i8_few(int64_t n, int64_t d) { return n <= 2 && d >= 512 && n * d <= 49152; }

}  // namespace
}  // namespace sdca_gpu

#endif  // SDCA_HIP_SCORES_I8_HPP
